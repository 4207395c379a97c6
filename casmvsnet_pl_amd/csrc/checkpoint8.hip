// 8-bit activation checkpoints (block8.h has the format): packing and reading back on their own, and the train-mode ABN that keeps, for its backward pass,
// 8 bits of the normalised input and one bit for the side of zero instead of its float32 input and output.
//
//   forward    xhat = (x - mean_c) rstd_c,  z = gamma_c xhat + beta_c,  y = z > 0 ? z : slope z;  kept: Q = 8 bits of xhat, s = [z > 0]
//   backward   g = gy (s ? 1 : slope),  gbeta = sum g,  ggamma = sum g Q,  gx = gamma rstd (g - gbeta / M - Q ggamma / M)
//
// xhat enters the gradient through ggamma and its product with Q only (both averages over the channel), so its 8 bits cost little there; the side of zero
// multiplies every gradient element, so it is kept exactly.  The statistics, xhat and z are computed in 64 bits: a block's codes and the sign of z are the
// ones of the definition, not of one order of float32 roundings.  y is formed in float32 from x - mean, with the mean as two floats, on the side of zero that z is
// on: at most four half steps of gamma xhat, wherever the channel lies, and both passes on the same side of the activation.
//
// Everything here waits for memory: forward 4 + 4 + 33/32 + 1/8 bytes read and written per element and 4 for the sums, backward sums 4 + 37/32, apply
// 8 + 37/32 (keeping x and y in float32 reads 12 and 12 and writes 4).  Measured, both launches of a pass together, forward / backward:
//   2 x 8 x 32 x 256 x 320   103 us (5.4 TB/s) / 95 us (6.3 TB/s: the second pass finds part of the first one's data in the caches)
//   6 x 8 x 512 x 640         39 us            / 38 us                 2 x 64 x 6 x 16 x 20   8.5 us / 6.8 us (one launch each)
// pack8 of 64 x 983040 float32 61 us, unpack8 47 us (5.2 and 6.7 TB/s), bf16 53 and 36 us (3.6 and 5.3); of 32 x 160 the time of a launch.
#include "block8.h"

namespace {
using casmvs::block8::kBlock;
using casmvs::block8::kLanes;
using casmvs::elem::Vec;

constexpr int kThreads = 256;
constexpr size_t kMostElements = (size_t)1 << 40;
constexpr int kGroups = kThreads / kLanes;   // blocks of 32 values that a workgroup works on at a time

// Four elements from `p` on, `left` of them real (0 .. 4); a missing one reads 0.
template <class T, bool WIDE>
__device__ __forceinline__ void load4(const T *p, int left, float (&v)[4]) {
  if (WIDE) {
    if (left > 0) {   // (planes of 4 n elements: all four or none)
      const Vec<T, 4> t = casmvs::elem::load<T, 4>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (float)t.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? (float)p[i] : 0.0f;
  }
}
// PAST: past the caches
template <class T, bool WIDE, bool PAST>
__device__ __forceinline__ void store4(T *p, int left, const float (&v)[4]) {
  if (WIDE) {
    if (left > 0) {
      Vec<T, 4> t;
#pragma unroll
      for (int i = 0; i < 4; ++i) t.v[i] = (T)v[i];
      if (PAST) casmvs::elem::store_past<T, 4>(p, t);
      else casmvs::elem::store<T, 4>(p, t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = (T)v[i];
  }
}
__device__ __forceinline__ int left_of(size_t n, size_t first) { return first >= n ? 0 : n - first < 4 ? (int)(n - first) : 4; }

// ---- pack / unpack ------------------------------------------------------------------------------------------------------------------------------------
constexpr int kAhead = 4;   // blocks per group of eight lanes whose loads are issued together

// Row and first value of a lane's four in block `blk` of (rows, nb); n % 32 == 0 came in as one long row.
__device__ __forceinline__ void place_of(size_t blk, size_t rows, size_t nb, int lane, size_t &row, size_t &first) {
  size_t in_row = blk;
  row = 0;
  if (rows > 1) casmvs::elem::divide(blk, nb, row, in_row);
  first = in_row * kBlock + 4 * lane;
}

template <class T, bool WIDE>
__global__ __launch_bounds__(kThreads) void pack8_kernel(const T *__restrict__ x, unsigned *__restrict__ codes, unsigned char *__restrict__ scales, size_t rows,
                                                        size_t n, size_t nb) {
  const size_t total = rows * nb, step = (size_t)gridDim.x * kGroups;
  const int lane = threadIdx.x & (kLanes - 1);
  // every lane of a wave takes the same number of turns (the exchanges inside a block need its eight lanes); a block past the end is empty
  for (size_t start = (size_t)blockIdx.x * kGroups; start < total; start += kAhead * step) {
    float v[kAhead][4];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const size_t blk = start + k * step + threadIdx.x / kLanes;
      size_t row, first;
      place_of(blk < total ? blk : 0, rows, nb, lane, row, first);
      load4<T, WIDE>(x + row * n + first, blk < total ? left_of(n, first) : 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const size_t blk = start + k * step + threadIdx.x / kLanes;
      const double d[4] = {v[k][0], v[k][1], v[k][2], v[k][3]};
      unsigned scale;
      const unsigned q = casmvs::block8::quantise(d, scale);
      if (blk < total) {
        codes[blk * kLanes + lane] = q;
        if (lane == 0) scales[blk] = (unsigned char)scale;
      }
    }
  }
}

// out = the held value, or (AFFINE) act(value * weight[c] + bias[c]) with c = row % C: an ABN's output from what its backward pass keeps
template <class T, bool WIDE, bool AFFINE, bool PAST>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(const unsigned *__restrict__ codes, const unsigned char *__restrict__ scales, T *__restrict__ out,
                                                          const float *__restrict__ weight, const float *__restrict__ bias, int C, float slope, size_t rows,
                                                          size_t n, size_t nb) {
  const size_t total = rows * nb, step = (size_t)gridDim.x * kGroups;
  const int lane = threadIdx.x & (kLanes - 1);
  for (size_t start = (size_t)blockIdx.x * kGroups + threadIdx.x / kLanes; start < total; start += kAhead * step) {
    unsigned q[kAhead], scale[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const size_t blk = start + k * step < total ? start + k * step : start;
      q[k] = codes[blk * kLanes + lane];
      scale[k] = scales[blk];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const size_t blk = start + k * step;
      if (blk >= total) break;
      size_t row, first;
      place_of(blk, rows, nb, lane, row, first);
      const float per = casmvs::block8::step_of(scale[k]);
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = casmvs::block8::value_of(q[k], i, per);
      if (AFFINE) {
        const int c = rows <= 0xFFFFFFFFu ? (int)((unsigned)row % (unsigned)C) : (int)(row % C);
        const float w = weight[c], b = bias[c];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float z = fmaf(v[i], w, b);
          v[i] = z > 0.0f ? z : z * slope;
        }
      }
      store4<T, WIDE, PAST>(out + row * n + first, left_of(n, first), v);
    }
  }
}

// ---- train-mode ABN -------------------------------------------------------------------------------------------------------------------------------------
// The sums over a channel are formed by kParts workgroups at most, each over its share [lo, hi) of every plane of the channel, and added up by every workgroup
// of the pass behind: one partial sum per lane of a wave, in a fixed order.  Few channels leave the chip short of workgroups by it: 16 M elements in 1 / 2 / 4 / 8
// channels take 98 / 65 / 48 / 42 us forward and 82 / 57 / 45 / 42 backward (no layer of the models has fewer than 8).
constexpr int kParts = 64;

// sums of two values per thread over a workgroup of THREADS, in every thread: lanes by exchange, then the waves' sums in their order
template <int THREADS>
__device__ __forceinline__ void workgroup_sums(double &s0, double &s1) {
  __shared__ double red[2][THREADS / 64];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    s0 += casmvs::elem::lane_xor(s0, d);
    s1 += casmvs::elem::lane_xor(s1, d);
  }
  if ((threadIdx.x & 63) == 0) {
    red[0][threadIdx.x >> 6] = s0;
    red[1][threadIdx.x >> 6] = s1;
  }
  __syncthreads();
  s0 = s1 = 0.0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    s0 += red[0][i];
    s1 += red[1][i];
  }
}

// The channel's two totals from its partial sums (C, parts, 2), parts <= 64, in every wave.
__device__ __forceinline__ void channel_totals(const double *__restrict__ sums, int parts, int c, double &t0, double &t1) {
  const int lane = threadIdx.x & 63;
  t0 = lane < parts ? sums[((size_t)c * parts + lane) * 2] : 0.0;
  t1 = lane < parts ? sums[((size_t)c * parts + lane) * 2 + 1] : 0.0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    t0 += casmvs::elem::lane_xor(t0, d);
    t1 += casmvs::elem::lane_xor(t1, d);
  }
}

// The channel's sums are of x - x0, x0 its first element: mean = x0 + s0 / M, var = s1 / M - (s0 / M)^2.  One element's distance to the mean squared is at most
// M var, whichever element it is, so the difference keeps var to M * 2^-53 however far from zero the channel lies (sums of x itself lose mean^2 / var * 2^-53 of it:
// 1e-3 at a mean of 3e6 and a spread of 1), and x0 is as a rule a few spreads from the mean: then all but var's last digits are right.
__device__ __forceinline__ float origin(const float *__restrict__ x, int c, size_t n) {
  const float x0 = x[c * n];
  return fabsf(x0) < INFINITY ? x0 : 0.0f;
}

// A workgroup's share [lo, hi) of a channel's planes, in words of four values, added to the sums of x - x0 and its square: in 64 bits from the first addition on,
// because xhat's codes and the side of zero hang on the mean.
template <bool WIDE, int THREADS>
__device__ __forceinline__ void add_squares(const float *__restrict__ x, float x0, int N, int C, int c, size_t n, size_t lo, size_t hi, double &s0, double &s1) {
  for (int img = 0; img < N; ++img) {
    const float *xp = x + ((size_t)img * C + c) * n;
    for (size_t e = lo + threadIdx.x; e < hi; e += 4 * THREADS) {
      float v[4][4];
      int left[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {   // four loads in flight, none of which waits for x0
        const size_t at = e + (size_t)k * THREADS;
        left[k] = at < hi ? left_of(n, 4 * at) : 0;
        load4<float, WIDE>(xp + 4 * at, left[k], v[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (left[k] == 0) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double d = (double)(WIDE || i < left[k] ? v[k][i] : x0) - (double)x0;
          s0 += d;
          s1 = fma(d, d, s1);
        }
      }
    }
  }
}

struct Channel {   // what the apply pass needs of a channel
  double mean, rstd;
  float high, low;   // of the mean
  float gamma, beta, scale;
};
struct Norm {      // arguments of either form of the forward pass
  const float *weight, *bias;
  float abs_eps, eps, momentum, slope;
  float *rmean, *rvar, *vec;   // vec (4, C): scale = gamma rstd, shift, gamma, beta of the forward pass
};
__device__ __forceinline__ Channel finish(const Norm &p, float x0, double s0, double s1, double M, int c, int C, bool write) {
  Channel k;
  const double off = s0 / M;
  k.mean = (double)x0 + off;
  double var = s1 / M - off * off;   // biased
  var = var > 0.0 ? var : (var != var ? var : 0.0);
  k.rstd = 1.0 / sqrt(var + (double)p.eps);
  k.gamma = p.abs_eps >= 0.0f ? fabsf(p.weight[c]) + p.abs_eps : p.weight[c];
  k.beta = p.bias[c];
  k.scale = (float)((double)k.gamma * k.rstd);
  k.high = (float)k.mean;
  k.low = (float)(k.mean - (double)k.high);
  if (write) {
    p.vec[c] = k.scale;
    p.vec[C + c] = (float)((double)k.beta - k.mean * (double)k.gamma * k.rstd);
    p.vec[2 * C + c] = k.gamma;
    p.vec[3 * C + c] = k.beta;
    if (p.rmean) {   // F.batch_norm: running = (1 - momentum) * running + momentum * batch (running_var: unbiased)
      const float keep = (float)(1.0 - (double)p.momentum);
      p.rmean[c] = p.rmean[c] * keep + p.momentum * (float)k.mean;
      p.rvar[c] = p.rvar[c] * keep + p.momentum * (float)(var * (M / (M > 1.0 ? M - 1.0 : 1.0)));
    }
  }
  return k;
}

struct Store {     // the 8-bit checkpoint of the normalised input and the signs of z
  unsigned *codes;
  unsigned char *scales;
  unsigned *signs;
};
// y and the checkpoint of the blocks blk0, blk0 + step, .. (kAhead of them, their loads issued together) of one plane.  Every lane of a wave comes here together.
template <bool WIDE, bool PAST>
__device__ __forceinline__ void apply_blocks(const float *__restrict__ xp, float *__restrict__ yp, const Store &to, size_t base, size_t blk0, size_t step, size_t n,
                                             size_t nb, int lane, const Channel &c, float slope) {
  float v[kAhead][4];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const size_t first = (blk0 + k * step) * kBlock + 4 * lane;
    load4<float, WIDE>(xp + first, left_of(n, first), v[k]);   // 0 past the plane's last block
  }
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const size_t blk = blk0 + k * step, first = blk * kBlock + 4 * lane;
    const int left = left_of(n, first);
    float o[4];
    double h[4];
    unsigned up = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[i] = i < left ? ((double)v[k][i] - c.mean) * c.rstd : 0.0;
      const bool above = fma(h[i], (double)c.gamma, (double)c.beta) > 0.0;
      up |= (above ? 1u : 0u) << i;
      // (z rounded from 64 bits instead: 60.2 -> 62.9 us at 2 x 8 x 32 x 256 x 320, 7.7 -> 8.6 at 2 x 32 x 24 x 32 x 40)
      const float t = fmaf((v[k][i] - c.high) - c.low, c.scale, c.beta);
      o[i] = above ? t : t * slope;
    }
    unsigned scale;
    const unsigned q = casmvs::block8::quantise(h, scale);
    const unsigned sign = casmvs::block8::over_block(up << (4 * lane), [](unsigned p, unsigned r) { return p | r; });
    store4<float, WIDE, PAST>(yp + first, left, o);
    if (blk < nb) {
      to.codes[(base + blk) * kLanes + lane] = q;
      if (lane == 0) {
        to.scales[base + blk] = (unsigned char)scale;
        to.signs[base + blk] = sign;
      }
    }
  }
}

// 512 threads: a pass that only reads needs more waves per CU than one that writes too (2 x 8 x 32 x 256 x 320 forward 111 us, with 256 threads 124; small maps lose with 1024)
constexpr int kSumThreads = 512;
template <bool WIDE>
__global__ __launch_bounds__(kSumThreads) void abn8_sums_kernel(const float *__restrict__ x, double *__restrict__ out, int N, int C, size_t n) {
  const int c = blockIdx.y;
  const size_t words = (n + 3) / 4, per = (words + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * per, hi = lo + per < words ? lo + per : words;
  double s0 = 0.0, s1 = 0.0;
  add_squares<WIDE, kSumThreads>(x, origin(x, c, n), N, C, c, n, lo, hi, s0, s1);
  workgroup_sums<kSumThreads>(s0, s1);
  if (threadIdx.x == 0) {
    out[((size_t)c * gridDim.x + blockIdx.x) * 2] = s0;
    out[((size_t)c * gridDim.x + blockIdx.x) * 2 + 1] = s1;
  }
}

constexpr int kTurns = 8;   // blocks per group of eight lanes and workgroup: 256 x 32 = 8192 elements share one read of the channel's partial sums

// blockIdx.x = (plane, chunk of kTurns * kGroups blocks)
template <bool WIDE, bool PAST>
__global__ __launch_bounds__(kThreads) void abn8_apply_kernel(const float *__restrict__ x, const double *__restrict__ sums, int parts, double M, Norm norm,
                                                             float *__restrict__ y, Store to, int C, size_t n, size_t nb, unsigned chunks) {
  const unsigned plane = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int c = (int)(plane % C);
  const float x0 = origin(x, c, n);   // (ahead of the totals' exchanges, which wait for whatever scalar load is under way)
  double s0, s1;
  channel_totals(sums, parts, c, s0, s1);
  const Channel k = finish(norm, x0, s0, s1, M, c, C, chunk == 0 && plane == (unsigned)c && threadIdx.x == 0);
  for (int turn = 0; turn < kTurns; turn += kAhead)
    apply_blocks<WIDE, PAST>(x + plane * n, y + plane * n, to, plane * nb, ((size_t)chunk * kTurns + turn) * kGroups + threadIdx.x / kLanes, kGroups, n, nb,
                       threadIdx.x & (kLanes - 1), k, norm.slope);
}

// A channel per workgroup, both passes: one launch where a channel is small (kOneLaunch)
constexpr int kWide = 1024;   // threads of the one-launch forms
template <bool WIDE>
__global__ __launch_bounds__(kWide) void abn8_forward_one_kernel(const float *__restrict__ x, double M, Norm norm, float *__restrict__ y, Store to, int N, int C, size_t n,
                                                                size_t nb) {
  constexpr int groups = kWide / kLanes;
  const int c = blockIdx.x;
  double s0 = 0.0, s1 = 0.0;
  const float x0 = origin(x, c, n);
  add_squares<WIDE, kWide>(x, x0, N, C, c, n, 0, (n + 3) / 4, s0, s1);
  workgroup_sums<kWide>(s0, s1);
  const Channel k = finish(norm, x0, s0, s1, M, c, C, threadIdx.x == 0);
  for (int img = 0; img < N; ++img) {
    const size_t plane = (size_t)img * C + c;
    for (size_t blk = 0; blk < nb; blk += kAhead * groups)
      apply_blocks<WIDE, false>(x + plane * n, y + plane * n, to, plane * nb, blk + threadIdx.x / kLanes, groups, n, nb, threadIdx.x & (kLanes - 1), k, norm.slope);
  }
}

// What the backward pass reads of four values: their gradient behind the activation and Q
struct Kept {
  float g[4];
  unsigned q, up;
  float step;
};
struct Checkpoint {
  const unsigned *codes;
  const unsigned char *scales;
  const unsigned *signs;
};
template <bool WIDE>
__device__ __forceinline__ void load_kept(const float *__restrict__ gy, const Checkpoint &from, size_t plane, size_t blk, size_t n, size_t nb, int lane, Kept &k) {
  const size_t first = blk * kBlock + 4 * lane, at = plane * nb + (blk < nb ? blk : 0);
  load4<float, WIDE>(gy + plane * n + first, left_of(n, first), k.g);   // 0 past the plane's last block
  k.q = from.codes[at * kLanes + lane];
  k.up = from.signs[at] >> (4 * lane);
  k.step = casmvs::block8::step_of(from.scales[at]);
}
__device__ __forceinline__ float behind_activation(const Kept &k, int i, float slope) { return k.g[i] * ((k.up >> i) & 1u ? 1.0f : slope); }

// the blocks [lo, hi) of a channel's planes, added to sum g and sum g Q
template <bool WIDE, int THREADS>
__device__ __forceinline__ void add_gradients(const float *__restrict__ gy, const Checkpoint &from, int N, int C, int c, size_t n, size_t nb, size_t lo, size_t hi,
                                              float slope, double &s0, double &s1) {
  constexpr int groups = THREADS / kLanes;
  const int lane = threadIdx.x & (kLanes - 1);
  for (int img = 0; img < N; ++img) {
    const size_t plane = (size_t)img * C + c;
    for (size_t blk = lo + threadIdx.x / kLanes; blk < hi; blk += kAhead * groups) {
      Kept k[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const size_t at = blk + (size_t)j * groups;
        load_kept<WIDE>(gy, from, plane, at < hi ? at : nb, n, nb, lane, k[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (blk + (size_t)j * groups >= hi) break;
        float p0 = 0.0f, p1 = 0.0f;   // four values in float32, then 64 bits
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = behind_activation(k[j], i, slope);
          p0 += g;
          p1 = fmaf(g, casmvs::block8::value_of(k[j].q, i, k[j].step), p1);
        }
        s0 += p0;
        s1 += p1;
      }
    }
  }
}

template <bool WIDE>
__global__ __launch_bounds__(kSumThreads) void abn8_backward_sums_kernel(const float *__restrict__ gy, Checkpoint from, double *__restrict__ out, int N, int C, size_t n,
                                                                     size_t nb, float slope) {
  const int c = blockIdx.y;
  const size_t per = (nb + gridDim.x - 1) / gridDim.x, lo = blockIdx.x * per, hi = lo + per < nb ? lo + per : nb;
  double s0 = 0.0, s1 = 0.0;
  add_gradients<WIDE, kSumThreads>(gy, from, N, C, c, n, nb, lo, hi, slope, s0, s1);
  workgroup_sums<kSumThreads>(s0, s1);
  if (threadIdx.x == 0) {
    out[((size_t)c * gridDim.x + blockIdx.x) * 2] = s0;
    out[((size_t)c * gridDim.x + blockIdx.x) * 2 + 1] = s1;
  }
}

struct Gradients {
  const float *weight, *vec;
  float abs_eps, slope;
  float *gweight, *gbias, *gx;   // gx may be null
};
struct Means {   // of g and g Q, and gamma rstd
  float m1, m2, a;
};
__device__ __forceinline__ Means finish_gradients(const Gradients &p, double s0, double s1, double M, int c, bool write) {
  if (write) {
    const float w = p.weight[c];
    const float sgn = p.abs_eps >= 0.0f ? (w > 0.0f ? 1.0f : (w < 0.0f ? -1.0f : 0.0f)) : 1.0f;   // d|w| / dw
    p.gweight[c] = (float)s1 * sgn;
    p.gbias[c] = (float)s0;
  }
  return Means{(float)(s0 / M), (float)(s1 / M), p.vec[c]};
}
template <bool WIDE, bool PAST>
__device__ __forceinline__ void gradient_blocks(const float *__restrict__ gy, const Checkpoint &from, float *__restrict__ gx, size_t plane, size_t blk0, size_t step, size_t n,
                                                size_t nb, const Means &m, float slope) {
  const int lane = threadIdx.x & (kLanes - 1);
  Kept k[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) load_kept<WIDE>(gy, from, plane, blk0 + j * step, n, nb, lane, k[j]);
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const size_t first = (blk0 + j * step) * kBlock + 4 * lane;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = m.a * (behind_activation(k[j], i, slope) - m.m1 - casmvs::block8::value_of(k[j].q, i, k[j].step) * m.m2);
    store4<float, WIDE, PAST>(gx + plane * n + first, left_of(n, first), o);
  }
}

template <bool WIDE, bool PAST>
__global__ __launch_bounds__(kThreads) void abn8_backward_apply_kernel(const float *__restrict__ gy, Checkpoint from, const double *__restrict__ sums, int parts, double M,
                                                                      Gradients p, int C, size_t n, size_t nb, unsigned chunks) {
  const unsigned plane = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const int c = (int)(plane % C);
  double s0, s1;
  channel_totals(sums, parts, c, s0, s1);
  const Means m = finish_gradients(p, s0, s1, M, c, chunk == 0 && plane == (unsigned)c && threadIdx.x == 0);
  if (!p.gx) return;
  for (int turn = 0; turn < kTurns; turn += kAhead)
    gradient_blocks<WIDE, PAST>(gy, from, p.gx, plane, ((size_t)chunk * kTurns + turn) * kGroups + threadIdx.x / kLanes, kGroups, n, nb, m, p.slope);
}

template <bool WIDE>
__global__ __launch_bounds__(kWide) void abn8_backward_one_kernel(const float *__restrict__ gy, Checkpoint from, double M, Gradients p, int N, int C, size_t n, size_t nb) {
  constexpr int groups = kWide / kLanes;
  const int c = blockIdx.x;
  double s0 = 0.0, s1 = 0.0;
  add_gradients<WIDE, kWide>(gy, from, N, C, c, n, nb, 0, nb, p.slope, s0, s1);
  workgroup_sums<kWide>(s0, s1);
  const Means m = finish_gradients(p, s0, s1, M, c, threadIdx.x == 0);
  if (!p.gx) return;
  for (int img = 0; img < N; ++img)
    for (size_t blk = 0; blk < nb; blk += kAhead * groups)
      gradient_blocks<WIDE, false>(gy, from, p.gx, (size_t)img * C + c, blk + threadIdx.x / kLanes, groups, n, nb, m, p.slope);
}

// Elements of a channel up to which one workgroup does both passes over it: one launch less, on as many CUs as there are channels.  Forward / backward in one launch
// and in two: 64 channels of 8192 elements 7.1 / 6.5 and 8.6 / 8.9 us, of 16384 8.4 / 8.5 and 9.2 / 8.8, of 32768 14.4 / 12.3 and 11.3 / 10.5; 256 of 16384
// 11.4 / 11.0 and 14.7 / 13.6.
constexpr size_t kOneLaunch = 16384;

// Workgroups that form a channel's sums: at least 4096 elements each, at most 1024 workgroups in all (four per CU)
int parts_of(int N, int C, size_t n) {
  const size_t most = 1024 / (size_t)C < 1 ? 1 : 1024 / (size_t)C, wanted = ((size_t)N * n + 4095) / 4096;
  const size_t parts = wanted < most ? wanted : most;
  return (int)(parts < 1 ? 1 : parts > kParts ? kParts : parts);
}
size_t blocks_of(size_t n) { return (n + kBlock - 1) / kBlock; }
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_planes(const char *what, int N, int C, size_t n) {
  CASMVS_REQUIRE(N > 0 && C > 0 && C <= 65535 && n > 0, "%s: N=%d C=%d n=%zu", what, N, C, n);
  const size_t chunks = (blocks_of(n) + kTurns * kGroups - 1) / (kTurns * kGroups);
  // (a launch has fewer than 2^32 threads)
  CASMVS_REQUIRE((size_t)N * C <= ((size_t)1 << 21) && chunks < ((size_t)1 << 24) / ((size_t)N * C), "%s: %d x %d planes of %zu elements", what, N, C, n);
  return CASMVS_OK;
}
}  // namespace

extern "C" int casmvs_pack8(const void *x, int dtype, size_t rows, size_t n, void *codes, void *scales, void *stream) {
  casmvs::clear_error();
  CASMVS_REQUIRE(casmvs::elem::known(dtype), "pack8: dtype %d", dtype);
  if (rows == 0 || n == 0) return CASMVS_OK;
  CASMVS_REQUIRE(x && codes && scales, "pack8: null pointer");
  CASMVS_REQUIRE(((uintptr_t)codes & 3) == 0, "pack8: codes are written four at a time (4-byte alignment)");
  CASMVS_REQUIRE(n <= kMostElements && rows <= kMostElements / n, "pack8: %zu rows of %zu", rows, n);
  if (n % kBlock == 0) { n *= rows; rows = 1; }   // blocks do not end inside a row: one long row
  const size_t nb = blocks_of(n), total = rows * nb;
  const size_t wanted = (total + kGroups - 1) / kGroups;
  const unsigned grid = (unsigned)(wanted < 8192 ? wanted : 8192);
  const bool wide = n % 4 == 0 && aligned16(x);
  CASMVS_WITH_DTYPE(dtype, {
    if (wide)
      hipLaunchKernelGGL((pack8_kernel<T, true>), dim3(grid), dim3(kThreads), 0, (hipStream_t)stream, (const T *)x, (unsigned *)codes, (unsigned char *)scales, rows, n, nb);
    else
      hipLaunchKernelGGL((pack8_kernel<T, false>), dim3(grid), dim3(kThreads), 0, (hipStream_t)stream, (const T *)x, (unsigned *)codes, (unsigned char *)scales, rows, n, nb);
  });
  return casmvs::check_launch("pack8_kernel");
}

extern "C" int casmvs_unpack8(const void *codes, const void *scales, const float *weight, const float *bias, int C, float slope, void *out, int dtype,
                              size_t rows, size_t n, void *stream) {
  casmvs::clear_error();
  CASMVS_REQUIRE(casmvs::elem::known(dtype), "unpack8: dtype %d", dtype);
  if (rows == 0 || n == 0) return CASMVS_OK;
  CASMVS_REQUIRE(codes && scales && out, "unpack8: null pointer");
  CASMVS_REQUIRE(((uintptr_t)codes & 3) == 0, "unpack8: codes are read four at a time (4-byte alignment)");
  CASMVS_REQUIRE((weight == nullptr) == (bias == nullptr) && (!weight || C > 0), "unpack8: weight and bias go together, with their number of channels");
  CASMVS_REQUIRE(n <= kMostElements && rows <= kMostElements / n, "unpack8: %zu rows of %zu", rows, n);
  if (n % kBlock == 0 && !weight) { n *= rows; rows = 1; }
  const size_t nb = blocks_of(n), total = rows * nb;
  const size_t wanted = (total + kGroups - 1) / kGroups;
  const unsigned grid = (unsigned)(wanted < 8192 ? wanted : 8192);
  const bool wide = n % 4 == 0 && aligned16(out);
  const bool past = wide && casmvs::elem::streams(rows * n * casmvs::elem::size_of(dtype));
#define CASMVS_UNPACK8(W, A, P)                                                                                                                       \
  hipLaunchKernelGGL((unpack8_kernel<T, W, A, P>), dim3(grid), dim3(kThreads), 0, (hipStream_t)stream, (const unsigned *)codes, (const unsigned char *)scales, \
                     (T *)out, weight, bias, C, slope, rows, n, nb)
  CASMVS_WITH_DTYPE(dtype, {
    if (weight) {
      if (past) CASMVS_UNPACK8(true, true, true); else if (wide) CASMVS_UNPACK8(true, true, false); else CASMVS_UNPACK8(false, true, false);
    } else {
      if (past) CASMVS_UNPACK8(true, false, true); else if (wide) CASMVS_UNPACK8(true, false, false); else CASMVS_UNPACK8(false, false, false);
    }
  });
#undef CASMVS_UNPACK8
  return casmvs::check_launch("unpack8_kernel");
}

extern "C" size_t casmvs_abn8_workspace_bytes(int N, int C, size_t n) {
  if (N <= 0 || C <= 0 || n == 0) return 0;
  return (size_t)C * parts_of(N, C, n) * 2 * sizeof(double);
}

extern "C" int casmvs_abn8_forward_f32(const float *x, const float *weight, const float *bias, float abs_eps, float eps, float momentum, float *running_mean,
                                       float *running_var, float *vec, float *y, void *codes, void *scales, void *signs, void *workspace, int N, int C,
                                       size_t n, float slope, void *stream) {
  casmvs::clear_error();
  if (int rc = check_planes("abn8_forward", N, C, n)) return rc;
  CASMVS_REQUIRE(x && weight && bias && vec && y && codes && scales && signs && workspace, "abn8_forward: null pointer");
  CASMVS_REQUIRE((running_mean == nullptr) == (running_var == nullptr), "abn8_forward: running_mean and running_var go together");
  CASMVS_REQUIRE((((uintptr_t)codes | (uintptr_t)signs) & 3) == 0 && ((uintptr_t)workspace & 7) == 0,
                 "abn8_forward: codes and signs are 4-byte words, the workspace 8-byte ones");
  const size_t nb = blocks_of(n), chunks = (nb + kTurns * kGroups - 1) / (kTurns * kGroups);
  const int parts = parts_of(N, C, n);
  const double count = (double)N * (double)n;
  double *sums = (double *)workspace;
  hipStream_t st = (hipStream_t)stream;
  const bool wide = n % 4 == 0 && aligned16(x) && aligned16(y);
  const Norm norm{weight, bias, abs_eps, eps, momentum, slope, running_mean, running_var, vec};
  const Store to{(unsigned *)codes, (unsigned char *)scales, (unsigned *)signs};
  if ((size_t)N * n <= kOneLaunch) {
    hipLaunchKernelGGL(wide ? abn8_forward_one_kernel<true> : abn8_forward_one_kernel<false>, dim3((unsigned)C), dim3(kWide), 0, st, x, count, norm, y, to, N, C, n, nb);
    return casmvs::check_launch("abn8_forward_one_kernel");
  }
  hipLaunchKernelGGL(wide ? abn8_sums_kernel<true> : abn8_sums_kernel<false>, dim3((unsigned)parts, (unsigned)C), dim3(kSumThreads), 0, st, x, sums, N, C, n);
  const bool past = wide && casmvs::elem::streams((size_t)N * C * n * sizeof(float));
  auto apply = past ? abn8_apply_kernel<true, true> : wide ? abn8_apply_kernel<true, false> : abn8_apply_kernel<false, false>;
  hipLaunchKernelGGL(apply, dim3((unsigned)((size_t)N * C * chunks)), dim3(kThreads), 0, st, x, sums, parts, count, norm,
                     y, to, C, n, nb, (unsigned)chunks);
  return casmvs::check_launch("abn8_forward");
}

extern "C" int casmvs_abn8_backward_f32(const float *grad_y, const void *codes, const void *scales, const void *signs, const float *weight, float abs_eps,
                                        const float *vec, float *grad_weight, float *grad_bias, float *grad_x, void *workspace, int N, int C, size_t n,
                                        float slope, void *stream) {
  casmvs::clear_error();
  if (int rc = check_planes("abn8_backward", N, C, n)) return rc;
  CASMVS_REQUIRE(grad_y && codes && scales && signs && weight && vec && grad_weight && grad_bias && workspace, "abn8_backward: null pointer");
  CASMVS_REQUIRE((((uintptr_t)codes | (uintptr_t)signs) & 3) == 0 && ((uintptr_t)workspace & 7) == 0,
                 "abn8_backward: codes and signs are 4-byte words, the workspace 8-byte ones");
  const size_t nb = blocks_of(n);
  size_t chunks = (nb + kTurns * kGroups - 1) / (kTurns * kGroups);
  const int parts = parts_of(N, C, n);
  const double count = (double)N * (double)n;
  double *sums = (double *)workspace;
  hipStream_t st = (hipStream_t)stream;
  const bool wide = n % 4 == 0 && aligned16(grad_y) && aligned16(grad_x);
  const Checkpoint from{(const unsigned *)codes, (const unsigned char *)scales, (const unsigned *)signs};
  const Gradients to{weight, vec, abs_eps, slope, grad_weight, grad_bias, grad_x};
  if ((size_t)N * n <= kOneLaunch) {
    hipLaunchKernelGGL(wide ? abn8_backward_one_kernel<true> : abn8_backward_one_kernel<false>, dim3((unsigned)C), dim3(kWide), 0, st, grad_y, from, count, to, N, C, n, nb);
    return casmvs::check_launch("abn8_backward_one_kernel");
  }
  hipLaunchKernelGGL(wide ? abn8_backward_sums_kernel<true> : abn8_backward_sums_kernel<false>, dim3((unsigned)parts, (unsigned)C), dim3(kSumThreads), 0, st, grad_y, from, sums,
                     N, C, n, nb, slope);
  // (without grad_x one workgroup per channel, as if a plane had one chunk, writes the two vectors)
  if (!grad_x) chunks = 1;
  const dim3 grid((unsigned)(grad_x ? (size_t)N * C * chunks : (size_t)C));
  const bool past = wide && casmvs::elem::streams((size_t)N * C * n * sizeof(float));
  auto apply = past ? abn8_backward_apply_kernel<true, true> : wide ? abn8_backward_apply_kernel<true, false> : abn8_backward_apply_kernel<false, false>;
  hipLaunchKernelGGL(apply, grid, dim3(kThreads), 0, st, grad_y, from, sums, parts, count, to, C, n, nb,
                     (unsigned)chunks);
  return casmvs::check_launch("abn8_backward");
}
