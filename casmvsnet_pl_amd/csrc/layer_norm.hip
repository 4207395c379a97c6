// Layer norm over the channel axis + leaky ReLU, forward and backward.
//
//   position p of (outer, C, inner), channels c:   mu = mean_c x,  v = mean_c (x - mu)^2,  r = 1 / sqrt(v + eps),  h = (x - mu) r
//   z = h w_c + b_c,   y = z > 0 ? z : slope z
//   g = gy (z > 0 ? 1 : slope),  m1 = mean_c (g w),  m2 = mean_c (g w h):   gx = r (g w - m1 - h m2),  gw_c = sum_p g h,  gb_c = sum_p g
//
// The backward pass takes x and recomputes mu, r and the side of zero that z lies on: x has to be read for h anyway, and two stored floats per position
// would be a quarter of the traffic at 8 channels.  Statistics, z and gx are held in 64 bits.  An element whose z is within float32's rounding of zero would
// otherwise get the slope in one computation and 1 in another, an error of the size of the gradient itself, and at two or three channels gx is what is left
// after cancellation.  The vector ALU does 64-bit multiply-adds at the rate of scalar float32 ones, and these kernels wait for memory.
//
// Three forms, by where a position's channels lie and how many there are:
//   planes  (inner > 1, C <= 512)   a thread holds 8 channels of 4 (or 1) consecutive positions in registers, up to 64 threads share a position;
//   rows    (inner = 1, C <= 8192)  up to 64 lanes of a wave, or a workgroup, hold a row in registers;
//   any     everything else: x is read once per use.
#include "elem_types.h"

namespace {
using casmvs::elem::lane_xor;
using casmvs::elem::Vec;

constexpr int kThreads = 256;
constexpr int kSlicePositions = 1024;   // (any) positions per slice of the weight gradient's partial sums, before kMostSlices is reached
constexpr int kMostSlices = 256;

// 1 / sqrt(a) for a > 0: the hardware's estimate (about 24 bits) and one Newton step (about 48 bits)
__device__ __forceinline__ double inverse_sqrt(double a) {
  const double r = __builtin_amdgcn_rsq(a);
  return r * (1.5 - 0.5 * a * r * r);
}

// ---- planes ----------------------------------------------------------------------------------------------------------------------------------------------
// The workgroup's tile is PL * V consecutive positions (PL = 256 / CG) x all channels: lane pl holds the V positions from (tile * PL + pl) * V on, channel
// group cg the channels cg, cg + CG, ...  A wave's loads run along the positions (PL * V elements), its channels are the same where PL >= 64.
constexpr int kHeld = 8;   // channels per thread

template <int CG, int V>
struct PlaneTile {
  static constexpr int PL = kThreads / CG;
  int pl, cg;
  __device__ __forceinline__ PlaneTile() {
    pl = threadIdx.x % PL;
    cg = PL >= 64 ? (int)__builtin_amdgcn_readfirstlane(threadIdx.x / PL) : threadIdx.x / PL;   // the same in a wave: its weights are scalar loads
  }
  // Sums over the channel groups of `N` <= MOST values for each of the thread's V positions, given to all of them.  lds: plane_lds(MOST) doubles; the totals lie
  // behind the MOST parts whatever N is, so that a thread may write the next sums' parts while another still reads these totals.
  template <int N, int MOST>
  __device__ __forceinline__ void over_groups(double (&v)[N][V], double *lds) const {
    if (CG == 1) return;
    constexpr int P = PL * V;   // positions of the tile
    double *total = lds + MOST * CG * P;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) lds[(k * CG + cg) * P + i * PL + pl] = v[k][i];
    __syncthreads();
    for (int o = threadIdx.x; o < N * P; o += kThreads) {
      double s = 0.0;
#pragma unroll
      for (int g = 0; g < CG; ++g) s += lds[((o / P) * CG + g) * P + o % P];
      total[o] = s;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = total[k * P + i * PL + pl];
  }
};
template <int CG, int V>
constexpr int plane_lds(int most) { return CG == 1 ? 1 : most * kThreads * V + most * kThreads / CG * V; }

template <class T, int V>
__device__ __forceinline__ void load_planes(const T *__restrict__ x, size_t base, size_t inner, int first, int step, int C, bool live, float (&v)[kHeld][V]) {
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    const int c = first + r * step;
    if (live && c < C) {
      const Vec<T, V> t = casmvs::elem::load<T, V>(x + base + c * inner);
#pragma unroll
      for (int i = 0; i < V; ++i) v[r][i] = (float)t.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[r][i] = 0.0f;
    }
  }
}

// mean and 1 / sqrt(var + eps) of the thread's positions
template <int MOST, int CG, int V>
__device__ __forceinline__ void plane_statistics(const PlaneTile<CG, V> &tile, const float (&v)[kHeld][V], int C, double per_c, float eps, double *lds, double (&mean)[V],
                                                 double (&rstd)[V]) {
  double s[1][V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[0][i] = 0.0;
#pragma unroll
  for (int r = 0; r < kHeld; ++r)
#pragma unroll
    for (int i = 0; i < V; ++i) s[0][i] += (double)v[r][i];   // (a missing channel holds 0)
  tile.template over_groups<1, MOST>(s, lds);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mean[i] = s[0][i] * per_c;
    s[0][i] = 0.0;
  }
#pragma unroll
  for (int r = 0; r < kHeld; ++r)
    if (tile.cg + r * CG < C) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = (double)v[r][i] - mean[i];
        s[0][i] = fma(d, d, s[0][i]);
      }
    }
  tile.template over_groups<1, MOST>(s, lds);
#pragma unroll
  for (int i = 0; i < V; ++i) rstd[i] = inverse_sqrt(s[0][i] * per_c + (double)eps);
}

template <class T, int CG, int V>
__global__ __launch_bounds__(kThreads) void ln_forward_planes_kernel(const T *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b,
                                                                    T *__restrict__ y, size_t positions, int C, size_t inner, double per_c, float eps,
                                                                    float slope) {
  __shared__ double lds[plane_lds<CG, V>(1)];
  const PlaneTile<CG, V> tile;
  const size_t p = ((size_t)blockIdx.x * PlaneTile<CG, V>::PL + tile.pl) * V;
  const bool live = p < positions;   // (V divides inner: all V positions or none, in one plane)
  const size_t n = live ? p / inner : 0, base = n * C * inner + (live ? p - n * inner : 0);
  float v[kHeld][V];
  load_planes<T, V>(x, base, inner, tile.cg, CG, C, live, v);
  double mean[V], rstd[V];
  plane_statistics<1, CG, V>(tile, v, C, per_c, eps, lds, mean, rstd);
  if (!live) return;
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    const int c = tile.cg + r * CG;
    if (c >= C) break;
    const double wc = w ? (double)w[c] : 1.0, bc = b ? (double)b[c] : 0.0;
    Vec<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double z = fma(((double)v[r][i] - mean[i]) * rstd[i], wc, bc);
      t.v[i] = (T)(float)(z > 0.0 ? z : z * slope);
    }
    casmvs::elem::store<T, V>(y + base + c * inner, t);
  }
}

// gx, and of every workgroup the sums over its tiles of g h and g per channel: partial[workgroup][0 / 1][c].  AFFINE: the weight gradient is wanted.
template <class T, int CG, int V, bool AFFINE>
__global__ __launch_bounds__(kThreads) void ln_backward_planes_kernel(const T *__restrict__ x, const T *__restrict__ gy, const float *__restrict__ w,
                                                                     const float *__restrict__ b, T *__restrict__ gx, float *__restrict__ partial,
                                                                     size_t positions, size_t tiles, int C, size_t inner, double per_c, float eps, float slope) {
  using Tile = PlaneTile<CG, V>;
  constexpr int kSums = plane_lds<CG, V>(2) > 2 * kHeld * kThreads / 2 ? plane_lds<CG, V>(2) : 2 * kHeld * kThreads / 2;
  __shared__ double lds[kSums];   // (the groups' sums; at the end 2 * kHeld * 256 floats)
  const Tile tile;
  float sw[kHeld], sb[kHeld];   // this thread's share of sum g h and sum g: positions / (workgroups * PL) values each
#pragma unroll
  for (int r = 0; r < kHeld; ++r) sw[r] = sb[r] = 0.0f;
  for (size_t k = blockIdx.x; k < tiles; k += gridDim.x) {
    const size_t p = (k * Tile::PL + tile.pl) * V;
    const bool live = p < positions;
    const size_t n = live ? p / inner : 0, base = n * C * inner + (live ? p - n * inner : 0);
    float v[kHeld][V], g[kHeld][V];
    load_planes<T, V>(x, base, inner, tile.cg, CG, C, live, v);
    load_planes<T, V>(gy, base, inner, tile.cg, CG, C, live, g);
    double mean[V], rstd[V], m[2][V];
    plane_statistics<2, CG, V>(tile, v, C, per_c, eps, lds, mean, rstd);
#pragma unroll
    for (int i = 0; i < V; ++i) m[0][i] = m[1][i] = 0.0;
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int c = tile.cg + r * CG;
      if (c < C) {
        const double wc = w ? (double)w[c] : 1.0, bc = b ? (double)b[c] : 0.0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const double h = ((double)v[r][i] - mean[i]) * rstd[i];
          g[r][i] *= fma(h, wc, bc) > 0.0 ? 1.0f : slope;
          const double gw = (double)g[r][i] * wc;
          m[0][i] += gw;
          m[1][i] = fma(gw, h, m[1][i]);
          if (AFFINE) {
            sb[r] += g[r][i];
            sw[r] = fmaf(g[r][i], (float)h, sw[r]);
          }
        }
      }
    }
    if (gx) {
      tile.template over_groups<2, 2>(m, lds);
      if (live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          m[0][i] *= per_c;
          m[1][i] *= per_c;
        }
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
          const int c = tile.cg + r * CG;
          if (c >= C) break;
          const double wc = w ? (double)w[c] : 1.0;
          Vec<T, V> t;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const double h = ((double)v[r][i] - mean[i]) * rstd[i];
            t.v[i] = (T)(float)(rstd[i] * ((double)g[r][i] * wc - m[0][i] - h * m[1][i]));
          }
          casmvs::elem::store<T, V>(gx + base + c * inner, t);
        }
      }
    }
  }
  if (!AFFINE) return;
  // Sums over the PL lanes of each (kind, held channel, group): first S of them per thread, PL / S apart or one behind the other ...
  float *red = reinterpret_cast<float *>(lds);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    red[r * kThreads + threadIdx.x] = sw[r];
    red[(kHeld + r) * kThreads + threadIdx.x] = sb[r];
  }
  __syncthreads();
  constexpr int J = Tile::PL >= 16 ? 16 : Tile::PL;   // threads per sum
  for (int o = threadIdx.x / J; o < 2 * kHeld * CG; o += kThreads / J) {
    const int j = threadIdx.x % J, value = o / CG, group = o % CG;
    double s = 0.0;
    for (int l = j; l < Tile::PL; l += J) s += (double)red[value * kThreads + group * Tile::PL + l];
    // ... then those J, by neighbouring lanes
#pragma unroll
    for (int d = 1; d < J; d <<= 1) s += lane_xor(s, d);
    const int c = group + (value % kHeld) * CG;
    if (j == 0 && c < C) partial[((size_t)blockIdx.x * 2 + value / kHeld) * C + c] = (float)s;
  }
}

// ---- rows -------------------------------------------------------------------------------------------------------------------------------------------------
// L lanes hold a row: vector j of lane t covers the channels (j L + t) V .. + V - 1, j < K.  L <= 64: a wave works on 64 / L rows; L = 256, 512: a workgroup on
// one.  At most 16 channels per lane: the backward pass holds six values for each (x, gy, the affine and its two sums), and 32 of them spill.
template <int L>
constexpr int row_threads() { return L < kThreads ? kThreads : L; }

template <int L, int N>
__device__ __forceinline__ void over_row(double (&v)[N], double *lds) {
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int d = 1; d < (L < 64 ? L : 64); d <<= 1) v[k] += lane_xor(v[k], d);
  if (L > 64) {
    constexpr int W = L / 64;
    __syncthreads();   // (lds may still be read from the last use)
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) lds[k * W + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = lds[k * W];
#pragma unroll
      for (int i = 1; i < W; ++i) v[k] += lds[k * W + i];
    }
  }
}

template <class T, int L, int V, int K>
__device__ __forceinline__ void load_row(const T *__restrict__ x, size_t base, int t, int C, bool live, float (&v)[K][V]) {
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int c = (j * L + t) * V;
    if (live && c < C) {
      const Vec<T, V> u = casmvs::elem::load<T, V>(x + base + c);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = (float)u.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = 0.0f;
    }
  }
}

template <int L, int V, int K>
__device__ __forceinline__ void row_statistics(const float (&v)[K][V], int t, int C, double per_c, float eps, double *lds, double &mean, double &rstd) {
  double s[1] = {0.0};
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) s[0] += (double)v[j][i];
  over_row<L, 1>(s, lds);
  mean = s[0] * per_c;
  s[0] = 0.0;
#pragma unroll
  for (int j = 0; j < K; ++j)
    if ((j * L + t) * V < C) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = (double)v[j][i] - mean;
        s[0] = fma(d, d, s[0]);
      }
    }
  over_row<L, 1>(s, lds);
  rstd = inverse_sqrt(s[0] * per_c + (double)eps);
}

template <class T, int L, int V, int K>
__global__ __launch_bounds__(row_threads<L>()) void ln_forward_rows_kernel(const T *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b, T *__restrict__ y,
                                                                  size_t rows, int C, double per_c, float eps, float slope) {
  __shared__ double lds[row_threads<L>() / 64];
  const int t = threadIdx.x % L;
  const size_t row = (size_t)blockIdx.x * (row_threads<L>() / L) + threadIdx.x / L;
  const bool live = row < rows;
  const size_t base = live ? row * C : 0;
  float v[K][V];
  load_row<T, L, V, K>(x, base, t, C, live, v);
  double mean, rstd;
  row_statistics<L, V, K>(v, t, C, per_c, eps, lds, mean, rstd);
  if (!live) return;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int c = (j * L + t) * V;
    if (c >= C) break;
    Vec<T, V> u;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double z = fma(((double)v[j][i] - mean) * rstd, w ? (double)w[c + i] : 1.0, b ? (double)b[c + i] : 0.0);
      u.v[i] = (T)(float)(z > 0.0 ? z : z * slope);
    }
    casmvs::elem::store<T, V>(y + base + c, u);
  }
}

// gx, and of every workgroup the sums over its rows of g h and g: a thread keeps its channels for all of them.  partial[workgroup][0 / 1][c].
template <class T, int L, int V, int K, bool AFFINE>
__global__ __launch_bounds__(row_threads<L>()) void ln_backward_rows_kernel(const T *__restrict__ x, const T *__restrict__ gy, const float *__restrict__ w,
                                                                   const float *__restrict__ b, T *__restrict__ gx, float *__restrict__ partial, size_t rows,
                                                                   int C, double per_c, float eps, float slope) {
  constexpr int BT = row_threads<L>(), G = BT / L;   // rows at a time
  __shared__ double lds[2 * BT / 64];
  __shared__ float red[AFFINE && G > 1 ? K * V * BT : 1];
  const int t = threadIdx.x % L;
  float wc[K][V], bc[K][V], sw[K][V], sb[K][V];
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (j * L + t) * V + i;
      wc[j][i] = w && c < C ? w[c] : 1.0f;
      bc[j][i] = b && c < C ? b[c] : 0.0f;
      sw[j][i] = sb[j][i] = 0.0f;
    }
  const size_t turns = (rows + (size_t)gridDim.x * G - 1) / ((size_t)gridDim.x * G);   // the same for every thread: the exchanges need all lanes
  for (size_t turn = 0; turn < turns; ++turn) {
    const size_t row = (turn * gridDim.x + blockIdx.x) * G + threadIdx.x / L;
    const bool live = row < rows;
    const size_t base = live ? row * C : 0;
    float v[K][V], g[K][V];
    load_row<T, L, V, K>(x, base, t, C, live, v);
    load_row<T, L, V, K>(gy, base, t, C, live, g);
    double mean, rstd, m[2] = {0.0, 0.0};
    row_statistics<L, V, K>(v, t, C, per_c, eps, lds, mean, rstd);
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {   // (g of a missing channel is 0)
        const double h = ((double)v[j][i] - mean) * rstd;
        g[j][i] *= fma(h, (double)wc[j][i], (double)bc[j][i]) > 0.0 ? 1.0f : slope;
        const double gw = (double)g[j][i] * (double)wc[j][i];
        m[0] += gw;
        m[1] = fma(gw, h, m[1]);
        if (AFFINE && live) {
          sb[j][i] += g[j][i];
          sw[j][i] = fmaf(g[j][i], (float)h, sw[j][i]);
        }
      }
    if (gx) {
      over_row<L, 2>(m, lds);
      if (live) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const int c = (j * L + t) * V;
          if (c >= C) break;
          Vec<T, V> u;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const double h = ((double)v[j][i] - mean) * rstd;
            u.v[i] = (T)(float)(rstd * ((double)g[j][i] * (double)wc[j][i] - m[0] * per_c - h * (m[1] * per_c)));
          }
          casmvs::elem::store<T, V>(gx + base + c, u);
        }
      }
    }
  }
  if (!AFFINE) return;
  float *out = partial + (size_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    if (G > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) red[(j * V + i) * BT + threadIdx.x] = kind ? sb[j][i] : sw[j][i];
      __syncthreads();
      for (int o = threadIdx.x; o < K * V * L; o += BT) {
        const int e = o / L, lane = o % L, c = (e / V * L + lane) * V + e % V;
        if (c < C) {
          double s = 0.0;
          for (int k = 0; k < G; ++k) s += (double)red[e * BT + k * L + lane];
          out[(size_t)kind * C + c] = (float)s;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < K; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = (j * L + t) * V + i;
          if (c < C) out[(size_t)kind * C + c] = kind ? sb[j][i] : sw[j][i];
        }
    }
  }
}

// grad_weight / grad_bias from the workgroups' partial sums (parts, 2 C), in their order: COLS columns and 1024 / COLS threads each
template <int COLS>
__global__ __launch_bounds__(1024) void ln_finish_parts_kernel(const float *__restrict__ partial, float *__restrict__ gw, float *__restrict__ gb, int parts, int C) {
  constexpr int J = 1024 / COLS;
  __shared__ double red[1024];
  const int col = threadIdx.x % COLS, j = threadIdx.x / COLS, i = blockIdx.x * COLS + col;
  double s = 0.0;
  if (i < 2 * C) {
    int k = j;
    for (; k + 3 * J < parts; k += 4 * J) {   // four loads in flight
      const float a0 = partial[(size_t)k * 2 * C + i], a1 = partial[(size_t)(k + J) * 2 * C + i];
      const float a2 = partial[(size_t)(k + 2 * J) * 2 * C + i], a3 = partial[(size_t)(k + 3 * J) * 2 * C + i];
      s += ((double)a0 + (double)a1) + ((double)a2 + (double)a3);
    }
    for (; k < parts; k += J) s += (double)partial[(size_t)k * 2 * C + i];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int st = J / 2; st > 0; st >>= 1) {
    if (j < st) red[threadIdx.x] += red[threadIdx.x + st * COLS];
    __syncthreads();
  }
  if (j == 0 && i < 2 * C) (i < C ? gw[i] : gb[i - C]) = (float)red[col];
}

// ---- any number of channels --------------------------------------------------------------------------------------------------------------------------
// ROWS (inner == 1): one workgroup per position, its threads along the channels.  Otherwise 64 consecutive positions per workgroup, four threads each.
// x is read once per use (three times forward, five backward): these forms serve the shapes that do not fit registers.
template <bool ROWS>
__device__ __forceinline__ double combine(double v, double *lds) {
  lds[threadIdx.x] = v;
  __syncthreads();
  double s;
  if (ROWS) {
    for (int st = kThreads / 2; st > 0; st >>= 1) {
      if ((int)threadIdx.x < st) lds[threadIdx.x] += lds[threadIdx.x + st];
      __syncthreads();
    }
    s = lds[0];
  } else {
    const int lane = threadIdx.x & 63;
    s = (lds[lane] + lds[lane + 64]) + (lds[lane + 128] + lds[lane + 192]);
  }
  __syncthreads();
  return s;
}

struct Place {   // this thread's position: the address of channel 0, the distance of two channels, first channel and step of its share
  size_t base, cs;
  int c0, step;
  size_t position;
  bool live;
};
template <bool ROWS>
__device__ __forceinline__ Place place_of(size_t outer, int C, size_t inner) {
  Place pl;
  if (ROWS) {
    pl.position = blockIdx.x;
    pl.live = true;
    pl.base = pl.position * (size_t)C;
    pl.cs = 1;
    pl.c0 = threadIdx.x;
    pl.step = kThreads;
  } else {
    pl.position = (size_t)blockIdx.x * 64 + (threadIdx.x & 63);
    pl.live = pl.position < outer * inner;
    const size_t n = pl.live ? pl.position / inner : 0, s = pl.live ? pl.position % inner : 0;
    pl.base = n * (size_t)C * inner + s;
    pl.cs = inner;
    pl.c0 = threadIdx.x >> 6;
    pl.step = kThreads / 64;
  }
  return pl;
}

template <class T, bool ROWS>
__device__ __forceinline__ void statistics(const T *__restrict__ x, const Place &pl, int C, float eps, double *lds, double &mean, double &rstd) {
  double s = 0.0;
  for (int c = pl.c0; c < C; c += pl.step) s += (double)(float)x[pl.base + c * pl.cs];
  mean = combine<ROWS>(s, lds) / C;
  s = 0.0;
  for (int c = pl.c0; c < C; c += pl.step) {
    const double d = (double)(float)x[pl.base + c * pl.cs] - mean;
    s += d * d;
  }
  rstd = 1.0 / sqrt(combine<ROWS>(s, lds) / C + (double)eps);
}

template <class T, bool ROWS>
__global__ __launch_bounds__(kThreads) void ln_forward_any_kernel(const T *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b,
                                                                 T *__restrict__ y, size_t outer, int C, size_t inner, float eps, float slope) {
  __shared__ double lds[kThreads];
  const Place pl = place_of<ROWS>(outer, C, inner);
  double mean, rstd;
  statistics<T, ROWS>(x, pl, C, eps, lds, mean, rstd);
  if (!pl.live) return;
  for (int c = pl.c0; c < C; c += pl.step) {
    const size_t at = pl.base + c * pl.cs;
    const double z = ((double)(float)x[at] - mean) * rstd * (w ? (double)w[c] : 1.0) + (b ? (double)b[c] : 0.0);
    y[at] = (T)(float)(z > 0.0 ? z : z * slope);
  }
}

// gx, and (mean, rstd) of every position for the weight gradient's kernel
template <class T, bool ROWS>
__global__ __launch_bounds__(kThreads) void ln_backward_any_kernel(const T *__restrict__ x, const T *__restrict__ gy, const float *__restrict__ w,
                                                                  const float *__restrict__ b, T *__restrict__ gx, double *__restrict__ stats,
                                                                  size_t outer, int C, size_t inner, float eps, float slope) {
  __shared__ double lds[kThreads];
  const Place pl = place_of<ROWS>(outer, C, inner);
  double mean, rstd;
  statistics<T, ROWS>(x, pl, C, eps, lds, mean, rstd);
  double s1 = 0.0, s2 = 0.0;
  for (int c = pl.c0; c < C; c += pl.step) {
    const size_t at = pl.base + c * pl.cs;
    const double h = ((double)(float)x[at] - mean) * rstd, wc = w ? (double)w[c] : 1.0;
    const double g = (double)(float)gy[at] * (h * wc + (b ? (double)b[c] : 0.0) > 0.0 ? 1.0 : (double)slope) * wc;
    s1 += g;
    s2 += g * h;
  }
  const double m1 = combine<ROWS>(s1, lds) / C, m2 = combine<ROWS>(s2, lds) / C;
  if (!pl.live) return;
  if (pl.c0 == 0) {
    stats[2 * pl.position] = mean;
    stats[2 * pl.position + 1] = rstd;
  }
  if (!gx) return;
  for (int c = pl.c0; c < C; c += pl.step) {
    const size_t at = pl.base + c * pl.cs;
    const double h = ((double)(float)x[at] - mean) * rstd, wc = w ? (double)w[c] : 1.0;
    const double g = (double)(float)gy[at] * (h * wc + (b ? (double)b[c] : 0.0) > 0.0 ? 1.0 : (double)slope) * wc;
    gx[at] = (T)(float)(rstd * (g - m1 - h * m2));
  }
}

// partial[slice][0 / 1][c] = sum of g h / of g over the slice's positions.  ROWS: 64 channels x 4 positions per workgroup, blockIdx.y = channel tile;
// otherwise one channel per workgroup, its threads along the positions.
template <class T, bool ROWS>
__global__ __launch_bounds__(kThreads) void ln_wgrad_any_kernel(const T *__restrict__ x, const T *__restrict__ gy, const float *__restrict__ w,
                                                               const float *__restrict__ b, const double *__restrict__ stats, double *__restrict__ partial,
                                                               size_t outer, int C, size_t inner, float slope) {
  __shared__ double lds[2][kThreads];
  const size_t positions = outer * inner, per = (positions + gridDim.x - 1) / gridDim.x;
  const size_t lo = blockIdx.x * per, hi = lo + per < positions ? lo + per : positions;
  const int c = ROWS ? (int)blockIdx.y * 64 + (int)(threadIdx.x & 63) : (int)blockIdx.y;
  double s0 = 0.0, s1 = 0.0;
  if (c < C) {
    const double wc = w ? (double)w[c] : 1.0, bc = b ? (double)b[c] : 0.0;
    for (size_t p = lo + (ROWS ? threadIdx.x >> 6 : threadIdx.x); p < hi; p += ROWS ? kThreads / 64 : kThreads) {
      const size_t at = ROWS ? p * (size_t)C + c : (p / inner * (size_t)C + c) * inner + p % inner;
      const double h = ((double)(float)x[at] - stats[2 * p]) * stats[2 * p + 1];
      const double g = (double)(float)gy[at] * (h * wc + bc > 0.0 ? 1.0 : (double)slope);
      s0 += g * h;
      s1 += g;
    }
  }
  lds[0][threadIdx.x] = s0;
  lds[1][threadIdx.x] = s1;
  __syncthreads();
  for (int st = kThreads / 2; st >= (ROWS ? 64 : 1); st >>= 1) {
    if ((int)threadIdx.x < st) {
      lds[0][threadIdx.x] += lds[0][threadIdx.x + st];
      lds[1][threadIdx.x] += lds[1][threadIdx.x + st];
    }
    __syncthreads();
  }
  if ((int)threadIdx.x < (ROWS ? 64 : 1) && c < C) {
    partial[((size_t)blockIdx.x * 2) * C + c] = lds[0][threadIdx.x];
    partial[((size_t)blockIdx.x * 2 + 1) * C + c] = lds[1][threadIdx.x];
  }
}

// grad_weight / grad_bias from the slices' partial sums, in their order
__global__ __launch_bounds__(kThreads) void ln_finish_kernel(const double *__restrict__ partial, float *__restrict__ gw, float *__restrict__ gb, int slices, int C) {
  const int i = blockIdx.x * kThreads + threadIdx.x;   // (kind, channel)
  if (i >= 2 * C) return;
  double s = 0.0;
  for (int k = 0; k < slices; ++k) s += partial[(size_t)k * 2 * C + i];
  (i < C ? gw[i] : gb[i - C]) = (float)s;
}

// ---- host ----------------------------------------------------------------------------------------------------------------------------------------------------
int slices_of(size_t positions) {
  const size_t n = (positions + kSlicePositions - 1) / kSlicePositions;
  return (int)(n < 1 ? 1 : n > kMostSlices ? kMostSlices : n);
}

// Which form a shape takes.  The vector width does not enter the sizes that the workspace is computed from: alignment is a pointer's, a workspace is a shape's.
enum Form { kAny, kPlanes, kRows };
Form form_of(int C, size_t inner) { return inner == 1 ? (C <= 8192 ? kRows : kAny) : (C <= 64 * kHeld ? kPlanes : kAny); }

// workgroups of the fused backward pass = rows of its partial sums: two per CU keep the memory busy (every thread has 16 loads in flight), and the finishing
// kernel reads few of them
constexpr size_t kBackwardBlocks = 512;

bool fits(const void *p, size_t bytes) { return p == nullptr || ((uintptr_t)p & (bytes - 1)) == 0; }

int check_sizes(const char *what, int dtype, size_t outer, int C, size_t inner) {
  CASMVS_REQUIRE(casmvs::elem::known(dtype), "%s: dtype %d", what, dtype);
  CASMVS_REQUIRE(C > 0 && C <= 65535, "%s: C=%d (1 .. 65535)", what, C);
  // (launches are at least one workgroup per row / per 64 positions)
  CASMVS_REQUIRE(inner == 0 || outer <= ((size_t)1 << 36) / inner, "%s: %zu x %zu positions", what, outer, inner);
  CASMVS_REQUIRE(inner != 1 || outer < ((size_t)1 << 31), "%s: %zu rows", what, outer);
  return CASMVS_OK;
}

struct Call {   // arguments of either direction
  const void *x, *gy;
  const float *w, *b;
  void *out;        // y, or gx (may be null)
  float *partial;   // null: no weight gradient
  float *gw, *gb;   // where it goes
  size_t outer, inner;
  int C;
  float eps, slope;
  hipStream_t stream;
  size_t positions() const { return outer * inner; }
  // One workgroup's sums are the gradients themselves, where grad_bias lies behind grad_weight: nothing is left to add up (parts = 0)
  float *sums(int &parts) const {
    if (!partial || parts != 1 || gb != gw + C) return partial;
    parts = 0;
    return gw;
  }
};

template <class T, int CG, int V>
void planes(const Call &a, int &parts) {
  const size_t tile = (size_t)(kThreads / CG) * V, tiles = (a.positions() + tile - 1) / tile;
  if (!a.gy) {
    hipLaunchKernelGGL((ln_forward_planes_kernel<T, CG, V>), dim3((unsigned)tiles), dim3(kThreads), 0, a.stream, (const T *)a.x, a.w, a.b, (T *)a.out, a.positions(), a.C,
                       a.inner, 1.0 / a.C, a.eps, a.slope);
    return;
  }
  const unsigned grid = (unsigned)(tiles < kBackwardBlocks ? tiles : kBackwardBlocks);
  parts = (int)grid;
  float *sums = a.sums(parts);
  auto kernel = a.partial ? ln_backward_planes_kernel<T, CG, V, true> : ln_backward_planes_kernel<T, CG, V, false>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, a.stream, (const T *)a.x, (const T *)a.gy, a.w, a.b, (T *)a.out, sums, a.positions(), tiles,
                     a.C, a.inner, 1.0 / a.C, a.eps, a.slope);
}
template <class T, int V>
void planes_by_groups(const Call &a, int &parts) {
  const int groups = (a.C + kHeld - 1) / kHeld;
  if (groups <= 1) planes<T, 1, V>(a, parts);
  else if (groups <= 2) planes<T, 2, V>(a, parts);
  else if (groups <= 4) planes<T, 4, V>(a, parts);
  else if (groups <= 8) planes<T, 8, V>(a, parts);
  else if (groups <= 16) planes<T, 16, V>(a, parts);
  else planes<T, 64, V>(a, parts);
}

template <class T, int L, int V, int K>
void rows(const Call &a, int &parts) {
  constexpr int threads = row_threads<L>();
  const size_t blocks = (a.outer + threads / L - 1) / (threads / L);
  if (!a.gy) {
    hipLaunchKernelGGL((ln_forward_rows_kernel<T, L, V, K>), dim3((unsigned)blocks), dim3(threads), 0, a.stream, (const T *)a.x, a.w, a.b, (T *)a.out, a.outer, a.C,
                       1.0 / a.C, a.eps, a.slope);
    return;
  }
  const unsigned grid = (unsigned)(blocks < kBackwardBlocks ? blocks : kBackwardBlocks);
  parts = (int)grid;
  float *sums = a.sums(parts);
  auto kernel = a.partial ? ln_backward_rows_kernel<T, L, V, K, true> : ln_backward_rows_kernel<T, L, V, K, false>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, a.stream, (const T *)a.x, (const T *)a.gy, a.w, a.b, (T *)a.out, sums, a.outer, a.C,
                     1.0 / a.C, a.eps, a.slope);
}
template <class T, int V>
void rows_by_width(const Call &a, int &parts) {
  const int vectors = (a.C + V - 1) / V;
  constexpr int k16 = 16 / V;   // 16 channels per lane
  if (vectors <= 4) rows<T, 4, V, 1>(a, parts);
  else if (vectors <= 8) rows<T, 8, V, 1>(a, parts);
  else if (vectors <= 16) rows<T, 16, V, 1>(a, parts);
  else if (vectors <= 64) rows<T, 64, V, 1>(a, parts);
  else if (vectors <= 128) rows<T, 64, V, 2>(a, parts);
  else if (vectors <= 256) rows<T, 64, V, 4>(a, parts);
  else if (a.C <= 64 * 16) rows<T, 64, V, k16>(a, parts);
  else if (a.C <= 256 * 16) rows<T, 256, V, k16>(a, parts);
  else rows<T, 512, V, k16>(a, parts);
}

// Either direction in the planes / rows form; `parts`: rows of partial sums that the backward pass wrote and are still to be added up.
void run_form(Form form, int dtype, const Call &a, int &parts) {
  CASMVS_WITH_DTYPE(dtype, {
    // four elements at a time where rows / planes keep their alignment
    const size_t bytes = 4 * sizeof(T);
    const bool wide = (form == kRows ? a.C : a.inner) % 4 == 0 && fits(a.x, bytes) && fits(a.gy, bytes) && fits(a.out, bytes);
    if (form == kPlanes) {
      if (wide) planes_by_groups<T, 4>(a, parts); else planes_by_groups<T, 1>(a, parts);
    } else {
      if (wide) rows_by_width<T, 4>(a, parts); else rows_by_width<T, 1>(a, parts);
    }
  });
}
}  // namespace

extern "C" int casmvs_layer_norm_forward(const void *x, const float *weight, const float *bias, void *y, int dtype, size_t outer, int C, size_t inner,
                                         float eps, float slope, void *stream) {
  casmvs::clear_error();
  if (int rc = check_sizes("layer_norm_forward", dtype, outer, C, inner)) return rc;
  if (outer == 0 || inner == 0) return CASMVS_OK;
  CASMVS_REQUIRE(x && y, "layer_norm_forward: null pointer");
  const Form form = form_of(C, inner);
  hipStream_t st = (hipStream_t)stream;
  if (form != kAny) {
    int parts = 0;
    run_form(form, dtype, Call{x, nullptr, weight, bias, y, nullptr, nullptr, nullptr, outer, inner, C, eps, slope, st}, parts);
    return casmvs::check_launch("layer_norm_forward");
  }
  const size_t positions = outer * inner;
  CASMVS_WITH_DTYPE(dtype, {
    if (inner == 1)
      hipLaunchKernelGGL((ln_forward_any_kernel<T, true>), dim3((unsigned)positions), dim3(kThreads), 0, st, (const T *)x, weight, bias, (T *)y, outer, C, inner, eps, slope);
    else
      hipLaunchKernelGGL((ln_forward_any_kernel<T, false>), dim3((unsigned)((positions + 63) / 64)), dim3(kThreads), 0, st, (const T *)x, weight, bias, (T *)y, outer, C, inner, eps, slope);
  });
  return casmvs::check_launch("ln_forward_any_kernel");
}

extern "C" size_t casmvs_layer_norm_backward_workspace_bytes(int dtype, size_t outer, int C, size_t inner) {
  if (!casmvs::elem::known(dtype) || C <= 0) return 0;
  const size_t positions = outer * inner;
  if (form_of(C, inner) != kAny) return (positions < kBackwardBlocks ? positions : kBackwardBlocks) * 2 * C * sizeof(float) + 16;
  return positions * 16 + (size_t)slices_of(positions) * 2 * C * 8 + 16;
}

extern "C" int casmvs_layer_norm_backward(const void *x, const void *grad_y, const float *weight, const float *bias, void *grad_x, float *grad_weight,
                                          float *grad_bias, void *workspace, int dtype, size_t outer, int C, size_t inner, float eps, float slope,
                                          void *stream) {
  casmvs::clear_error();
  if (int rc = check_sizes("layer_norm_backward", dtype, outer, C, inner)) return rc;
  CASMVS_REQUIRE((grad_weight == nullptr) == (grad_bias == nullptr), "layer_norm_backward: grad_weight and grad_bias go together");
  CASMVS_REQUIRE(workspace && fits(workspace, 8), "layer_norm_backward: workspace (8-byte aligned)");
  const size_t positions = outer * inner;
  CASMVS_REQUIRE(!positions || (x && grad_y), "layer_norm_backward: null pointer");
  hipStream_t st = (hipStream_t)stream;
  const Form form = form_of(C, inner);
  if (form != kAny || !positions) {
    int parts = 0;
    if (positions) run_form(form, dtype, Call{x, grad_y, weight, bias, grad_x, grad_weight ? (float *)workspace : nullptr, grad_weight, grad_bias, outer, inner, C, eps, slope, st}, parts);
    if (grad_weight && (parts || !positions)) {
      if (C <= 32)
        hipLaunchKernelGGL(ln_finish_parts_kernel<16>, dim3((unsigned)((2 * C + 15) / 16)), dim3(1024), 0, st, (const float *)workspace, grad_weight, grad_bias, parts, C);
      else
        hipLaunchKernelGGL(ln_finish_parts_kernel<64>, dim3((unsigned)((2 * C + 63) / 64)), dim3(1024), 0, st, (const float *)workspace, grad_weight, grad_bias, parts, C);
    }
    return casmvs::check_launch("layer_norm_backward");
  }
  double *stats = (double *)workspace, *partial = stats + 2 * positions;
  const int slices = slices_of(positions);
  CASMVS_WITH_DTYPE(dtype, {
    const T *xp = (const T *)x, *gp = (const T *)grad_y;
    if (inner == 1) {
      hipLaunchKernelGGL((ln_backward_any_kernel<T, true>), dim3((unsigned)positions), dim3(kThreads), 0, st, xp, gp, weight, bias, (T *)grad_x, stats, outer, C, inner, eps, slope);
      if (grad_weight)
        hipLaunchKernelGGL((ln_wgrad_any_kernel<T, true>), dim3(slices, (unsigned)((C + 63) / 64)), dim3(kThreads), 0, st, xp, gp, weight, bias, stats, partial, outer, C, inner, slope);
    } else {
      hipLaunchKernelGGL((ln_backward_any_kernel<T, false>), dim3((unsigned)((positions + 63) / 64)), dim3(kThreads), 0, st, xp, gp, weight, bias, (T *)grad_x, stats, outer, C, inner, eps, slope);
      if (grad_weight)
        hipLaunchKernelGGL((ln_wgrad_any_kernel<T, false>), dim3(slices, (unsigned)C), dim3(kThreads), 0, st, xp, gp, weight, bias, stats, partial, outer, C, inner, slope);
    }
  });
  if (grad_weight)
    hipLaunchKernelGGL(ln_finish_kernel, dim3((unsigned)((2 * (size_t)C + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, partial, grad_weight, grad_bias, slices, C);
  return casmvs::check_launch("layer_norm_backward");
}
