// Layer norm over the channel axis + leaky ReLU, forward and backward.
//
//   position p of (outer, C, inner), channels c:   mu = mean_c x,  v = mean_c (x - mu)^2,  r = 1 / sqrt(v + eps),  h = (x - mu) r
//   z = h w_c + b_c,   y = z > 0 ? z : slope z
//   g = gy (z > 0 ? 1 : slope),  m1 = mean_c (g w),  m2 = mean_c (g w h):   gx = r (g w - m1 - h m2),  gw_c = sum_p g h,  gb_c = sum_p g
//
// The backward pass takes x and recomputes mu, r and the side of zero that z lies on: x has to be read for h anyway, and two stored floats per position
// would be a quarter of the traffic at 8 channels.
//
// What is 64 bits wide: the statistics and x - mu (a row far from zero keeps its spread), and the side of zero of a z that float32 cannot tell - an element
// within its rounding of zero would otherwise get the slope in one computation and 1 in another, an error of the size of the gradient itself.  Those are
// found by |z| <= 2^-18 |b| (near zero h w is about -b, and the float32 z is off by at most 4 * 2^-24 of it) and decided again from x; they are one in 10^5.
// Everything else is float32 from the rounded x - mu on, but at fewer than 8 channels (FEW), where gx is what is left after cancellation: all 64 bits there.
//
// Three forms, by where a position's channels lie and how many there are:
//   planes  (inner > 1, C <= 512)   a thread holds 8 channels of 2 (or 1) consecutive positions in registers, up to 64 threads share a position;
//   rows    (inner = 1, C <= 8192)  up to 64 lanes of a wave, or a workgroup, hold a row in registers;
//   any     everything else: x is read once per use.
//
// Planes and rows touch each element once and wait for memory: 8 bytes per float32 element forward, 12 backward (a copy of gigabytes reaches 4.7 to 5.1 TB/s, one
// that the caches hold more).  Float32, forward / backward with the weight gradients, the launches and the sums' second kernel included:
//   2 x 8 x 32 x 256 x 320   60 us (5.6 TB/s) / 99 us (5.1 TB/s)      6 x 8 x 512 x 640   20 us (6.4) / 35 us (5.3)      6 x 16 x 256 x 320   11 / 25 us
//   983040 rows of 32        45 us (5.6)      / 71 us (5.3)           8192 rows of 1024   14 us (4.9) / 27 us (3.7)
// and in bf16: 2 x 8 x 32 x 256 x 320   40 us (4.2) / 49 us (5.1)     8191 rows of 1000   11 us (3.0) / 24 us (2.1)     65536 rows of 1024   68 us (3.9) / 93 us (4.3).
// Small tensors cost their launches: 2 x 64 x 6 x 16 x 20 9 / 17 us.
// Maps of more channels, 67 MB, us forward / backward (a copy of them takes 27, the bytes of the backward pass 40):
//   channels   64         96         128        192         256         384         512         520 (any)
//   float32    24 / 50    25 / 56    24 / 52    58 / 142    59 / 122    62 / 120    61 / 109    134 / 296
//   bf16       38 / 66    47 / 95    42 / 79    157 / 492   143 / 379   133 / 272   127 / 231   147 / 348
// From 129 channels on 64 groups leave a tile 4 x V positions: a wave's loads are runs of 8 (32 bytes in float32, 16 in bf16), and below 256
// channels more than half of what a thread could hold is missing.  In bf16 that form's backward pass is no faster than the any form's there.
#include "elem_types.h"

namespace {
using casmvs::elem::Floats;
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

// What a thread loads of a tile, as loaded; 0 for a channel or position that is not there
template <class T, int V>
struct PlaneLoads {
  Vec<T, V> t[kHeld];
  template <bool FULL>
  __device__ __forceinline__ void load(const T *__restrict__ x, size_t base, size_t inner, int first, int step, int C, bool live) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int c = first + r * step;
      if (live && (FULL || c < C)) {
        t[r] = casmvs::elem::load<T, V>(x + base + c * inner);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) t[r].v[i] = (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ void widen(float (&v)[kHeld][V]) const {
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
#pragma unroll
      for (int i = 0; i < V; ++i) v[r][i] = (float)t[r].v[i];
  }
};

// mean and 1 / sqrt(var + eps) of the thread's positions; CENTRE: v becomes x - mean
template <int MOST, bool CENTRE, bool FULL, int CG, int V>
__device__ __forceinline__ void plane_statistics(const PlaneTile<CG, V> &tile, float (&v)[kHeld][V], int C, double per_c, float eps, double *lds, double (&mean)[V],
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
    if (FULL || tile.cg + r * CG < C) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double d = (double)v[r][i] - mean[i];
        s[0][i] = fma(d, d, s[0][i]);
        if (CENTRE) v[r][i] = (float)d;
      }
    }
  tile.template over_groups<1, MOST>(s, lds);
#pragma unroll
  for (int i = 0; i < V; ++i) rstd[i] = inverse_sqrt(s[0][i] * per_c + (double)eps);
}

// A float32 z of magnitude up to this cannot tell its side of zero.  slope 1: the side does not matter.
__device__ __forceinline__ float near_zero(float bias, float slope) { return slope == 1.0f ? -1.0f : 0x1p-18f * fabsf(bias); }
__device__ __forceinline__ double z_of(float x, double mean, double rstd, float w, float b) { return fma(((double)x - mean) * rstd, (double)w, (double)b); }

// The thread's weights: kept over its tiles; 1 and 0 for what is missing
template <int CG>
struct PlaneWeights {
  float w[kHeld], b[kHeld];
  __device__ __forceinline__ PlaneWeights(const float *__restrict__ wp, const float *__restrict__ bp, int cg, int C) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int c = cg + r * CG < C ? cg + r * CG : C - 1;
      w[r] = wp ? wp[c] : 1.0f;
      b[r] = bp ? bp[c] : 0.0f;
    }
  }
};

// The forward pass in 16-bit types goes over several tiles per workgroup, the next one's loads ahead: 2 x 8 x 32 x 256 x 320 in bf16 50 -> 40 us.  In float32, with
// twice the bytes per tile in flight, one tile per workgroup is faster: 61 and 63 us, 6 x 16 x 256 x 320 11.4 and 13.5.
template <class T>
constexpr bool loops() { return sizeof(T) == 2; }
constexpr size_t kForwardBlocks = 1024;

// PAST: y goes past the caches
template <class T, int CG, int V, bool FEW, bool PAST>
__global__ __launch_bounds__(kThreads) void ln_forward_planes_kernel(const T *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b,
                                                                    T *__restrict__ y, size_t first, size_t positions, size_t tiles, int C, size_t inner,
                                                                    double per_c, float eps, float slope) {
  __shared__ double lds[plane_lds<CG, V>(1)];
  const PlaneTile<CG, V> tile;
  const PlaneWeights<CG> a(w, b, tile.cg, C);
  PlaneLoads<T, V> xs;
  size_t base_ahead;
  bool live_ahead;
  auto load_ahead = [&](size_t k) {
    const size_t p = (k * PlaneTile<CG, V>::PL + tile.pl) * V;
    live_ahead = p < positions;   // (V divides inner: all V positions or none, in one plane)
    size_t n, at;
    casmvs::elem::divide(live_ahead ? p : 0, inner, n, at);
    base_ahead = n * C * inner + at;
    xs.template load<false>(x, base_ahead, inner, tile.cg, CG, C, live_ahead);
  };
  load_ahead(first + blockIdx.x);
  for (size_t k = first + blockIdx.x; k < tiles; k += gridDim.x) {
    const size_t base = base_ahead;
    const bool live = live_ahead;
    float v[kHeld][V];
    xs.widen(v);
    if (loops<T>() && k + gridDim.x < tiles) load_ahead(k + gridDim.x);
    double mean[V], rstd[V];
    plane_statistics<1, !FEW, false, CG, V>(tile, v, C, per_c, eps, lds, mean, rstd);
    if (live) {
#pragma unroll
      for (int r = 0; r < kHeld; ++r) {
        const int c = tile.cg + r * CG;
        if (c >= C) break;
        Vec<T, V> t;
        bool near = FEW;   // (a channel's store leaves as soon as its z are known: one test for all of them holds every store back, 62 -> 70 us at 2 x 8 x 32 x 256 x 320)
        if (!FEW) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float z = v[r][i] * (float)rstd[i] * a.w[r] + a.b[r];
            near |= fabsf(z) <= near_zero(a.b[r], slope);
            t.v[i] = (T)(z > 0.0f ? z : z * slope);
          }
        }
        if (near) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const double z = z_of(FEW ? v[r][i] : (float)x[base + c * inner + i], mean[i], rstd[i], a.w[r], a.b[r]);
            t.v[i] = (T)(float)(z > 0.0 ? z : z * slope);
          }
        }
        if (PAST) casmvs::elem::store_past<T, V>(y + base + c * inner, t);
        else casmvs::elem::store<T, V>(y + base + c * inner, t);
      }
    }
    if (!loops<T>()) break;
  }
}

// How the backward pass counts its channels: fewer than 8 (all in 64 bits), any number, or exactly 8 per group (no test at a channel).  The forward pass has no
// form of the last kind: without the tests the compiler holds every channel's values at once, 88 registers instead of 56, and the pass is 15 % slower.
enum Channels { kFew, kSome, kFull };

// gx, and of every workgroup the sums over its tiles of g h and g per channel: partial[workgroup][0 / 1][c].  AFFINE: the weight gradient is wanted.  PAST: gx goes
// past the caches.
template <class T, int CG, int V, bool AFFINE, Channels CH, bool PAST>
__global__ __launch_bounds__(kThreads) void ln_backward_planes_kernel(const T *__restrict__ x, const T *__restrict__ gy, const float *__restrict__ w,
                                                                     const float *__restrict__ b, T *__restrict__ gx, float *__restrict__ partial,
                                                                     size_t positions, size_t tiles, int C, size_t inner, double per_c, float eps, float slope) {
  using Tile = PlaneTile<CG, V>;
  constexpr bool FEW = CH == kFew, FULL = CH == kFull;
  constexpr int kSums = plane_lds<CG, V>(2) > 2 * kHeld * kThreads / 2 ? plane_lds<CG, V>(2) : 2 * kHeld * kThreads / 2;
  __shared__ double lds[kSums];   // (the groups' sums; at the end 2 * kHeld * 256 floats)
  const Tile tile;
  const PlaneWeights<CG> a(w, b, tile.cg, C);
  float sw[kHeld], sb[kHeld];   // this thread's share of sum g h and sum g: positions / (workgroups * PL) values each
#pragma unroll
  for (int r = 0; r < kHeld; ++r) sw[r] = sb[r] = 0.0f;
  // The next tile's loads are issued before this one is worked on: with two waves per SIMD three quarters of the time went by waiting for them
  PlaneLoads<T, V> xs, gs;
  size_t base_ahead;
  bool live_ahead;
  auto load_ahead = [&](size_t k) {
    const size_t p = (k * Tile::PL + tile.pl) * V;
    live_ahead = k < tiles && p < positions;
    size_t n, at;
    casmvs::elem::divide(live_ahead ? p : 0, inner, n, at);
    base_ahead = n * C * inner + at;
    xs.template load<FULL>(x, base_ahead, inner, tile.cg, CG, C, live_ahead);
    gs.template load<FULL>(gy, base_ahead, inner, tile.cg, CG, C, live_ahead);
  };
  load_ahead(blockIdx.x);
  for (size_t k = blockIdx.x; k < tiles; k += gridDim.x) {
    const size_t base = base_ahead;
    const bool live = live_ahead;
    float v[kHeld][V], g[kHeld][V];
    xs.widen(v);
    gs.widen(g);
    if (k + gridDim.x < tiles) load_ahead(k + gridDim.x);
    double mean[V], rstd[V], m[2][V];
    plane_statistics<2, !FEW, FULL, CG, V>(tile, v, C, per_c, eps, lds, mean, rstd);
    // A thread without a position holds zeros, and eps = 0 leaves it 1 / sqrt(0): its h has to stay 0 for the sums over positions
#pragma unroll
    for (int i = 0; i < V; ++i) rstd[i] = live ? rstd[i] : 0.0;
    if (FEW) {
#pragma unroll
      for (int i = 0; i < V; ++i) m[0][i] = m[1][i] = 0.0;
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const double h = ((double)v[r][i] - mean[i]) * rstd[i];
          g[r][i] *= fma(h, (double)a.w[r], (double)a.b[r]) > 0.0 ? 1.0f : slope;
          const double gw = (double)g[r][i] * (double)a.w[r];
          m[0][i] += gw;
          m[1][i] = fma(gw, h, m[1][i]);
          if (AFFINE) {
            sw[r] = fmaf(g[r][i], (float)h, sw[r]);
            sb[r] += g[r][i];
          }
        }
    } else {
      bool near = false;
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[r][i] *= (float)rstd[i];   // h from here on
          const float z = v[r][i] * a.w[r] + a.b[r];
          near |= fabsf(z) <= near_zero(a.b[r], slope);
          g[r][i] *= z > 0.0f ? 1.0f : slope;
        }
      if (near && live) {
#pragma unroll
        for (int r = 0; r < kHeld; ++r) {
          const int c = tile.cg + r * CG;
          if (FULL || c < C) {
#pragma unroll
            for (int i = 0; i < V; ++i)
              g[r][i] = (float)gy[base + c * inner + i] * (z_of((float)x[base + c * inner + i], mean[i], rstd[i], a.w[r], a.b[r]) > 0.0 ? 1.0f : slope);
          }
        }
      }
      float f[2][V];   // sum g w and sum g w h over this thread's 8 channels; in 64 bits over the groups
#pragma unroll
      for (int i = 0; i < V; ++i) f[0][i] = f[1][i] = 0.0f;
#pragma unroll
      for (int r = 0; r < kHeld; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float gw = g[r][i] * a.w[r];
          f[0][i] += gw;
          f[1][i] = fmaf(gw, v[r][i], f[1][i]);
          if (AFFINE) {
            sw[r] = fmaf(g[r][i], v[r][i], sw[r]);
            sb[r] += g[r][i];
          }
        }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        m[0][i] = f[0][i];
        m[1][i] = f[1][i];
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
          if (!FULL && c >= C) break;
          Vec<T, V> t;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (FEW) {
              const double h = ((double)v[r][i] - mean[i]) * rstd[i];
              t.v[i] = (T)(float)(rstd[i] * ((double)g[r][i] * (double)a.w[r] - m[0][i] - h * m[1][i]));
            } else {
              t.v[i] = (T)((float)rstd[i] * (g[r][i] * a.w[r] - (float)m[0][i] - v[r][i] * (float)m[1][i]));
            }
          }
          if (PAST) casmvs::elem::store_past<T, V>(gx + base + c * inner, t);
          else casmvs::elem::store<T, V>(gx + base + c * inner, t);
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
    constexpr int W = L / 64, waves = row_threads<L>() / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;   // the row's first wave
    __syncthreads();   // (lds may still be read from the last use)
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) lds[k * waves + wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = lds[k * waves + first];
#pragma unroll
      for (int i = 1; i < W; ++i) v[k] += lds[k * waves + first + i];
    }
  }
}

// A lane's part of a row, as loaded; 0 for a channel or row that is not there
template <class T, int L, int V, int K>
struct RowLoads {
  Vec<T, V> t[K];
  __device__ __forceinline__ void load(const T *__restrict__ x, size_t base, int lane, int C, bool live) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int c = (j * L + lane) * V;
      if (live && c < C) {
        t[j] = casmvs::elem::load<T, V>(x + base + c);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) t[j].v[i] = (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ void widen(float (&v)[K][V]) const {
#pragma unroll
    for (int j = 0; j < K; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = (float)t[j].v[i];
  }
};

// (as plane_statistics)
template <int L, int V, int K, bool CENTRE>
__device__ __forceinline__ void row_statistics(float (&v)[K][V], int t, int C, double per_c, float eps, double *lds, double &mean, double &rstd) {
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
        if (CENTRE) v[j][i] = (float)d;
      }
    }
  over_row<L, 1>(s, lds);
  rstd = inverse_sqrt(s[0] * per_c + (double)eps);
}

template <class T, int L, int V, int K, bool FEW>
__global__ __launch_bounds__(row_threads<L>()) void ln_forward_rows_kernel(const T *__restrict__ x, const float *__restrict__ w, const float *__restrict__ b, T *__restrict__ y,
                                                                          size_t first, size_t rows, int C, double per_c, float eps, float slope) {
  __shared__ double lds[row_threads<L>() / 64];
  const int t = threadIdx.x % L;
  const size_t row = (first + blockIdx.x) * (row_threads<L>() / L) + threadIdx.x / L;
  const bool live = row < rows;
  const size_t base = live ? row * C : 0;
  RowLoads<T, L, V, K> xs;
  xs.load(x, base, t, C, live);
  float v[K][V];
  xs.widen(v);
  double mean, rstd;
  row_statistics<L, V, K, !FEW>(v, t, C, per_c, eps, lds, mean, rstd);
  if (!live) return;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const int c = (j * L + t) * V;
    if (c >= C) break;
    Floats<V> wc, bc;   // (V divides C)
    if (w) wc = *reinterpret_cast<const Floats<V> *>(w + c);
    if (b) bc = *reinterpret_cast<const Floats<V> *>(b + c);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!w) wc.v[i] = 1.0f;
      if (!b) bc.v[i] = 0.0f;
    }
    Vec<T, V> u;
    bool near = FEW;
    if (!FEW) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float z = v[j][i] * (float)rstd * wc.v[i] + bc.v[i];
        near |= fabsf(z) <= near_zero(bc.v[i], slope);
        u.v[i] = (T)(z > 0.0f ? z : z * slope);
      }
    }
    if (near) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double z = z_of(FEW ? v[j][i] : (float)x[base + c + i], mean, rstd, wc.v[i], bc.v[i]);
        u.v[i] = (T)(float)(z > 0.0 ? z : z * slope);
      }
    }
    casmvs::elem::store<T, V>(y + base + c, u);
  }
}

// gx, and of every workgroup the sums over its rows of g h and g: a thread keeps its channels for all of them.  partial[workgroup][0 / 1][c].
template <class T, int L, int V, int K, bool AFFINE, bool FEW>
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
  // The next turn's loads are issued before this one is worked on: bf16 65536 x 1024 202 -> 93 us, 8191 x 1000 30 -> 24 (float32: no difference at 8192 x 1024)
  RowLoads<T, L, V, K> xs, gs;
  size_t base_ahead;
  bool live_ahead;
  auto load_ahead = [&](size_t turn) {
    const size_t row = (turn * gridDim.x + blockIdx.x) * G + threadIdx.x / L;
    live_ahead = row < rows;
    base_ahead = live_ahead ? row * C : 0;
    xs.load(x, base_ahead, t, C, live_ahead);
    gs.load(gy, base_ahead, t, C, live_ahead);   // (g of a missing channel or row is 0)
  };
  load_ahead(0);
  for (size_t turn = 0; turn < turns; ++turn) {
    const size_t base = base_ahead;
    const bool live = live_ahead;
    float v[K][V], g[K][V];
    xs.widen(v);
    gs.widen(g);
    if (turn + 1 < turns) load_ahead(turn + 1);
    double mean, rstd, m[2] = {0.0, 0.0};
    row_statistics<L, V, K, !FEW>(v, t, C, per_c, eps, lds, mean, rstd);
    const float r32 = (float)rstd;
    float f0 = 0.0f, f1 = 0.0f;   // sum g w and sum g w h over this thread's channels; in 64 bits over the row
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (FEW) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const double h = ((double)v[j][i] - mean) * rstd;
          g[j][i] *= fma(h, (double)wc[j][i], (double)bc[j][i]) > 0.0 ? 1.0f : slope;
          const double gw = (double)g[j][i] * (double)wc[j][i];
          m[0] += gw;
          m[1] = fma(gw, h, m[1]);
          if (AFFINE && live) sw[j][i] = fmaf(g[j][i], (float)h, sw[j][i]);
        }
      } else {
        bool near = false;
        float factor[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[j][i] *= r32;   // h from here on
          const float z = v[j][i] * wc[j][i] + bc[j][i];
          near |= fabsf(z) <= near_zero(bc[j][i], slope);
          factor[i] = z > 0.0f ? 1.0f : slope;
        }
        const int c = (j * L + t) * V;
        if (near && live && c < C) {
#pragma unroll
          for (int i = 0; i < V; ++i) factor[i] = z_of((float)x[base + c + i], mean, rstd, wc[j][i], bc[j][i]) > 0.0 ? 1.0f : slope;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[j][i] *= factor[i];
          const float gw = g[j][i] * wc[j][i];
          f0 += gw;
          f1 = fmaf(gw, v[j][i], f1);
          if (AFFINE && live) sw[j][i] = fmaf(g[j][i], v[j][i], sw[j][i]);
        }
      }
      if (AFFINE && live) {
#pragma unroll
        for (int i = 0; i < V; ++i) sb[j][i] += g[j][i];
      }
    }
    if (gx) {
      if (!FEW) {
        m[0] = f0;
        m[1] = f1;
      }
      over_row<L, 2>(m, lds);
      const float m0 = (float)(m[0] * per_c), m1 = (float)(m[1] * per_c);
      if (live) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const int c = (j * L + t) * V;
          if (c >= C) break;
          Vec<T, V> u;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (FEW) {
              const double h = ((double)v[j][i] - mean) * rstd;
              u.v[i] = (T)(float)(rstd * ((double)g[j][i] * (double)wc[j][i] - m[0] * per_c - h * (m[1] * per_c)));
            } else {
              u.v[i] = (T)(r32 * (g[j][i] * wc[j][i] - m0 - v[j][i] * m1));
            }
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

// Workgroups of the fused backward pass = rows of its partial sums.  Three per CU are resident (registers) and keep the memory busiest: bf16 2 x 8 x 32 x 256 x 320
// 49 us with 768, 54 with 512, 57 with 1024.  Past 256 channels a row of sums is as long as a row of data and there are few rows: bf16 8191 x 1000 24 us with
// 512, 30 with 768 (65536 x 1024 93 and 111; but 983040 x 32 in float32 83 and 72), and past 2048 the same again: bf16 1000 x 4096 23 us with 256, 30 with 512
// (2000 x 2048 in float32 28 and 24).
size_t backward_blocks(int C) { return C > 2048 ? 256 : C > 256 ? 512 : 768; }

// A launch has fewer than 2^32 threads: a larger forward pass (more than 2^31 elements and up) goes in several
constexpr size_t kLaunchBlocks = (size_t)1 << 22;
unsigned launch_blocks(size_t left) { return (unsigned)(left < kLaunchBlocks ? left : kLaunchBlocks); }

bool fits(const void *p, size_t bytes) { return p == nullptr || ((uintptr_t)p & (bytes - 1)) == 0; }

int check_sizes(const char *what, int dtype, size_t outer, int C, size_t inner) {
  CASMVS_REQUIRE(casmvs::elem::known(dtype), "%s: dtype %d", what, dtype);
  CASMVS_REQUIRE(C > 0 && C <= 65535, "%s: C=%d (1 .. 65535)", what, C);
  // rows / planes: what a launch's block count holds; any: 256 threads per row / per 64 positions in one launch
  const Form form = form_of(C, inner);
  const size_t most = form == kRows ? ((size_t)1 << 31) - 1 : form == kPlanes ? (size_t)1 << 36 : inner == 1 ? ((size_t)1 << 24) - 1 : ((size_t)1 << 30) - 64;
  CASMVS_REQUIRE(inner == 0 || outer <= most / inner, "%s: %zu x %zu positions of %d channels (at most %zu)", what, outer, inner, C, most);
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

template <class T, int CG, int V, Channels CH>
void planes(const Call &a, int &parts) {
  const size_t tile = (size_t)(kThreads / CG) * V, tiles = (a.positions() + tile - 1) / tile;
  // Large outputs go past the caches (8 channels per group, pairs of positions; a branch in the kernel gains nothing): a forward pass then leaves x there for the
  // backward pass instead of y.  2 x 8 x 32 x 256 x 320 in float32, forward and the backward pass right behind it 51 + 116 -> 59 + 84 us; on their own 61 -> 60 and
  // 104 -> 99 us (bf16 backward 53 -> 49).  In a training step other tensors lie between the two passes: of two samples at 640x512, 3 views, whose largest outputs this
  // concerns, 17.08 ms with it and 17.14 without (medians of three).
  constexpr bool may = CH == kFull && V > 1;
  const bool past = may && casmvs::elem::streams(a.positions() * a.C * sizeof(T));
  if (!a.gy) {
    const size_t most = loops<T>() ? kForwardBlocks : kLaunchBlocks;
    auto kernel = past ? ln_forward_planes_kernel<T, CG, V, CH == kFew, may> : ln_forward_planes_kernel<T, CG, V, CH == kFew, false>;
    for (size_t first = 0; first < tiles; first += loops<T>() ? tiles : most)
      hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles - first < most ? tiles - first : most)), dim3(kThreads), 0, a.stream, (const T *)a.x, a.w, a.b, (T *)a.out, first,
                         a.positions(), tiles, a.C, a.inner, 1.0 / a.C, a.eps, a.slope);
    return;
  }
  const unsigned grid = (unsigned)(tiles < backward_blocks(a.C) ? tiles : backward_blocks(a.C));
  parts = (int)grid;
  float *sums = a.sums(parts);
  auto kernel = past ? (a.partial ? ln_backward_planes_kernel<T, CG, V, true, CH, may> : ln_backward_planes_kernel<T, CG, V, false, CH, may>)
                     : (a.partial ? ln_backward_planes_kernel<T, CG, V, true, CH, false> : ln_backward_planes_kernel<T, CG, V, false, CH, false>);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, a.stream, (const T *)a.x, (const T *)a.gy, a.w, a.b, (T *)a.out, sums, a.positions(), tiles,
                     a.C, a.inner, 1.0 / a.C, a.eps, a.slope);
}
template <class T, int V>
void planes_by_groups(const Call &a, int &parts) {
  switch (a.C) {
    case kHeld: return planes<T, 1, V, kFull>(a, parts);
    case 2 * kHeld: return planes<T, 2, V, kFull>(a, parts);
    case 4 * kHeld: return planes<T, 4, V, kFull>(a, parts);
    case 8 * kHeld: return planes<T, 8, V, kFull>(a, parts);
    default: break;
  }
  if (a.C < kHeld) planes<T, 1, V, kFew>(a, parts);
  else if (a.C <= 2 * kHeld) planes<T, 2, V, kSome>(a, parts);
  else if (a.C <= 4 * kHeld) planes<T, 4, V, kSome>(a, parts);
  else if (a.C <= 8 * kHeld) planes<T, 8, V, kSome>(a, parts);
  else if (a.C <= 16 * kHeld) planes<T, 16, V, kSome>(a, parts);   // (67 MB of 100 channels in float32: 26 / 55 us, in 64 groups 74 / 248; bf16 48 / 91 and 231 / 903)
  else planes<T, 64, V, kSome>(a, parts);
}

template <class T, int L, int V, int K, bool FEW = false>
void rows(const Call &a, int &parts) {
  constexpr int threads = row_threads<L>();
  const size_t blocks = (a.outer + threads / L - 1) / (threads / L);
  if (!a.gy) {
    for (size_t first = 0; first < blocks; first += kLaunchBlocks)
      hipLaunchKernelGGL((ln_forward_rows_kernel<T, L, V, K, FEW>), dim3(launch_blocks(blocks - first)), dim3(threads), 0, a.stream, (const T *)a.x, a.w, a.b, (T *)a.out,
                         first, a.outer, a.C, 1.0 / a.C, a.eps, a.slope);
    return;
  }
  const unsigned grid = (unsigned)(blocks < backward_blocks(a.C) ? blocks : backward_blocks(a.C));
  parts = (int)grid;
  float *sums = a.sums(parts);
  auto kernel = a.partial ? ln_backward_rows_kernel<T, L, V, K, true, FEW> : ln_backward_rows_kernel<T, L, V, K, false, FEW>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), 0, a.stream, (const T *)a.x, (const T *)a.gy, a.w, a.b, (T *)a.out, sums, a.outer, a.C, 1.0 / a.C, a.eps, a.slope);
}
template <class T, int V>
void rows_by_width(const Call &a, int &parts) {
  const int vectors = (a.C + V - 1) / V;
  constexpr int k16 = 16 / V;   // 16 channels per lane
  if (a.C < kHeld) return rows<T, 8 / V, V, 1, true>(a, parts);
  if constexpr (V > 1)   // (4 lanes, one channel each: fewer than 8)
    if (vectors <= 4) return rows<T, 4, V, 1>(a, parts);
  if (vectors <= 8) rows<T, 8, V, 1>(a, parts);
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
      if (wide) planes_by_groups<T, 2>(a, parts); else planes_by_groups<T, 1>(a, parts);
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
  if (form_of(C, inner) != kAny) return (positions < backward_blocks(C) ? positions : backward_blocks(C)) * 2 * C * sizeof(float) + 16;
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
