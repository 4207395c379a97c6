// Layer norm over the channel axis + leaky ReLU, forward and backward.
//
//   position p of (outer, C, inner), channels c:   mu = mean_c x,  v = mean_c (x - mu)^2,  r = 1 / sqrt(v + eps),  h = (x - mu) r
//   z = h w_c + b_c,   y = z > 0 ? z : slope z
//   g = gy (z > 0 ? 1 : slope),  m1 = mean_c (g w),  m2 = mean_c (g w h):   gx = r (g w - m1 - h m2),  gw_c = sum_p g h,  gb_c = sum_p g
//
// The backward pass takes x and recomputes mu, r and the side of zero that z lies on: x has to be read for h anyway, and two stored floats per position
// would be a quarter of the traffic at 8 channels.  Statistics and z are held in 64 bits: an element whose z is within float32's rounding of zero would
// otherwise get the slope in one computation and 1 in another, an error of the size of the gradient itself; the vector ALU does 64-bit multiply-adds at the
// rate of scalar float32 ones, and these kernels wait for memory.
#include "elem_types.h"

namespace {
using casmvs::elem::Vec;

constexpr int kThreads = 256;
constexpr int kSlicePositions = 1024;   // positions per slice of the weight gradient's partial sums, before kMostSlices is reached
constexpr int kMostSlices = 256;

// ---- any number of channels --------------------------------------------------------------------------------------------------------------------------
// ROWS (inner == 1): one workgroup per position, its threads along the channels.  Otherwise 64 consecutive positions per workgroup, four threads each.
// x is read once per use (three times forward, three backward): these forms serve the shapes that do not fit registers.
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

// grad_weight / grad_bias from the slices' partial sums, in their order (no slices: zeros)
__global__ __launch_bounds__(kThreads) void ln_finish_kernel(const double *__restrict__ partial, float *__restrict__ gw, float *__restrict__ gb, int slices, int C) {
  const int i = blockIdx.x * kThreads + threadIdx.x;   // (kind, channel)
  if (i >= 2 * C) return;
  double s = 0.0;
  for (int k = 0; k < slices; ++k) s += partial[(size_t)k * 2 * C + i];
  (i < C ? gw[i] : gb[i - C]) = (float)s;
}

int slices_of(size_t positions) {
  const size_t n = (positions + kSlicePositions - 1) / kSlicePositions;
  return (int)(n < 1 ? 1 : n > kMostSlices ? kMostSlices : n);
}

int check_sizes(const char *what, int dtype, size_t outer, int C, size_t inner) {
  CASMVS_REQUIRE(casmvs::elem::known(dtype), "%s: dtype %d", what, dtype);
  CASMVS_REQUIRE(C > 0 && C <= 65535, "%s: C=%d (1 .. 65535)", what, C);
  // (launches are one workgroup per row / per 64 positions)
  CASMVS_REQUIRE(inner == 0 || outer <= ((size_t)1 << 36) / inner, "%s: %zu x %zu positions", what, outer, inner);
  CASMVS_REQUIRE(inner != 1 || outer < ((size_t)1 << 31), "%s: %zu rows", what, outer);
  return CASMVS_OK;
}
}  // namespace

extern "C" int casmvs_layer_norm_forward(const void *x, const float *weight, const float *bias, void *y, int dtype, size_t outer, int C, size_t inner,
                                         float eps, float slope, void *stream) {
  casmvs::clear_error();
  if (int rc = check_sizes("layer_norm_forward", dtype, outer, C, inner)) return rc;
  if (outer == 0 || inner == 0) return CASMVS_OK;
  CASMVS_REQUIRE(x && y, "layer_norm_forward: null pointer");
  hipStream_t st = (hipStream_t)stream;
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
  return positions * 16 + (size_t)slices_of(positions) * 2 * C * 8 + 16;
}

extern "C" int casmvs_layer_norm_backward(const void *x, const void *grad_y, const float *weight, const float *bias, void *grad_x, float *grad_weight,
                                          float *grad_bias, void *workspace, int dtype, size_t outer, int C, size_t inner, float eps, float slope,
                                          void *stream) {
  casmvs::clear_error();
  if (int rc = check_sizes("layer_norm_backward", dtype, outer, C, inner)) return rc;
  CASMVS_REQUIRE((grad_weight == nullptr) == (grad_bias == nullptr), "layer_norm_backward: grad_weight and grad_bias go together");
  const size_t positions = outer * inner;
  hipStream_t st = (hipStream_t)stream;
  CASMVS_REQUIRE(workspace, "layer_norm_backward: null workspace");
  double *stats = (double *)workspace, *partial = stats + 2 * positions;
  const int slices = positions ? slices_of(positions) : 0;
  if (positions) {
    CASMVS_REQUIRE(x && grad_y, "layer_norm_backward: null pointer");
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
  }
  if (grad_weight)
    hipLaunchKernelGGL(ln_finish_kernel, dim3((unsigned)((2 * (size_t)C + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, partial, grad_weight, grad_bias, slices, C);
  return casmvs::check_launch("layer_norm_backward");
}
