// Softmax cross entropy over the depth hypotheses, forward and backward.
//
//   t = argmin_k |d_k - gt| (lowest k on ties);  a pixel counts if its mask is set, min_k d_k <= gt <= max_k d_k and some cost is above -inf
//   loss = mean over the counted pixels of (log sum_k exp(c_k) - c_t);   d loss / d c_k = (exp(c_k - m) / s - [k = t]) / count
//
// One pass over the hypothesis axis with the running maximum m and the sum s of exp(c_k - m); what the backward pass needs beside the costs is m, 1 / s and
// t (12 bytes per pixel), never a volume of probabilities.  m and 1 / s are kept apart: their sum m + log s, rounded to float32, would move every
// probability by the rounding of a number as large as the costs.  The distances to gt are compared in float32; rounding keeps their order or makes two of them
// equal, and only where equal ones were met they are compared again in 64 bits, where differences of float32 depths are exact: which of two planes is the nearer one does not
// depend on a rounding.
// Both passes wait for memory: forward cost + depth value per hypothesis, backward cost in and gradient out.  A pixel whose mask is not set reads nothing.
// Forward (two launches) / backward: 2 x 48 x 128 x 160 9.3 / 5.5 us - launches -, 2 x 32 x 256 x 320 14 / 9.3, 2 x 8 x 512 x 640 16 / 11 us; bf16 with one set of
// planes per sample, 192 x 295 x 399: 28 / 24 us (45 MB in, 45 MB out: strides of 117705 elements, so 2-byte loads).
#include "elem_types.h"

namespace {
using casmvs::elem::Vec;

constexpr int kThreads = 256;
constexpr int kChunk = 8;   // hypotheses loaded before they are used

struct Running {   // of one pixel over some of its hypotheses
  float m, s;         // the largest cost, sum of exp(cost - m)
  float near;         // the smallest distance to gt, rounded to float32, and where it is first
  int at;
  float low, high;    // smallest / largest depth
};

// exp(a - m) for a <= m by the hardware's 2^x, the argument rounded once more (2^-24 of at most 127, for a probability of 2^-127).  m may be -inf (then a is, too): 0.
__device__ __forceinline__ float exp_below(float a, float m) { return __builtin_amdgcn_exp2f((a - (m == -INFINITY ? 0.0f : m)) * 1.44269504088896341f); }

// Is depth `a` nearer to `gt` than `b`, whose rounded distances are equal?
__device__ __forceinline__ bool nearer(float a, float b, float gt) { return __builtin_fabs((double)a - (double)gt) < __builtin_fabs((double)b - (double)gt); }

// o: the hypotheses behind r's; dp, dstep: the pixel's depths.  A piece without a finite distance has no nearest one to compare: a pixel between its lowest and highest
// hypothesis is less than float32's largest number away from one of the two.
__device__ __forceinline__ void join(Running &r, const Running &o, const float *__restrict__ dp, size_t dstep, float gt) {
  const float m = fmaxf(r.m, o.m);
  r.s = r.s * exp_below(r.m, m) + o.s * exp_below(o.m, m);
  r.m = m;
  bool take = o.near < r.near;
  if (o.near == r.near && o.near < INFINITY) take = nearer(dp[o.at * dstep], dp[r.at * dstep], gt);
  r.at = take ? o.at : r.at;
  r.near = fminf(r.near, o.near);
  r.low = fminf(r.low, o.low);
  r.high = fmaxf(r.high, o.high);
}

// PIECES threads share a pixel: each takes its piece of the hypothesis axis, joined at the end
template <class T, bool PER_PIXEL, int PIECES>
__global__ __launch_bounds__(kThreads) void depth_ce_forward_kernel(const T *__restrict__ cost, const float *__restrict__ depth, const float *__restrict__ gt,
                                                                   const unsigned char *__restrict__ mask, float2 *__restrict__ stats, int *__restrict__ target,
                                                                   double *__restrict__ partial, size_t pixels, int D, size_t hw) {
  constexpr int kPixels = kThreads / PIECES;
  const int lane = threadIdx.x % kPixels, piece = threadIdx.x / kPixels;
  const size_t p = (size_t)blockIdx.x * kPixels + lane;
  const bool live = p < pixels && (!mask || mask[p]);
  size_t b, s;
  casmvs::elem::divide(live ? p : 0, hw, b, s);
  Running r = {-INFINITY, 0.0f, INFINITY, 0, INFINITY, -INFINITY};
  float true_depth = 0.0f;
  const T *cp = cost + (b * D) * hw + s;
  const float *dp = PER_PIXEL ? depth + (b * D) * hw + s : depth + b * D;
  const size_t dstep = PER_PIXEL ? hw : 1;
  if (live) {
    const int per = (D + PIECES - 1) / PIECES, lo = piece * per, hi = lo + per < D ? lo + per : D;
    true_depth = gt[p];
    for (int k0 = lo; k0 < hi; k0 += kChunk) {
      float c[kChunk], d[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const int k = k0 + i < hi ? k0 + i : hi - 1;
        c[i] = (float)cp[(size_t)k * hw];
        d[i] = dp[k * dstep];
      }
      float m = r.m;
      const float near = r.near;
      const int at = r.at;
      bool tied = false;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) m = fmaxf(m, c[i]);
      r.s *= exp_below(r.m, m);
      r.m = m;
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        if (k0 + i < hi) {
          r.s += exp_below(c[i], m);
          const float far = fabsf(d[i] - true_depth);
          tied |= far == r.near;
          r.at = far < r.near ? k0 + i : r.at;
          r.near = fminf(r.near, far);
          r.low = fminf(r.low, d[i]);
          r.high = fmaxf(r.high, d[i]);
        }
      if (tied) {   // two roundings were equal (a lane in thousands): the chunk again, in 64 bits where they are
        r.near = near;
        r.at = at;
        float depth_at = dp[at * dstep];
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          const float far = fabsf(d[i] - true_depth);
          if (k0 + i < hi && (far < r.near || (far == r.near && nearer(d[i], depth_at, true_depth)))) {
            r.near = far;
            r.at = k0 + i;
            depth_at = d[i];
          }
        }
      }
    }
  }
  __shared__ Running joined[PIECES > 1 ? kThreads : 1];
  __shared__ double red[2][kPixels];
  if (PIECES > 1) {
    joined[piece * kPixels + lane] = r;
    __syncthreads();
  }
  if (piece == 0) {
    if (live)
      for (int q = 1; q < PIECES; ++q) join(r, joined[q * kPixels + lane], dp, dstep, true_depth);
    bool counted = false;
    float cost_at = 0.0f;
    if (live) {
      counted = true_depth >= r.low && true_depth <= r.high && !(r.m == -INFINITY && r.s == 0.0f);
      cost_at = (float)cp[(size_t)r.at * hw];
    }
    if (p < pixels) {
      stats[p] = float2{counted ? r.m : 0.0f, counted ? 1.0f / r.s : 0.0f};
      target[p] = counted ? r.at : -1;
    }
    red[0][lane] = counted ? (double)(logf(r.s) + (r.m - cost_at)) : 0.0;
    red[1][lane] = counted ? 1.0 : 0.0;
  }
  __syncthreads();
  for (int st = kPixels / 2; st > 0; st >>= 1) {
    if ((int)threadIdx.x < st) {
      red[0][threadIdx.x] += red[0][threadIdx.x + st];
      red[1][threadIdx.x] += red[1][threadIdx.x + st];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    partial[2 * (size_t)blockIdx.x] = red[0][0];
    partial[2 * (size_t)blockIdx.x + 1] = red[1][0];
  }
}

// loss = the mean, share = 1 / count (0 where no pixel counts: the loss and every gradient are 0 then)
__global__ __launch_bounds__(kThreads) void depth_ce_finish_kernel(const double *__restrict__ partial, size_t blocks, float *__restrict__ loss,
                                                                  float *__restrict__ share) {
  __shared__ double red[2][kThreads];
  double s0 = 0.0, s1 = 0.0;
  for (size_t b = threadIdx.x; b < blocks; b += kThreads) {
    s0 += partial[2 * b];
    s1 += partial[2 * b + 1];
  }
  red[0][threadIdx.x] = s0;
  red[1][threadIdx.x] = s1;
  __syncthreads();
  for (int st = kThreads / 2; st > 0; st >>= 1) {
    if ((int)threadIdx.x < st) {
      red[0][threadIdx.x] += red[0][threadIdx.x + st];
      red[1][threadIdx.x] += red[1][threadIdx.x + st];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *loss = red[1][0] > 0.0 ? (float)(red[0][0] / red[1][0]) : 0.0f;
    *share = red[1][0] > 0.0 ? (float)(1.0 / red[1][0]) : 0.0f;
  }
}

template <class T>
__global__ __launch_bounds__(kThreads) void depth_ce_backward_kernel(const T *__restrict__ cost, const float2 *__restrict__ stats, const int *__restrict__ target,
                                                                    const float *__restrict__ share_of_one, const float *__restrict__ gloss,
                                                                    T *__restrict__ grad, size_t pixels, int D, size_t hw) {
  const size_t p = (size_t)blockIdx.x * kThreads + threadIdx.x;
  if (p >= pixels) return;
  size_t b, s;
  casmvs::elem::divide(p, hw, b, s);
  const int t = target[p];
  const float2 st = stats[p];
  const float share = *share_of_one * *gloss;
  const int per = (D + (int)gridDim.y - 1) / (int)gridDim.y, lo = (int)blockIdx.y * per, hi = lo + per < D ? lo + per : D;
  const T *cp = cost + (b * D) * hw + s;
  T *gp = grad + (b * D) * hw + s;
#pragma unroll 8
  for (int k = lo; k < hi; ++k) {
    const float q = t < 0 ? 0.0f : (exp_below((float)cp[(size_t)k * hw], st.x) * st.y - (k == t ? 1.0f : 0.0f)) * share;
    gp[(size_t)k * hw] = (T)q;
  }
}

int check_sizes(const char *what, int dtype, int B, int D, size_t hw) {
  CASMVS_REQUIRE(casmvs::elem::known(dtype), "%s: dtype %d", what, dtype);
  CASMVS_REQUIRE(B > 0 && D > 0 && D <= 65536 && hw < ((size_t)1 << 31) / (size_t)B, "%s: B=%d D=%d h*w=%zu (B h w < 2^31)", what, B, D, hw);
  return CASMVS_OK;
}
// Pieces of the hypothesis axis: few pixels with many hypotheses would leave CUs idle, each thread walking its axis alone.  1 or 4 pieces, us: 32 hypotheses of
// 163840 pixels 14.3 / 15.8, 48 of 40960 10.9 / 9.4, 192 of 118400 38 / 30, 256 of 20480 42 / 17.  4 or 16: 192 of 2000 pixels 10.2 / 8.1, 512 of 1600 17.6 / 10.5,
// 1024 of 80 29.4 / 12.4, 64 of 2000 7.0 / 7.1.
int pieces_of(size_t pixels, int D) { return D < 16 || pixels >= (D <= 32 ? 65536u : 524288u) ? 1 : pixels >= 2048 || D < 64 ? 4 : 16; }
size_t forward_blocks(size_t pixels, int D) { return (pixels * pieces_of(pixels, D) + kThreads - 1) / kThreads; }
}  // namespace

extern "C" size_t casmvs_depth_ce_workspace_bytes(int B, int D, size_t hw) {
  if (B <= 0 || D <= 0) return 0;
  return forward_blocks((size_t)B * hw, D) * 16 + 16;
}

extern "C" int casmvs_depth_ce_forward(const void *cost, const float *depth_values, const float *depth_gt, const void *mask, float *stats, int *target,
                                       float *loss, float *share, void *workspace, int dtype, int B, int D, size_t hw, int per_pixel, void *stream) {
  casmvs::clear_error();
  if (int rc = check_sizes("depth_ce_forward", dtype, B, D, hw)) return rc;
  CASMVS_REQUIRE(loss && share && workspace, "depth_ce_forward: null pointer");
  const size_t pixels = (size_t)B * hw, blocks = pixels ? forward_blocks(pixels, D) : 0;
  CASMVS_REQUIRE(!pixels || (cost && depth_values && depth_gt && stats && target), "depth_ce_forward: null pointer");
  CASMVS_REQUIRE((((uintptr_t)stats | (uintptr_t)workspace) & 7) == 0, "depth_ce_forward: stats and workspace on 8-byte boundaries");
  hipStream_t st = (hipStream_t)stream;
  double *partial = (double *)workspace;
  if (pixels) {
    CASMVS_WITH_DTYPE(dtype, {
      const int pieces = pieces_of(pixels, D);
      auto kernel = pieces == 1   ? (per_pixel ? depth_ce_forward_kernel<T, true, 1> : depth_ce_forward_kernel<T, false, 1>)
                    : pieces == 4 ? (per_pixel ? depth_ce_forward_kernel<T, true, 4> : depth_ce_forward_kernel<T, false, 4>)
                                  : (per_pixel ? depth_ce_forward_kernel<T, true, 16> : depth_ce_forward_kernel<T, false, 16>);
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, (const T *)cost, depth_values, depth_gt, (const unsigned char *)mask,
                         (float2 *)stats, target, partial, pixels, D, hw);
    });
  }
  hipLaunchKernelGGL(depth_ce_finish_kernel, dim3(1), dim3(kThreads), 0, st, partial, blocks, loss, share);
  return casmvs::check_launch("depth_ce_forward");
}

extern "C" int casmvs_depth_ce_backward(const void *cost, const float *stats, const int *target, const float *share, const float *grad_loss, void *grad_cost,
                                        int dtype, int B, int D, size_t hw, void *stream) {
  casmvs::clear_error();
  if (int rc = check_sizes("depth_ce_backward", dtype, B, D, hw)) return rc;
  const size_t pixels = (size_t)B * hw;
  if (!pixels) return CASMVS_OK;
  CASMVS_REQUIRE(cost && stats && target && share && grad_loss && grad_cost, "depth_ce_backward: null pointer");
  CASMVS_REQUIRE(((uintptr_t)stats & 7) == 0, "depth_ce_backward: stats on an 8-byte boundary");
  const size_t blocks = (pixels + kThreads - 1) / kThreads;
  size_t split = 2048 / blocks;   // few pixels: pieces of the hypothesis axis
  split = split < 1 ? 1 : split > (size_t)D ? (size_t)D : split;
  CASMVS_WITH_DTYPE(dtype, {
    hipLaunchKernelGGL(depth_ce_backward_kernel<T>, dim3((unsigned)blocks, (unsigned)split), dim3(kThreads), 0, (hipStream_t)stream, (const T *)cost,
                       (const float2 *)stats, target, share, grad_loss, (T *)grad_cost, pixels, D, hw);
  });
  return casmvs::check_launch("depth_ce_backward_kernel");
}
