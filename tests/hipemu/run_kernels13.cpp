// As run_kernels2.cpp, for the training-side operators (layer_norm.hip, checkpoint8.hip, depth_ce.hip): the kernels' own source against the definition in
// float64 - one channel to more than a workgroup holds, odd planes, misaligned widths, one position, masked pixels, non-finite blocks.  Every buffer is a heap allocation of
// exactly its size, so a build with the address sanitizer reports an access outside it.
#define __shared__ static   // the kernels keep their LDS in function-scope arrays (workgroups run one after the other here)
#include "support.h"

// what these sources use beyond the emulated subset
inline double hipemu_rsq(double a) { return (double)(float)(1.0 / std::sqrt(a)); }   // an estimate of 24 bits
#define __builtin_amdgcn_rsq hipemu_rsq
#define __builtin_amdgcn_exp2f(x) exp2f(x)
#define __builtin_nontemporal_store(v, p) (*(p) = (v))
inline int hipemu_bpermute(int from, int v) { return hipemu_lane_exchange(v, (from >> 2) & 63); }
#define __builtin_amdgcn_ds_bpermute hipemu_bpermute

#include "block8.h"
#include "elem_types.h"

// (the three sources name their constants alike; their entry points are the ones casmvs.h declares)
namespace ln {
#include "layer_norm.hip"
}
namespace c8 {
#include "checkpoint8.hip"
}
namespace ce {
#include "depth_ce.hip"
}

template <class T>
static T *heap(size_t n) { return (T *)std::malloc(n * sizeof(T) ? n * sizeof(T) : 1); }
template <class T>
static double value(T v) { return (double)(float)v; }

static double g_worst = 0;
static void take(const char *what, double err, double limit) {
  printf("%s: %.2e of the limit\n", what, err / limit);
  g_worst = std::fmax(g_worst, std::isfinite(err) ? err / limit : 1e9);
}

template <class T>
static void layer_norm_check(const char *name, int dtype, double half_step, size_t outer, int C, size_t inner, float slope, bool affine) {
  const size_t numel = outer * C * inner, positions = outer * inner;
  T *x = heap<T>(numel), *gy = heap<T>(numel), *y = heap<T>(numel), *gx = heap<T>(numel);
  float *w = heap<float>(C), *b = heap<float>(C), *gw = heap<float>(C), *gb = heap<float>(C);
  for (size_t i = 0; i < numel; ++i) { x[i] = (T)(rnd() * 2.0f + 0.3f); gy[i] = (T)rnd(); }
  for (int c = 0; c < C; ++c) { w[c] = 1.0f + 0.4f * rnd(); b[c] = 0.3f * rnd(); }
  void *ws = std::malloc(casmvs_layer_norm_backward_workspace_bytes(dtype, outer, C, inner));
  if (casmvs_layer_norm_forward(x, affine ? w : nullptr, affine ? b : nullptr, y, dtype, outer, C, inner, 1e-5f, slope, nullptr) ||
      casmvs_layer_norm_backward(x, gy, affine ? w : nullptr, affine ? b : nullptr, gx, gw, gb, ws, dtype, outer, C, inner, 1e-5f, slope, nullptr)) {
    printf("%s: %s\n", name, casmvs_last_error());
    g_worst = 1e9;
  }
  std::vector<double> sw(C, 0.0), sb(C, 0.0), aw(C, 0.0), ab(C, 0.0);
  const double subnormal = half_step == 0x1p-11 ? 0x1p-25 : 0.0;   // half a step of float16's subnormal values (small z times the slope)
  double ey = 0, ex = 0;   // in units of half a step of the type at the value (plus float32's of the terms)
  for (size_t p = 0; p < positions; ++p) {
    const size_t base = p / inner * C * inner + p % inner;
    double mean = 0, var = 0, m1 = 0, m2 = 0, a1 = 0, a2 = 0;
    for (int c = 0; c < C; ++c) mean += value(x[base + c * inner]) / C;
    for (int c = 0; c < C; ++c) var += (value(x[base + c * inner]) - mean) * (value(x[base + c * inner]) - mean) / C;
    const double r = 1.0 / std::sqrt(var + 1e-5f);
    for (int c = 0; c < C; ++c) {
      const double h = (value(x[base + c * inner]) - mean) * r, wc = affine ? w[c] : 1.0, z = h * wc + (affine ? b[c] : 0.0);
      const double want = z > 0 ? z : z * slope, g = value(gy[base + c * inner]) * (z > 0 ? 1.0 : slope);
      ey = std::fmax(ey, std::fabs(value(y[base + c * inner]) - want) / (std::fabs(want) * half_step + 0x1p-24 * (4 * std::fabs(h * wc) + 2 * std::fabs(z)) + subnormal + 1e-12));
      m1 += g * wc / C;
      m2 += g * wc * h / C;
      a1 += std::fabs(g * wc) / C;
      a2 += std::fabs(g * wc * h) / C;
      sw[c] += g * h;
      sb[c] += g;
      aw[c] += std::fabs(g * h);
      ab[c] += std::fabs(g);
    }
    for (int c = 0; c < C; ++c) {
      const double h = (value(x[base + c * inner]) - mean) * r, wc = affine ? w[c] : 1.0, z = h * wc + (affine ? b[c] : 0.0);
      const double g = value(gy[base + c * inner]) * (z > 0 ? 1.0 : slope) * wc, want = r * (g - m1 - h * m2);
      // every term passes at most 16 float32 roundings; the means' go by the sizes of what is averaged, which cancels in the means themselves
      ex = std::fmax(ex, std::fabs(value(gx[base + c * inner]) - want) / (std::fabs(want) * half_step + 16 * 0x1p-24 * r * (std::fabs(g) + a1 + std::fabs(h) * a2) + subnormal + 1e-12));
    }
  }
  double ea = 0;
  for (int c = 0; c < C; ++c) {
    ea = std::fmax(ea, std::fabs(gw[c] - sw[c]) / (1e-6 * aw[c] + 1e-12));
    ea = std::fmax(ea, std::fabs(gb[c] - sb[c]) / (1e-6 * ab[c] + 1e-12));
  }
  char what[200];
  snprintf(what, sizeof(what), "layer_norm %s (%zu, %d, %zu) y / gx / gw, gb %.2f %.2f %.2f", name, outer, C, inner, ey, ex, ea);
  take(what, std::fmax(ey, std::fmax(ex, ea)), 1.05);
  std::free(x); std::free(gy); std::free(y); std::free(gx); std::free(w); std::free(b); std::free(gw); std::free(gb); std::free(ws);
}

static double held(double v, double top) {   // what a block whose largest magnitude is `top` holds of v
  if (!std::isfinite(top)) return NAN;
  const int e = top > 0 ? std::max((int)std::floor(std::log2(top)), -127) : -127;
  const double step = std::ldexp(1.0, e - 6), q = std::min(127.0, std::nearbyint(std::fabs(v) / step)) * step;
  return v < 0 ? -q : q;
}

template <class T>
static void pack_check(const char *name, int dtype, size_t rows, size_t n) {
  const size_t nb = (n + 31) / 32;
  T *x = heap<T>(rows * n), *out = heap<T>(rows * n);
  unsigned char *codes = heap<unsigned char>(rows * nb * 32), *scales = heap<unsigned char>(rows * nb);
  for (size_t i = 0; i < rows * n; ++i) x[i] = (T)(i % 97 < 40 ? 0.0f : rnd() * (1 + i % 5));
  if (rows * n > 70) { x[64] = (T)(float)INFINITY; x[rows * n - 1] = (T)(float)NAN; }
  if (casmvs_pack8(x, dtype, rows, n, codes, scales, nullptr) || casmvs_unpack8(codes, scales, nullptr, nullptr, 1, 1.0f, out, dtype, rows, n, nullptr)) {
    printf("%s: %s\n", name, casmvs_last_error());
    g_worst = 1e9;
  }
  size_t wrong = 0;
  for (size_t r = 0; r < rows; ++r)
    for (size_t i = 0; i < n; ++i) {
      double top = 0;
      for (size_t j = i / 32 * 32; j < std::min(n, i / 32 * 32 + 32); ++j) {
        const double a = std::fabs(value(x[r * n + j]));
        top = std::isnan(a) || a > top ? a : top;
        if (std::isnan(top)) break;
      }
      const double want = value((T)(float)held(value(x[r * n + i]), top)), got = value(out[r * n + i]);
      wrong += !(want == got || (std::isnan(want) && std::isnan(got)));
    }
  char what[160];
  snprintf(what, sizeof(what), "pack8 %s (%zu, %zu): %zu wrong", name, rows, n, wrong);
  take(what, (double)wrong, 0.5);
  std::free(x); std::free(out); std::free(codes); std::free(scales);
}

static void abn_check(int N, int C, size_t n, float slope, float abs_eps) {
  const size_t numel = (size_t)N * C * n, nb = (n + 31) / 32, planes = (size_t)N * C;
  const double M = (double)N * n;
  float *x = heap<float>(numel), *gy = heap<float>(numel), *y = heap<float>(numel), *gx = heap<float>(numel), *again = heap<float>(numel);
  float *w = heap<float>(C), *b = heap<float>(C), *rm = heap<float>(C), *rv = heap<float>(C), *vec = heap<float>(4 * C), *gw = heap<float>(C), *gb = heap<float>(C);
  unsigned char *codes = heap<unsigned char>(planes * nb * 32), *scales = heap<unsigned char>(planes * nb);
  unsigned *signs = heap<unsigned>(planes * nb);
  void *ws = std::malloc(casmvs_abn8_workspace_bytes(N, C, n));
  for (size_t i = 0; i < numel; ++i) { x[i] = rnd() * 2.0f + 0.3f * (float)((i / n) % C); gy[i] = rnd(); }
  for (int c = 0; c < C; ++c) { w[c] = (c & 1 ? -1.0f : 1.0f) * (0.9f + 0.4f * rnd()); b[c] = 0.3f * rnd(); rm[c] = 0.5f; rv[c] = 2.0f; }
  std::vector<double> mean(C, 0.0), var(C, 0.0);
  for (size_t i = 0; i < numel; ++i) mean[i / n % C] += x[i] / M;
  for (size_t i = 0; i < numel; ++i) var[i / n % C] += (x[i] - mean[i / n % C]) * (x[i] - mean[i / n % C]) / M;
  if (casmvs_abn8_forward_f32(x, w, b, abs_eps, 1e-5f, 0.1f, rm, rv, vec, y, codes, scales, signs, ws, N, C, n, slope, nullptr) ||
      casmvs_abn8_backward_f32(gy, codes, scales, signs, w, abs_eps, vec, gw, gb, gx, ws, N, C, n, slope, nullptr) ||
      casmvs_unpack8(codes, scales, vec + 2 * C, vec + 3 * C, C, slope, again, CASMVS_DTYPE_F32, planes, n, nullptr)) {
    printf("abn8: %s\n", casmvs_last_error());
    g_worst = 1e9;
  }
  std::vector<double> xq(numel), up(numel), sw(C, 0.0), sb(C, 0.0), aw(C, 0.0), ab(C, 0.0);
  double ey = 0, eu = 0, ex = 0, ew = 0, er = 0;
  for (size_t p = 0; p < planes; ++p) {
    const int c = (int)(p % C);
    const double gamma = abs_eps >= 0 ? std::fabs(w[c]) + abs_eps : w[c], r = 1.0 / std::sqrt(var[c] + 1e-5f);
    for (size_t i = 0; i < n; ++i) {
      double top = 0;
      for (size_t j = i / 32 * 32; j < std::min(n, i / 32 * 32 + 32); ++j) top = std::fmax(top, std::fabs((x[p * n + j] - mean[c]) * r));
      const double h = (x[p * n + i] - mean[c]) * r, z = h * gamma + b[c];
      xq[p * n + i] = held(h, top);
      up[p * n + i] = z > 0 ? 1.0 : slope;
      const double want = z > 0 ? z : z * slope, g = gy[p * n + i] * up[p * n + i], zq = xq[p * n + i] * gamma + b[c];
      ey = std::fmax(ey, std::fabs(y[p * n + i] - want) / (2e-6 * (std::fabs(z) + std::fabs(mean[c] * r * gamma) + 1)));
      eu = std::fmax(eu, std::fabs(again[p * n + i] - (zq > 0 ? zq : zq * slope)) / (2e-7 * (std::fabs(zq) + std::fabs(b[c]) + 1e-3)));
      sw[c] += g * xq[p * n + i];
      sb[c] += g;
      aw[c] += std::fabs(g * xq[p * n + i]);
      ab[c] += std::fabs(g);
    }
  }
  for (size_t i = 0; i < numel; ++i) {
    const int c = (int)(i / n % C);
    const double gamma = abs_eps >= 0 ? std::fabs(w[c]) + abs_eps : w[c], a = gamma / std::sqrt(var[c] + 1e-5f), g = gy[i] * up[i];
    const double want = a * (g - sb[c] / M - xq[i] * sw[c] / M);
    ex = std::fmax(ex, std::fabs(gx[i] - want) / (1e-6 * std::fabs(a) * (std::fabs(g) + std::fabs(sb[c] / M) + std::fabs(xq[i] * sw[c] / M)) + 1e-9));
  }
  for (int c = 0; c < C; ++c) {
    const double sgn = abs_eps >= 0 ? (w[c] > 0 ? 1 : -1) : 1;
    ew = std::fmax(ew, std::fabs(gw[c] - sw[c] * sgn) / (1e-6 * aw[c] + 1e-9));
    ew = std::fmax(ew, std::fabs(gb[c] - sb[c]) / (1e-6 * ab[c] + 1e-9));
    er = std::fmax(er, std::fabs(rm[c] - (0.45 + 0.1 * mean[c])) / 1e-6);
    er = std::fmax(er, std::fabs(rv[c] - (1.8 + 0.1 * var[c] * M / std::max(M - 1, 1.0))) / 1e-6);
  }
  char what[200];
  snprintf(what, sizeof(what), "abn8 (%d, %d, %zu) y / y again / gx / gw, gb / running %.2f %.2f %.2f %.2f %.2f", N, C, n, ey, eu, ex, ew, er);
  take(what, std::fmax(std::fmax(ey, eu), std::fmax(ex, std::fmax(ew, er))), 1.0);
  for (void *p : {(void *)x, (void *)gy, (void *)y, (void *)gx, (void *)again, (void *)w, (void *)b, (void *)rm, (void *)rv, (void *)vec, (void *)gw, (void *)gb, (void *)codes,
                  (void *)scales, (void *)signs, ws})
    std::free(p);
}

template <class T>
static void ce_check(const char *name, int dtype, double half_step, int B, int D, size_t hw, bool per_pixel, bool with_mask) {
  const size_t pixels = B * hw, numel = pixels * D;
  T *cost = heap<T>(numel), *grad = heap<T>(numel);
  float *depth = heap<float>(per_pixel ? numel : (size_t)B * D), *gt = heap<float>(pixels), *stats = heap<float>(2 * pixels), loss = -1, share = -1, up = 2.0f;
  unsigned char *mask = heap<unsigned char>(pixels);
  int *target = heap<int>(pixels);
  for (size_t i = 0; i < numel; ++i) cost[i] = (T)(rnd() * 3.0f);
  for (int b = 0; b < B; ++b)
    for (int k = 0; k < D; ++k)
      for (size_t s = 0; s < (per_pixel ? hw : 1); ++s)
        depth[per_pixel ? ((size_t)b * D + k) * hw + s : (size_t)b * D + k] = 400.0f + b + (per_pixel ? (float)(s % 7) : 0.0f) + 2.0f * k;
  for (size_t p = 0; p < pixels; ++p) {
    gt[p] = p % 5 == 3 ? 405.0f + (float)(p % 7) : 400.0f + rnd() * 2.2f * D;   // some exactly between two planes
    mask[p] = p % 3 != 1;
  }
  for (int k = 0; k < D && pixels > 5; ++k) cost[(size_t)k * hw + (hw > 2 ? 2 : 0)] = (T)(k ? -INFINITY : 1.0f);   // all but one masked by -inf
  if (pixels > 20)
    for (int k = 0; k < D; ++k) cost[(size_t)k * hw + (hw > 9 ? 9 : 0)] = (T)-INFINITY;   // nothing left
  void *ws = std::malloc(casmvs_depth_ce_workspace_bytes(B, D, hw));
  if (casmvs_depth_ce_forward(cost, depth, gt, with_mask ? mask : nullptr, stats, target, &loss, &share, ws, dtype, B, D, hw, per_pixel, nullptr) ||
      casmvs_depth_ce_backward(cost, stats, target, &share, &up, grad, dtype, B, D, hw, nullptr)) {
    printf("%s: %s\n", name, casmvs_last_error());
    g_worst = 1e9;
  }
  double want = 0, count = 0, eg = 0;
  size_t wrong = 0;
  std::vector<int> at(pixels, -1);
  std::vector<double> m(pixels), sum(pixels, 0.0);
  for (size_t p = 0; p < pixels; ++p) {
    const size_t b = p / hw, s = p % hw;
    auto d = [&](int k) { return (double)depth[per_pixel ? (b * D + k) * hw + s : b * D + k]; };
    auto c = [&](int k) { return value(cost[(b * D + k) * hw + s]); };
    double low = INFINITY, high = -INFINITY;
    int near = 0;
    m[p] = -INFINITY;
    for (int k = 0; k < D; ++k) {
      low = std::fmin(low, d(k));
      high = std::fmax(high, d(k));
      if (std::fabs(d(k) - gt[p]) < std::fabs(d(near) - gt[p])) near = k;
      m[p] = std::fmax(m[p], c(k));
    }
    if ((with_mask && !mask[p]) || gt[p] < low || gt[p] > high || m[p] == -INFINITY) near = -1;
    at[p] = near;
    wrong += target[p] != near;
    if (near < 0) continue;
    for (int k = 0; k < D; ++k) sum[p] += std::exp(c(k) - m[p]);
    want += std::log(sum[p]) + m[p] - c(near);
    count += 1;
  }
  want = count ? want / count : 0.0;
  for (size_t p = 0; p < pixels; ++p)
    for (int k = 0; k < D; ++k) {
      const size_t i = (p / hw * D + k) * hw + p % hw;
      const double q = at[p] < 0 ? 0.0 : 2.0 * (std::exp(value(cost[i]) - m[p]) / sum[p] - (k == at[p])) / count;
      eg = std::fmax(eg, std::fabs(value(grad[i]) - q) / (std::fabs(q) * half_step + (at[p] < 0 ? 1e-30 : 4e-6 / count + (half_step > 1e-4 ? 6e-8 : 0.0))));
    }
  const bool same = std::isinf(want) ? std::isinf(loss) : std::fabs(loss - want) <= 4e-6 * std::fabs(want) + 1e-7;
  char what[200];
  snprintf(what, sizeof(what), "depth_ce %s (%d, %d, %zu): %zu targets wrong, loss %.6g (%.6g), grad %.2f", name, B, D, hw, wrong, loss, want, eg);
  take(what, (wrong || !same) ? 1e9 : eg, 1.05);
  for (void *p : {(void *)cost, (void *)grad, (void *)depth, (void *)gt, (void *)stats, (void *)mask, (void *)target, ws}) std::free(p);
}

int main(int argc, char **argv) {
  hipemu::g_lds = smem_raw;
  const bool quick = argc > 1 && std::string(argv[1]) == "quick";
  using casmvs::elem::bf16;
  using casmvs::elem::f16;
  const double h32 = 0x1p-24, h16 = 0x1p-11, hb = 0x1p-8;
  const int F32 = CASMVS_DTYPE_F32, F16 = CASMVS_DTYPE_F16, BF16 = CASMVS_DTYPE_BF16;
  layer_norm_check<float>("f32", F32, h32, 2, 8, 65, 0.01f, true);
  layer_norm_check<float>("f32", F32, h32, 2, 32, 12, 0.01f, true);
  layer_norm_check<float>("f32", F32, h32, 1, 1, 3, 0.01f, true);
  layer_norm_check<float>("f32", F32, h32, 3, 2, 20, 1.0f, false);
  layer_norm_check<float>("f32", F32, h32, 1, 100, 12, 0.01f, true);
  layer_norm_check<float>("f32", F32, h32, 2, 520, 3, 0.01f, true);
  layer_norm_check<float>("f32", F32, h32, 5, 20, 1, 0.01f, true);
  layer_norm_check<float>("f32", F32, h32, 1, 300, 1, 1.0f, true);
  layer_norm_check<bf16>("bf16", BF16, hb, 3, 40, 1, 1.0f, true);
  layer_norm_check<f16>("f16", F16, h16, 2, 19, 24, 0.0f, true);
  if (!quick) {
    layer_norm_check<float>("f32", F32, h32, 2, 4100, 1, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 2, 8, 2304, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 1, 600, 9, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 1, 500, 40, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 1, 60, 1100, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 1, 12, 33, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 130, 16, 1, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 70, 31, 1, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 6, 2050, 1, 0.01f, true);
    layer_norm_check<float>("f32", F32, h32, 2, 9000, 1, 0.01f, true);
    layer_norm_check<bf16>("bf16", BF16, hb, 7, 1000, 1, 1.0f, true);
    layer_norm_check<bf16>("bf16", BF16, hb, 1, 8, 1040, 0.01f, true);
    layer_norm_check<f16>("f16", F16, h16, 9, 257, 1, 0.01f, false);
    layer_norm_check<f16>("f16", F16, h16, 1, 64, 130, 0.01f, true);
  }
  pack_check<float>("f32", F32, 3, 40);
  pack_check<float>("f32", F32, 1, 1);
  pack_check<float>("f32", F32, 5, 96);
  pack_check<bf16>("bf16", BF16, 2, 71);
  pack_check<f16>("f16", F16, 4, 44);
  if (!quick) { pack_check<float>("f32", F32, 7, 1033); pack_check<bf16>("bf16", BF16, 2, 9000); }
  abn_check(2, 3, 70, 0.01f, -1.0f);
  abn_check(1, 2, 64, 0.01f, 1e-5f);
  if (!quick) { abn_check(2, 4, 9001, 0.0f, -1.0f); abn_check(2, 2, 8448, 1.0f, -1.0f); abn_check(1, 64, 16, 0.01f, -1.0f); }
  ce_check<float>("f32", F32, h32, 2, 8, 45, true, true);
  ce_check<float>("f32", F32, h32, 1, 1, 3, true, false);
  ce_check<bf16>("bf16", BF16, hb, 2, 33, 30, false, true);
  ce_check<f16>("f16", F16, h16, 1, 5, 70, true, false);
  if (!quick) { ce_check<float>("f32", F32, h32, 3, 192, 100, false, true); ce_check<float>("f32", F32, h32, 2, 48, 200, true, true); ce_check<bf16>("bf16", BF16, hb, 1, 30, 264, true, true); }
  printf(g_worst < 1.0 ? "ALL OK (worst %.2e)\n" : "FAILED (worst %.2e)\n", g_worst);
  return g_worst < 1.0 ? 0 : 1;
}
