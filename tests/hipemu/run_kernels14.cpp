// The training-side operators (layer_norm.hip, checkpoint8.hip, depth_ce.hip) on the CPU, as run_kernels13.cpp: the calls at the edge of what their entry points allow.
// The argument names the part that runs.  Every buffer is a heap allocation of exactly its size.
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

namespace ln {
#include "layer_norm.hip"
}
namespace c8 {
#include "checkpoint8.hip"
}
namespace ce {
#include "depth_ce.hip"
}
#include <sys/mman.h>

template <class T>
static double value(T v) { return (double)(float)v; }

static double g_worst = 0;
static void take(const char *what, double err, double limit) {
  printf("%s: %.2e of the limit\n", what, err / limit);
  g_worst = std::fmax(g_worst, std::isfinite(err) ? err / limit : 1e9);
}

// eps = 0: a thread without a position has no spread to divide by, and nothing of it may reach a sum
template <class T>
static void no_eps_check(const char *name, int dtype, double half_step, size_t outer, int C, size_t inner) {
  const size_t numel = outer * C * inner, positions = outer * inner;
  std::vector<T> x(numel), gy(numel), y(numel), gx(numel);
  std::vector<float> w(C), b(C), gw(C), gb(C);
  const float slope = 0.01f;
  for (size_t i = 0; i < numel; ++i) { x[i] = (T)(rnd() * 2.0f + 0.3f); gy[i] = (T)rnd(); }
  for (int c = 0; c < C; ++c) { w[c] = 1.0f + 0.4f * rnd(); b[c] = 0.3f * rnd(); }
  std::vector<char> ws(casmvs_layer_norm_backward_workspace_bytes(dtype, outer, C, inner));
  if (casmvs_layer_norm_forward(x.data(), w.data(), b.data(), y.data(), dtype, outer, C, inner, 0.0f, slope, nullptr) ||
      casmvs_layer_norm_backward(x.data(), gy.data(), w.data(), b.data(), gx.data(), gw.data(), gb.data(), ws.data(), dtype, outer, C, inner, 0.0f, slope, nullptr)) {
    printf("%s: %s\n", name, casmvs_last_error());
    g_worst = 1e9;
  }
  std::vector<double> sw(C, 0.0), sb(C, 0.0), aw(C, 0.0), ab(C, 0.0);
  double e = 0;
  auto worse = [&](double off, double limit) { e = std::isfinite(off) ? std::fmax(e, off / limit) : 1e9; };
  for (size_t p = 0; p < positions; ++p) {
    const size_t base = p / inner * C * inner + p % inner;
    double mean = 0, var = 0, m1 = 0, m2 = 0, a1 = 0, a2 = 0;
    for (int c = 0; c < C; ++c) mean += value(x[base + c * inner]) / C;
    for (int c = 0; c < C; ++c) var += (value(x[base + c * inner]) - mean) * (value(x[base + c * inner]) - mean) / C;
    const double r = 1.0 / std::sqrt(var);
    for (int pass = 0; pass < 2; ++pass)
      for (int c = 0; c < C; ++c) {
        const size_t at = base + c * inner;
        const double h = (value(x[at]) - mean) * r, z = h * w[c] + b[c], g = value(gy[at]) * (z > 0 ? 1.0 : slope), want = z > 0 ? z : z * slope;
        if (pass == 0) {
          // z: the rounded x - mean, 1 / sqrt, two products, the sum and the slope, each half a step; then the type's own
          worse(std::fabs(value(y[at]) - want), std::fabs(want) * half_step + 0x1p-24 * (4 * std::fabs(h * w[c]) + 2 * std::fabs(z)) + 1e-12);
          m1 += g * w[c] / C;
          m2 += g * w[c] * h / C;
          a1 += std::fabs(g * w[c]) / C;
          a2 += std::fabs(g * w[c] * h) / C;
          sw[c] += g * h;
          sb[c] += g;
          aw[c] += std::fabs(g * h);
          ab[c] += std::fabs(g);
        } else {   // at most 16 float32 roundings a term, and the type's own
          const double gxw = r * (g * w[c] - m1 - h * m2);
          worse(std::fabs(value(gx[at]) - gxw), std::fabs(gxw) * half_step + 16 * 0x1p-24 * r * (std::fabs(g * w[c]) + a1 + std::fabs(h) * a2) + 1e-12);
        }
      }
  }
  for (int c = 0; c < C; ++c) {
    worse(std::fabs(gw[c] - sw[c]), 64 * 0x1p-24 * aw[c] + 1e-12);
    worse(std::fabs(gb[c] - sb[c]), 64 * 0x1p-24 * ab[c] + 1e-12);
  }
  char what[120];
  snprintf(what, sizeof(what), "eps 0 %s (%zu, %d, %zu)", name, outer, C, inner);
  take(what, e, 1.05);
}

// ABN with 8-bit checkpoints where the channels' means are many times their spread, where the first element of a channel is far from all others, and where all of
// them are equal: y, the signs, vec and the running statistics are those of 64 bits.
enum Channels { kShifted, kFirstApart, kConstant };
static void far_check(int N, int C, size_t n, float offset, Channels kind) {
  const size_t numel = (size_t)N * C * n, nb = (n + 31) / 32, planes = (size_t)N * C;
  const double M = (double)N * n;
  std::vector<float> x(numel), y(numel), w(C), b(C), rm(C, 0.5f), rv(C, 2.0f), vec(4 * C);
  std::vector<unsigned char> codes(planes * nb * 32), scales(planes * nb);
  std::vector<unsigned> signs(planes * nb);
  std::vector<char> ws(casmvs_abn8_workspace_bytes(N, C, n));
  const float slope = 0.01f;
  for (size_t i = 0; i < numel; ++i)
    x[i] = kind == kConstant ? offset : kind == kFirstApart ? (i % n == 0 && i / n < (size_t)C ? offset : rnd()) : 2.0f * rnd() + offset;
  for (int c = 0; c < C; ++c) { w[c] = (c & 1 ? -1.0f : 1.0f) * (0.9f + 0.4f * rnd()); b[c] = 0.3f * rnd(); }
  if (casmvs_abn8_forward_f32(x.data(), w.data(), b.data(), -1.0f, 1e-5f, 0.1f, rm.data(), rv.data(), vec.data(), y.data(), codes.data(), scales.data(), signs.data(),
                              ws.data(), N, C, n, slope, nullptr)) {
    printf("abn8: %s\n", casmvs_last_error());
    g_worst = 1e9;
  }
  double e = 0;
  size_t wrong = 0;
  auto worse = [&](double off, double limit) { e = std::isfinite(off) ? std::fmax(e, off / limit) : 1e9; };
  for (int c = 0; c < C; ++c) {
    // two passes over x - x0: a distance from the first element is exact, its sum as good as M values of that size allow
    double s = 0, var = 0;
    for (int img = 0; img < N; ++img)
      for (size_t i = 0; i < n; ++i) s += ((double)x[((size_t)img * C + c) * n + i] - x[c * n]) / M;
    const double mean = x[c * n] + s;
    for (int img = 0; img < N; ++img)
      for (size_t i = 0; i < n; ++i) {
        const double d = ((double)x[((size_t)img * C + c) * n + i] - x[c * n]) - s;
        var += d * d / M;
      }
    const double r = 1.0 / std::sqrt(var + 1e-5f);
    // one-pass sums: M 2^-53 of var where the first element is all there is, and as much again for the additions
    const double rel = 4 * M * 0x1p-53 + 1e-13, mean_off = 8 * 0x1p-53 * std::fabs(mean) + 1e-13 * std::fabs(s);
    for (int img = 0; img < N; ++img)
      for (size_t i = 0; i < n; ++i) {
        const size_t plane = (size_t)img * C + c, at = plane * n + i;
        const double h = ((double)x[at] - mean) * r, z = h * w[c] + b[c], want = z > 0 ? z : z * slope;
        const double z_off = mean_off * r * std::fabs(w[c]) + rel * std::fabs(h * w[c]);
        // y in float32: x - mean's two differences, scale and the product half a step each of |h w|, the sum and the slope of |z|; the mean as two floats
        const double y_off = 0x1p-24 * 1.001 * (4 * std::fabs(h * w[c]) + 2 * std::fabs(z)) + 0x1p-47 * std::fabs(mean) * r * std::fabs(w[c]) + z_off;
        worse(std::fabs(y[at] - want), (z > 0 ? 1.0 : slope) * y_off + 1e-30);
        const bool up = signs[plane * nb + i / 32] >> (i % 32) & 1;
        wrong += std::fabs(z) > z_off && up != (z > 0);
        // ... on the side of the activation that the backward pass takes
        const double side = up ? z : z * slope;
        worse(std::fabs(y[at] - side), (up ? 1.0 : slope) * y_off + 1e-30);
      }
    worse(std::fabs(vec[c] - w[c] * r), 0x1p-24 * 1.001 * std::fabs(w[c] * r) + rel * std::fabs(w[c] * r));
    worse(std::fabs(rm[c] - (0.45 + 0.1 * mean)), 4 * 0x1p-24 * (0.45 + 0.1 * std::fabs(mean)));
    worse(std::fabs(rv[c] - (1.8 + 0.1 * var * M / (M - 1))), 4 * 0x1p-24 * (1.8 + 0.1 * var) + rel * var);
  }
  char what[120];
  snprintf(what, sizeof(what), "abn8 %s (%d, %d, %zu) at %g: %zu signs wrong", kind == kConstant ? "constant" : kind == kFirstApart ? "first apart" : "shifted", N, C, n, offset, wrong);
  take(what, wrong ? 1e9 : e, 1.0);
}

// Cross entropy where every pixel is masked: costs, hypotheses and ground truth lie in memory that must not be read (a read ends the process).
static void masked_check(int B, int D, size_t hw, bool per_pixel) {
  const size_t pixels = B * hw, numel = pixels * D;
  void *apart = mmap(nullptr, numel * 4, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  std::vector<float> stats(2 * pixels, -1.0f), grad(numel, -1.0f);
  std::vector<int> target(pixels, 7);
  std::vector<unsigned char> mask(pixels, 0);
  std::vector<char> ws(casmvs_depth_ce_workspace_bytes(B, D, hw));
  float loss = -1, share = -1, up = 1;
  printf("depth_ce masked (%d, %d, %zu)%s\n", B, D, hw, per_pixel ? " per pixel" : "");
  fflush(stdout);
  if (apart == MAP_FAILED ||
      casmvs_depth_ce_forward(apart, (const float *)apart, (const float *)apart, mask.data(), stats.data(), target.data(), &loss, &share, ws.data(), CASMVS_DTYPE_F32, B, D, hw,
                              per_pixel, nullptr) ||
      casmvs_depth_ce_backward(apart, stats.data(), target.data(), &share, &up, grad.data(), CASMVS_DTYPE_F32, B, D, hw, nullptr))
    g_worst = 1e9;
  if (loss != 0.0f || share != 0.0f) g_worst = 1e9;
  for (int t : target)
    if (t != -1) g_worst = 1e9;
  for (float q : grad)
    if (q != 0.0f) g_worst = 1e9;
  munmap(apart, numel * 4);
}

// ... and where a piece of the axis has no hypotheses, or only ones whose distance is beyond float32: the nearest one is still the class
static void pieces_check(int D, size_t hw, float scale) {
  std::vector<float> cost(D * hw), depth(D), gt(hw), stats(2 * hw);
  std::vector<int> target(hw);
  std::vector<char> ws(casmvs_depth_ce_workspace_bytes(1, D, hw));
  float loss = -1, share = -1;
  for (float &c : cost) c = rnd();
  for (int k = 0; k < D; ++k) depth[k] = scale * (2.0f * k / (D - 1) - 1.0f);   // from -scale to scale
  for (size_t s = 0; s < hw; ++s) gt[s] = scale * rnd();
  if (casmvs_depth_ce_forward(cost.data(), depth.data(), gt.data(), nullptr, stats.data(), target.data(), &loss, &share, ws.data(), CASMVS_DTYPE_F32, 1, D, hw, 0, nullptr))
    g_worst = 1e9;
  size_t wrong = 0;
  for (size_t s = 0; s < hw; ++s) {
    int near = 0;
    for (int k = 1; k < D; ++k)
      if (std::fabs((double)depth[k] - gt[s]) < std::fabs((double)depth[near] - gt[s])) near = k;
    wrong += target[s] != near;
  }
  char what[120];
  snprintf(what, sizeof(what), "depth_ce pieces (%d, %zu) to %g: %zu targets wrong", D, hw, scale, wrong);
  take(what, (double)wrong, 0.5);
}

int main(int argc, char **argv) {
  hipemu::g_lds = smem_raw;
  const std::string part = argc > 1 ? argv[1] : "";
  using casmvs::elem::bf16;
  if (part == "eps0") {
    // fewer positions than a tile holds, or a last tile that is not full: 1, 2, 4, 8, 16 and 64 groups of channels, fewer than 8 channels, pairs and single positions
    for (size_t inner : {size_t(65), size_t(52)}) {
      no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 2, 8, inner);
      no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 3, inner);
      no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 16, inner);
      no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 20, inner);
    }
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 2, 32, 12);
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 3, 64, 21);
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 100, 17);
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 200, 9);
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 520, 3);
    no_eps_check<bf16>("bf16", CASMVS_DTYPE_BF16, 0x1p-8, 2, 8, 300);
    no_eps_check<bf16>("bf16", CASMVS_DTYPE_BF16, 0x1p-8, 1, 6, 10);
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 1, 8, 1024);   // a full tile
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 5, 20, 1);     // rows
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 3, 5, 1);
    no_eps_check<float>("f32", CASMVS_DTYPE_F32, 0x1p-24, 2, 300, 1);
  } else if (part == "far") {
    for (float offset : {0.0f, 1e4f, -3e6f}) {
      far_check(2, 3, 70, offset, kShifted);
      far_check(2, 2, 64, offset, kShifted);
    }
    far_check(1, 1, 16500, 3e6f, kShifted);   // (two launches)
    far_check(1, 1, 16501, -1e5f, kShifted);
    for (Channels kind : {kFirstApart, kConstant}) {
      far_check(2, 3, 70, 1e6f, kind);
      if (kind == kConstant) far_check(1, 1, 16500, 1e4f, kind);
    }
  } else if (part == "masked") {
    for (bool per_pixel : {true, false}) {
      masked_check(2, 8, 45, per_pixel);      // one piece of the axis
      masked_check(1, 33, 30, per_pixel);     // four, the last one shorter
      masked_check(1, 192, 20, per_pixel);    // sixteen
    }
    for (float scale : {1.0f, 3e38f}) {
      pieces_check(33, 300, scale);
      pieces_check(65, 40, scale);            // sixteen pieces of 5: three are empty
    }
  } else {
    printf("no part named %s\n", part.c_str());
    return 2;
  }
  printf(g_worst < 1.0 ? "ALL OK (worst %.2e)\n" : "FAILED (worst %.2e)\n", g_worst);
  return g_worst < 1.0 ? 0 : 1;
}
