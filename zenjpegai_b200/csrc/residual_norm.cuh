// Shared by the residual step with its norms, gate and scale in one kernel (residual_norm.cu,
// zjai_gated_residual_norm) and its backward pass (residual_norm_bwd.cu,
// zjai_gated_residual_norm_backward).
//
// Per position, over its c channels, with LN(v) = (v - mean v) / sqrt(var v + 1e-5):
//   u = LN(f) w1 + b1, q = s sigmoid(g), y = x + q u, z = LN(y) w2 + b2      (parts optional)
// and backward, with fn = LN(f), yn = LN(y), r1, r2 = 1 / sigma of f and y:
//   a = dz w2, D = dy + (a - mean a - yn mean(a yn)) r2, dx = D
//   du = D q, dg = D s u sigma(g) (1 - sigma(g)), ds = sum D sigma(g) u
//   b = du w1, df = (b - mean b - fn mean(b fn)) r1
//   dw1 = sum du fn, db1 = sum du, dw2 = sum dz yn, db2 = sum dz             (sums over positions)
// Maps are planar: a channel row holds a picture's positions. A block takes tiles of 32 consecutive
// positions of one picture, which are one group of each row's 8-bit tape. A lane has four
// neighbouring positions, eight lanes a row, a warp four rows at a time: vector loads and stores,
// packed f32x2 arithmetic, and a group's maximum within eight lanes (one position a lane needed
// three times the instructions, and issue slots bounded the kernels, not HBM). Up to 256 channels
// a block holds its tile in registers (kRows rows a thread) and reads everything once; above, rows
// are read again for each pass, mostly from the caches. A position's sums go over the warps'
// shared-memory partials, gathered by one warp. Statistics: a mean and sum of squared deviations
// per warp, joined by their exact update formula (sums of squares would cancel).
// The products in a - mean a and b - mean b are the ones that were summed (not fused): with one
// channel they cancel to zero. Both kernels are bound by HBM at large sizes.
#pragma once
#include <algorithm>
#include <type_traits>

#include "quad.cuh"
#include "train.h"

namespace zjai {
namespace {

constexpr float kEps = 1e-5f;
constexpr int kMaxC = 8192;  // the parameter sums of a block sit in shared memory, 20 B a channel
constexpr int kMaxWarps = 16;

// sigmoid(g) and 1 - sigmoid(g), neither by cancellation and both finite for every g but NaN
__device__ __forceinline__ void sigmoid2(float g, float* s, float* one_minus) {
  const float a = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + a), ar = a * r;
  *s = g >= 0.f ? r : ar;
  *one_minus = g >= 0.f ? ar : r;
}
__device__ __forceinline__ void sigmoid4(F4 g, F4* s, F4* one_minus) {
  sigmoid2(g.a.x, &s->a.x, &one_minus->a.x);
  sigmoid2(g.a.y, &s->a.y, &one_minus->a.y);
  sigmoid2(g.b.x, &s->b.x, &one_minus->b.x);
  sigmoid2(g.b.y, &s->b.y, &one_minus->b.y);
}

// over the four rows of a warp: lanes with the same positions
__device__ __forceinline__ F4 over_rows(F4 v) {
  float f[4] = {v.a.x, v.a.y, v.b.x, v.b.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] += __shfl_xor_sync(0xffffffffu, f[i], 8);
    f[i] += __shfl_xor_sync(0xffffffffu, f[i], 16);
  }
  return {make_float2(f[0], f[1]), make_float2(f[2], f[3])};
}

// The block's partial sums per warp and position, and their totals.
template <int kVals>
struct Exchange {
  float part[kMaxWarps][kVals][32], total[kVals][32];
};

// Rows of the calling thread: row(j) for j < rows(). kRows > 0: held in registers, consecutive
// groups of four per warp; 0: any number, strided over the block.
template <int kRows>
struct Rows {
  int c, first, step, n, warp_rows;
  __device__ __forceinline__ Rows(int c_, int warps) : c(c_) {
    const int wp = threadIdx.x >> 5, rg = (threadIdx.x & 31) >> 3;
    if (kRows) {
      first = wp * 4 * kRows + rg;
      step = 4;
      n = kRows;
      warp_rows = max(0, min(c - wp * 4 * kRows, 4 * kRows));
    } else {
      first = wp * 4 + rg;
      step = 4 * warps;
      n = (c + step - 1) / step;
      const int whole = c / step, rest = c - whole * step - wp * 4;
      warp_rows = whole * 4 + max(0, min(4, rest));
    }
  }
  __device__ __forceinline__ int row(int j) const { return first + j * step; }
  __device__ __forceinline__ bool on(int j) const { return row(j) < c; }
  // a row that exists, to read for one that does not
  __device__ __forceinline__ int param(int j) const { return min(row(j), c - 1); }
};
#define FOR_ROWS(j) _Pragma("unroll") for (int j = 0; j < (kRows ? kRows : rows.n); ++j)

// Per warp the sum and the squared deviations from the warp's own mean of v(j), to ex.part at val,
// val + 1.
template <int kRows, int kVals, class V>
__device__ __forceinline__ void stats_part(const Rows<kRows>& rows, V&& v, Exchange<kVals>& ex,
                                           int val) {
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  F4 s = all(0.f), q = all(0.f);
  FOR_ROWS(j) if (rows.on(j)) s = s + v(j);
  s = over_rows(s);
  const F4 m = s * all(rows.warp_rows ? 1.f / (float)rows.warp_rows : 0.f);
  FOR_ROWS(j) if (rows.on(j)) {
    const F4 d = v(j) - m;
    q = fma4(d, d, q);
  }
  q = over_rows(q);
  if (lane < 8) {
    *reinterpret_cast<float4*>(&ex.part[wp][val][lane * 4]) = flat(s);
    *reinterpret_cast<float4*>(&ex.part[wp][val + 1][lane * 4]) = flat(q);
  }
}
// Joined by one warp: ex.total at val, val + 1 the mean and 1 / sigma.
template <int kRows, int kVals>
__device__ __forceinline__ void stats_join(Exchange<kVals>& ex, int val, int c, int warps) {
  const int lane = threadIdx.x & 31;
  float s = 0.f, q = 0.f;
  for (int w = 0; w < warps; ++w) s += ex.part[w][val][lane];
  const float m = s / (float)c;
  for (int w = 0; w < warps; ++w) {
    // rows of warp w, as in Rows
    int n;
    if (kRows) {
      n = max(0, min(c - w * 4 * kRows, 4 * kRows));
    } else {
      const int whole = c / (4 * warps);
      n = whole * 4 + max(0, min(4, c - whole * 4 * warps - w * 4));
    }
    if (!n) continue;
    const float d = ex.part[w][val][lane] / (float)n - m;
    q += ex.part[w][val + 1][lane] + (float)n * d * d;
  }
  ex.total[val][lane] = m;
  ex.total[val + 1][lane] = rsqrtf(q / (float)c + kEps);
}
template <int kVals>
__device__ __forceinline__ F4 total4(const Exchange<kVals>& ex, int val) {
  return make4(*reinterpret_cast<const float4*>(&ex.total[val][(threadIdx.x & 7) * 4]));
}
// Sums s (already over the thread's rows) to ex.part, and their joining.
template <int kVals>
__device__ __forceinline__ void sum_part(F4 s, Exchange<kVals>& ex, int val) {
  s = over_rows(s);
  if ((threadIdx.x & 31) < 8)
    *reinterpret_cast<float4*>(&ex.part[threadIdx.x >> 5][val][(threadIdx.x & 7) * 4]) = flat(s);
}
template <int kVals>
__device__ __forceinline__ void sum_join(Exchange<kVals>& ex, int val, int warps) {
  const int lane = threadIdx.x & 31;
  float s = 0.f;
  for (int w = 0; w < warps; ++w) s += ex.part[w][val][lane];
  ex.total[val][lane] = s;
}

constexpr int kThreadsMost = 32 * kMaxWarps;

int stage_param(Ctx* ctx, const float* p, int c, int mem, const char* what, const float** out) {
  return stage_bytes_in(ctx, p, (size_t)c * sizeof(float), sizeof(float), mem, what, out);
}

int stage_params(Ctx* ctx, const zjai_residual_params& in, int c, int mem,
                 zjai_residual_params* out) {
  ZJAI_TRY(stage_param(ctx, in.post_weight, c, mem, "post_weight", &out->post_weight));
  ZJAI_TRY(stage_param(ctx, in.post_bias, c, mem, "post_bias", &out->post_bias));
  ZJAI_TRY(stage_param(ctx, in.scale, c, mem, "scale", &out->scale));
  ZJAI_TRY(stage_param(ctx, in.pre_weight, c, mem, "pre_weight", &out->pre_weight));
  return stage_param(ctx, in.pre_bias, c, mem, "pre_bias", &out->pre_bias);
}

// Rows a thread holds for c channels (0: not held) and the block's warps.
struct Shape {
  int rows, warps, per_sm;
};
Shape shape_of(int c) {
  const int rows = c <= 64 ? 1 : c <= 128 ? 2 : c <= 256 ? 4 : 0;
  const int warps = rows ? (c + 4 * rows - 1) / (4 * rows) : kMaxWarps;
  // blocks that are resident at the register limits of __launch_bounds__
  const int least = rows == 4 ? 1 : 2;
  return {rows, warps, std::max(1, std::min(16, least * kMaxWarps / warps))};
}
// f(std::integral_constant) with the rows held
template <class F>
int by_rows(int rows, F&& f) {
  if (rows == 1) return f(std::integral_constant<int, 1>());
  if (rows == 2) return f(std::integral_constant<int, 2>());
  if (rows == 4) return f(std::integral_constant<int, 4>());
  return f(std::integral_constant<int, 0>());
}
// Four neighbouring positions can be loaded and stored at once: rows of a multiple of four
// positions, maps aligned to four elements and codes to four bytes.
struct VecCheck {
  bool ok;
  explicit VecCheck(int p) : ok(p % 4 == 0) {}
  VecCheck& map(const void* q, size_t es) {
    ok = ok && reinterpret_cast<uintptr_t>(q) % (4 * es) == 0;
    return *this;
  }
};

int check_step(const char* what, int c, int gate_channels, const zjai_residual_params* prm) {
  if (c > kMaxC)
    return fail(ZJAI_UNSUPPORTED, std::string(what) + ": more than 8192 channels");
  if (gate_channels != 0 && gate_channels != 1 && gate_channels != c)
    return fail(ZJAI_INVALID_ARGUMENT, std::string(what) + ": gate_channels must be 0, 1 or c");
  if (!prm || (prm->post_weight != nullptr) != (prm->post_bias != nullptr) ||
      (prm->pre_weight != nullptr) != (prm->pre_bias != nullptr))
    return fail(ZJAI_INVALID_ARGUMENT, std::string(what) + ": a norm needs weight and bias");
  return ZJAI_OK;
}

}  // namespace
}  // namespace zjai
