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
// shared-memory partials, gathered by four lanes each. Statistics: a mean and sum of squared
// deviations per warp, joined by their exact update formula (sums of squares would cancel).
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

// Sum over the four rows of a warp (lanes with the same positions), to all of them.
__device__ __forceinline__ F4 over_rows(F4 v) {
  float f[4] = {v.a.x, v.a.y, v.b.x, v.b.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] += __shfl_xor_sync(0xffffffffu, f[i], 8);
    f[i] += __shfl_xor_sync(0xffffffffu, f[i], 16);
  }
  return {make_float2(f[0], f[1]), make_float2(f[2], f[3])};
}
// The same sum, one position a lane, to part[position]: halves of the positions are exchanged, so
// that three shuffles do for four values.
__device__ __forceinline__ void rows_to_part(F4 v, float* part) {
  const int lane = threadIdx.x & 31;
  const bool b3 = lane & 8, b4 = lane & 16;
  float x = b3 ? v.b.x : v.a.x, y = b3 ? v.b.y : v.a.y;
  x += __shfl_xor_sync(0xffffffffu, b3 ? v.a.x : v.b.x, 8);
  y += __shfl_xor_sync(0xffffffffu, b3 ? v.a.y : v.b.y, 8);
  float t = b4 ? y : x;
  t += __shfl_xor_sync(0xffffffffu, b4 ? x : y, 16);
  part[(lane & 7) * 4 + (b3 ? 2 : 0) + (b4 ? 1 : 0)] = t;
}

// The block's partial sums per warp and position, and their totals.
template <int kVals>
struct Exchange {
  float part[kVals][kMaxWarps][32], total[kVals][32];
};

// Rows of the calling thread: row(j) for j < rows(). kRows > 0: held in registers, consecutive
// groups of four per warp; 0: any number, strided over the block.
template <int kRows>
struct Rows {
  int c, first, step, n;
  __device__ __forceinline__ Rows(int c_, int warps) : c(c_) {
    const int wp = threadIdx.x >> 5, rg = (threadIdx.x & 31) >> 3;
    first = wp * 4 * (kRows ? kRows : 1) + rg;
    step = kRows ? 4 : 4 * warps;
    n = kRows ? kRows : (c + step - 1) / step;
  }
  __device__ __forceinline__ int row(int j) const { return first + j * step; }
  __device__ __forceinline__ bool on(int j) const { return row(j) < c; }
  // a row that exists, to read for one that does not
  __device__ __forceinline__ int param(int j) const { return min(row(j), c - 1); }
  // rows of a warp
  __device__ __forceinline__ int of_warp(int w, int warps) const {
    if (kRows) return max(0, min(c - w * 4 * kRows, 4 * kRows));
    const int whole = c / (4 * warps);
    return whole * 4 + max(0, min(4, c - whole * 4 * warps - w * 4));
  }
};
#define FOR_ROWS(j) _Pragma("unroll") for (int j = 0; j < (kRows ? kRows : rows.n); ++j)

// Per warp the sum and the squared deviations from the warp's own mean of v(j), to ex.part at val,
// val + 1.
template <int kRows, int kVals, class V>
__device__ __forceinline__ void stats_part(const Rows<kRows>& rows, V&& v, Exchange<kVals>& ex,
                                           int val, int warps) {
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  F4 s = all(0.f), q = all(0.f);
  FOR_ROWS(j) if (rows.on(j)) s = s + v(j);
  s = over_rows(s);
  const int n = rows.of_warp(wp, warps);
  const F4 nm = s * all(n ? __fdividef(-1.f, (float)n) : 0.f);
  FOR_ROWS(j) if (rows.on(j)) {
    const F4 d = v(j) + nm;
    q = fma4(d, d, q);
  }
  if (lane < 8) *reinterpret_cast<float4*>(&ex.part[val][wp][lane * 4]) = flat(s);
  rows_to_part(q, ex.part[val + 1][wp]);
}
// A quarter of the positions per warp (of `of` that call, the `nth`): four lanes a position, each
// with every fourth warp's partials.
template <class F>
__device__ __forceinline__ void by_position(int nth, int of, F&& f) {
  const int lane = threadIdx.x & 31;
  for (int b = nth; b < 4; b += of) f(b * 8 + (lane & 7), lane >> 3);
}
__device__ __forceinline__ float over_subs(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
// Joined: ex.total at val, val + 1 the negated mean and 1 / sigma. Partials' means are joined by
// M2 = sum of M2_w + n_w (mean_w - mean)^2.
template <int kRows, int kVals>
__device__ __forceinline__ void stats_join(const Rows<kRows>& rows, Exchange<kVals>& ex, int val,
                                           float inv_c, int warps, int nth, int of) {
  by_position(nth, of, [&](int pos, int sub) {
    float s[kMaxWarps / 4], sum = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i) {
      const int w = i * 4 + sub;
      s[i] = w < warps ? ex.part[val][w][pos] : 0.f;
      sum += s[i];
    }
    const float m = over_subs(sum) * inv_c;
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i) {
      const int w = i * 4 + sub, n = w < warps ? rows.of_warp(w, warps) : 0;
      if (n) {
        const float d = __fdividef(s[i], (float)n) - m;
        q += fmaf((float)n * d, d, ex.part[val + 1][w][pos]);
      }
    }
    q = over_subs(q);
    if (sub == 0) {
      ex.total[val][pos] = -m;
      ex.total[val + 1][pos] = rsqrtf(fmaf(q, inv_c, kEps));
    }
  });
}
template <int kVals>
__device__ __forceinline__ F4 total4(const Exchange<kVals>& ex, int val) {
  return make4(*reinterpret_cast<const float4*>(&ex.total[val][(threadIdx.x & 7) * 4]));
}
// Sums over the warps of ex.part at val, times k.
template <int kVals>
__device__ __forceinline__ void sum_join(Exchange<kVals>& ex, int val, float k, int warps, int nth,
                                         int of) {
  by_position(nth, of, [&](int pos, int sub) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i)
      if (i * 4 + sub < warps) s += ex.part[val][i * 4 + sub][pos];
    s = over_subs(s);
    if (sub == 0) ex.total[val][pos] = s * k;
  });
}

// The parameters of a channel in all four positions: doubled in shared memory where rows are held
// (up to kHeldC channels), else from global memory. Absent ones are those of the identity.
constexpr int kHeldC = 256;
enum { kPostW, kPostB, kScale, kPreW, kPreB, kParams };
template <int kRows>
struct Params {
  float2 v[kRows ? kParams : 1][kRows ? kHeldC : 1];
  static __device__ __forceinline__ const float* of(const zjai_residual_params& p, int k) {
    return k == kPostW ? p.post_weight : k == kPostB ? p.post_bias : k == kScale ? p.scale
           : k == kPreW ? p.pre_weight : p.pre_bias;
  }
  static __device__ __forceinline__ float one(const zjai_residual_params& p, int k, int ch) {
    const float* q = of(p, k);
    return q ? __ldg(q + ch) : (k == kPostB || k == kPreB ? 0.f : 1.f);
  }
  __device__ __forceinline__ void load(const zjai_residual_params& p, int c) {
    if (kRows)
      for (int i = threadIdx.x; i < kParams * c; i += blockDim.x) {
        const float x = one(p, i / c, i % c);
        v[i / c][i % c] = make_float2(x, x);
      }
  }
  __device__ __forceinline__ F4 get(const zjai_residual_params& p, int k, int ch) const {
    if (!kRows) return all(one(p, k, ch));
    const float2 x = v[k][ch];
    return {x, x};
  }
};

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

// Rows a thread holds for c channels (0: not held) and the block's warps. Sixteen warps an SM are
// resident at the registers that __launch_bounds__ leaves, so blocks of few warps come in numbers.
struct Shape {
  int rows, warps, per_sm;
};
Shape shape_of(int c, bool backward) {
  // the backward pass holds twice as much a row: two rows a thread where the warps allow it
  const int rows = c > kHeldC ? 0 : backward && c <= kHeldC / 2 ? 2 : 4;
  const int warps = rows ? (c + 4 * rows - 1) / (4 * rows) : kMaxWarps;
  return {rows, warps, kMaxWarps / warps};
}
// f(std::integral_constant) with the rows held
template <class F>
int by_rows(int rows, F&& f) {
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
