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
constexpr int kStagedRows = 4;  // rows a thread holds

// sigmoid(g) and sigmoid(g) (1 - sigmoid(g)), an even function of g: with a = exp(-|g|) and
// r = 1 / (1 + a), sigmoid is r or a r and the product a r^2, nothing by cancellation and both finite
// for every g but NaN.
__device__ __forceinline__ void sigmoid2(float g, float* s, float* slope) {
  const float a = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + a), ar = a * r;
  *s = g >= 0.f ? r : ar;
  *slope = ar * r;
}
__device__ __forceinline__ void sigmoid4(F4 g, F4* s, F4* slope) {
  sigmoid2(g.a.x, &s->a.x, &slope->a.x);
  sigmoid2(g.a.y, &s->a.y, &slope->a.y);
  sigmoid2(g.b.x, &s->b.x, &slope->b.x);
  sigmoid2(g.b.y, &s->b.y, &slope->b.y);
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
template <int kVals, int kTotals>
struct Exchange {
  float part[kVals][kMaxWarps][32], total[kTotals][32];
};

// Rows of the calling thread: row(j) for j < n, a warp's consecutive groups of four. kRows > 0: as
// many, held; 0: as many as c takes. kAll: all rows exist. The same rows to the same warps either way
// (up to 256 channels), so that results do not depend on alignment.
template <int kRows, bool kAll = false>
struct Rows {
  int c, first, n;
  __device__ __forceinline__ Rows(int c_, int warps) : c(c_) {
    n = kRows ? kRows : max(kStagedRows, (c + 4 * warps - 1) / (4 * warps));
    first = (threadIdx.x >> 5) * 4 * n + ((threadIdx.x & 31) >> 3);
  }
  __device__ __forceinline__ int row(int j) const { return first + j * 4; }
  __device__ __forceinline__ bool on(int j) const { return kAll || row(j) < c; }
  // a row that exists, to read for one that does not
  __device__ __forceinline__ int param(int j) const { return min(row(j), c - 1); }
  // rows of a warp
  __device__ __forceinline__ int of_warp(int w) const {
    return kAll ? 4 * kRows : max(0, min(c - w * 4 * n, 4 * n));
  }
};
#define FOR_ROWS(j) _Pragma("unroll") for (int j = 0; j < (kRows ? kRows : rows.n); ++j)

// Per warp the sum and the squared deviations from the warp's own mean of v(j), to ex.part at val,
// val + 1.
template <int kRows, bool kAll, class V, class E>
__device__ __forceinline__ void stats_part(const Rows<kRows, kAll>& rows, V&& v, E& ex, int val) {
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  F4 s = all(0.f), q = all(0.f);
  FOR_ROWS(j) if (rows.on(j)) s = s + v(j);
  s = over_rows(s);
  const int n = rows.of_warp(wp);
  const F4 nm = s * all(kAll ? -1.f / (4 * kRows) : n ? __fdividef(-1.f, (float)n) : 0.f);
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
template <int kRows, bool kAll, class E>
__device__ __forceinline__ void stats_join(const Rows<kRows, kAll>& rows, E& ex, int val,
                                           float inv_c, int warps, int nth, int of) {
  by_position(nth, of, [&](int pos, int sub) {
    float s[kMaxWarps / 4], sum = 0.f, q = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i) {
      const int w = i * 4 + sub;
      s[i] = w < warps ? ex.part[val][w][pos] : 0.f;
      sum += s[i];
    }
    // products rounded on their own: the same bits wherever this is compiled in
    const float m = __fmul_rn(over_subs(sum), inv_c);
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i) {
      const int w = i * 4 + sub, n = w < warps ? rows.of_warp(w) : 0;
      if (n) {
        // (whole warps: by a constant)
        const float d = __fsub_rn(kAll ? __fmul_rn(s[i], 1.f / (4 * kRows)) : __fdividef(s[i], (float)n), m);
        q = __fadd_rn(q, fmaf(__fmul_rn((float)n, d), d, ex.part[val + 1][w][pos]));
      }
    }
    q = over_subs(q);
    if (sub == 0) {
      ex.total[val][pos] = -m;
      ex.total[val + 1][pos] = rsqrtf(fmaf(q, inv_c, kEps));
    }
  });
}
template <class E>
__device__ __forceinline__ F4 total4(const E& ex, int val) {
  return make4(*reinterpret_cast<const float4*>(&ex.total[val][(threadIdx.x & 7) * 4]));
}
// Sums over the warps of ex.part at val, times k, to ex.total at to.
template <class E>
__device__ __forceinline__ void sum_join(E& ex, int val, int to, float k, int warps, int nth,
                                         int of) {
  by_position(nth, of, [&](int pos, int sub) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i)
      if (i * 4 + sub < warps) s += ex.part[val][i * 4 + sub][pos];
    s = over_subs(s);
    if (sub == 0) ex.total[to][pos] = s * k;
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

// The tiles of a block, one after the other: picture and group of positions, without a division.
struct Tiles {
  int img, g, groups, step_img, step_g;
  long long left;  // tiles from the current one on, of the whole grid
  __device__ __forceinline__ Tiles(long long tiles, int groups_) : groups(groups_) {
    img = (int)(blockIdx.x / (unsigned)groups);
    g = (int)(blockIdx.x - (unsigned)img * groups);
    step_img = (int)(gridDim.x / (unsigned)groups);
    step_g = (int)(gridDim.x - (unsigned)step_img * groups);
    left = tiles - blockIdx.x;
  }
  __device__ __forceinline__ bool on() const { return left > 0; }
  __device__ __forceinline__ void next() {
    left -= gridDim.x;
    img += step_img;
    g += step_g;
    if (g >= groups) g -= groups, ++img;
  }
};

// Staged loads (rows held): a thread copies what it will itself read of the next tile to its own
// places in shared memory (cp.async, no thread waits for another) while it works on the current one.
// A place holds four positions of a row. By alignment:
//   kWholeTiles: a multiple of 16 channels and of 32 positions, all aligned: no bounds to check;
//   kAligned: rows of a multiple of four positions on aligned bases: all four in the row or behind;
//   kAnywhere: rows start anywhere, on bases of whole words: f32 comes one by one, f16 and bf16 as
//     the three words and codes as the two words that hold the four, shifted into place when read.
enum { kWholeTiles, kAligned, kAnywhere };
// the first `bytes` (1 to 4) of an aligned word, zeros behind them
__device__ __forceinline__ void stage_copy_some(char* dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void stage_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kNewer>
__device__ __forceinline__ void stage_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kNewer) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void stage_copy_all(char* dst, const void* src, bool on) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(on ? 16 : 0)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(src), "n"(kBytes),
                 "r"(on ? kBytes : 0)
                 : "memory");
}
// Places of E (float, __half, __nv_bfloat16, or int8_t for codes): bytes, copies and reads. on: the
// row exists; nv: how many of the four positions lie in it; end: behind the tensor's last element.
template <int kMode, class E>
struct Place {
  static constexpr int kSize = (int)sizeof(E);
  static constexpr int kBytes =
      kMode != kAnywhere || kSize == 4 ? 4 * kSize : kSize == 2 ? 16 : 8;
  static __device__ __forceinline__ void copy(char* dst, const E* src, bool on, int nv,
                                              const E* end) {
    if constexpr (kMode != kAnywhere) {
      stage_copy_all<4 * kSize>(dst, src, kMode == kWholeTiles || (on && nv > 0));
    } else if constexpr (kSize == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) stage_copy_some(dst + 4 * i, src + i, on && i < nv ? 4 : 0);
    } else {
      const char* a = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)3);
      const long long left = reinterpret_cast<const char*>(end) - a;
      const int l = on ? (int)min(left, 12LL) : 0;
#pragma unroll
      for (int j = 0; j < (kSize == 2 ? 3 : 2); ++j)
        stage_copy_some(dst + 4 * j, a + 4 * j, max(0, min(4, l - 4 * j)));
    }
  }
  // two words (halves) or one (codes) in place; src: where it was copied from
  static __device__ __forceinline__ uint2 words(const char* q, const E* src, int nv) {
    if constexpr (kMode != kAnywhere) {
      if constexpr (kSize == 2) return *reinterpret_cast<const uint2*>(q);
      else return make_uint2(*reinterpret_cast<const uint32_t*>(q), 0u);
    } else {
      const uint32_t sh = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 3) * 8;
      if constexpr (kSize == 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(q);
        const uint32_t lo = nv >= 2 ? ~0u : nv == 1 ? 0xffffu : 0u;
        const uint32_t hi = nv >= 4 ? ~0u : nv == 3 ? 0xffffu : 0u;
        return make_uint2(__funnelshift_r(w.x, w.y, sh) & lo, __funnelshift_r(w.y, w.z, sh) & hi);
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(q);
        const uint32_t in = nv >= 4 ? ~0u : nv <= 0 ? 0u : ~0u >> (32 - 8 * nv);
        return make_uint2(__funnelshift_r(w.x, w.y, sh) & in, 0u);
      }
    }
  }
  static __device__ __forceinline__ F4 get(const char* q, const E* src, int nv) {
    if constexpr (kSize == 4)
      return make4(*reinterpret_cast<const float4*>(q));
    else
      return halves4<E>(words(q, src, nv));
  }
};
// four positions of a row to q, nv of them in the row
template <int kMode, class T>
__device__ __forceinline__ void staged_store(T* q, F4 v, bool on, int nv) {
  if constexpr (kMode == kWholeTiles) {
    store4_in(q, v);
  } else if constexpr (kMode == kAligned) {
    if (on && nv > 0) store4_in(q, v);
  } else {
    if (on) store4<false>(q, 0, nv, v);
  }
}

// The rows of the calling thread in a picture: their offsets from the picture's first element, with
// the lane's four positions, and of their exponents from the picture's first (held rows: 32 bits
// do).
template <int kMode>
struct StagedRows {
  static constexpr bool kWhole = kMode == kWholeTiles;
  uint32_t e0, x0, e4, x4;
  int ch0, c;
  __device__ __forceinline__ StagedRows(int c_, int p, int groups) : c(c_) {
    const int lane = threadIdx.x & 31;
    ch0 = (threadIdx.x >> 5) * 4 * kStagedRows + (lane >> 3);
    e0 = (uint32_t)ch0 * (uint32_t)p + (lane & 7) * 4;
    x0 = (uint32_t)ch0 * (uint32_t)groups;
    e4 = 4u * (uint32_t)p;
    x4 = 4u * (uint32_t)groups;
  }
  __device__ __forceinline__ uint32_t e(int j) const { return e0 + j * e4; }
  __device__ __forceinline__ uint32_t x(int j) const { return x0 + j * x4; }
  __device__ __forceinline__ bool on(int j) const { return kWhole || ch0 + 4 * j < c; }
  // a channel that exists, for the parameters
  __device__ __forceinline__ int ch(int j) const {
    return kWhole ? ch0 + 4 * j : min(ch0 + 4 * j, c - 1);
  }
};

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

// How c channels at p positions are taken: staged (rows held) in a mode, or read again for each
// pass (mode -1). Sixteen warps an SM are resident at the registers that __launch_bounds__ leaves,
// so blocks of few warps come in numbers.
struct Shape {
  int mode, warps, per_sm;
};
Shape shape_of(int c, int p, bool vec, bool words) {
  // held rows are addressed by 32-bit offsets from their picture
  const bool held = c <= kHeldC && (long long)c * p < (1LL << 32) - 64;
  const int mode = !held                                                  ? -1
                   : vec && c % (4 * kStagedRows) == 0 && p % kTapeGroup == 0 ? kWholeTiles
                   : vec                                                  ? kAligned
                   : words                                                ? kAnywhere
                                                                          : -1;
  const int warps = std::min(kMaxWarps, (c + 4 * kStagedRows - 1) / (4 * kStagedRows));
  return {mode, warps, kMaxWarps / warps};
}
// f(std::integral_constant) with a staged mode
template <class F>
auto by_mode(int mode, F&& f) {
  if (mode == kWholeTiles) return f(std::integral_constant<int, kWholeTiles>());
  if (mode == kAligned) return f(std::integral_constant<int, kAligned>());
  return f(std::integral_constant<int, kAnywhere>());
}
// ok: four neighbouring positions can be loaded and stored at once (rows of a multiple of four
// positions, maps aligned to four elements and codes to four bytes); words: all on whole words.
struct VecCheck {
  bool ok, words = true;
  explicit VecCheck(int p) : ok(p % 4 == 0) {}
  VecCheck& map(const void* q, size_t es) {
    ok = ok && reinterpret_cast<uintptr_t>(q) % (4 * es) == 0;
    words = words && reinterpret_cast<uintptr_t>(q) % 4 == 0;
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
