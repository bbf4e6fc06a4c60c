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

// Rows of the calling thread: row(j) for j < rows(). kRows > 0: held in registers, consecutive
// groups of four per warp; 0: any number, strided over the block. kAll: all rows exist.
template <int kRows, bool kAll = false>
struct Rows {
  int c, first, step, n;
  __device__ __forceinline__ Rows(int c_, int warps) : c(c_) {
    const int wp = threadIdx.x >> 5, rg = (threadIdx.x & 31) >> 3;
    first = wp * 4 * (kRows ? kRows : 1) + rg;
    step = kRows ? 4 : 4 * warps;
    n = kRows ? kRows : (c + step - 1) / step;
  }
  __device__ __forceinline__ int row(int j) const { return first + j * step; }
  __device__ __forceinline__ bool on(int j) const { return kAll || row(j) < c; }
  // a row that exists, to read for one that does not
  __device__ __forceinline__ int param(int j) const { return min(row(j), c - 1); }
  // rows of a warp
  __device__ __forceinline__ int of_warp(int w, int warps) const {
    if (kAll) return 4 * kRows;
    if (kRows) return max(0, min(c - w * 4 * kRows, 4 * kRows));
    const int whole = c / (4 * warps);
    return whole * 4 + max(0, min(4, c - whole * 4 * warps - w * 4));
  }
};
#define FOR_ROWS(j) _Pragma("unroll") for (int j = 0; j < (kRows ? kRows : rows.n); ++j)

// Per warp the sum and the squared deviations from the warp's own mean of v(j), to ex.part at val,
// val + 1.
template <int kRows, bool kAll, class V, class E>
__device__ __forceinline__ void stats_part(const Rows<kRows, kAll>& rows, V&& v, E& ex, int val,
                                           int warps) {
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  F4 s = all(0.f), q = all(0.f);
  FOR_ROWS(j) if (rows.on(j)) s = s + v(j);
  s = over_rows(s);
  const int n = rows.of_warp(wp, warps);
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
    const float m = over_subs(sum) * inv_c;
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i) {
      const int w = i * 4 + sub, n = w < warps ? rows.of_warp(w, warps) : 0;
      if (n) {
        // (whole warps: by a constant)
        const float d = (kAll ? s[i] * (1.f / (4 * kRows)) : __fdividef(s[i], (float)n)) - m;
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

// Staged loads (rows held, vector accesses): a thread copies what it will itself read of the next
// tile to its own places in shared memory (cp.async, no thread waits for another) while it works on
// the current one. A place is four positions of a row, of kBytes.
template <int kBytes>
__device__ __forceinline__ void stage_copy(char* dst, const void* src, bool on) {
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(on ? 16 : 0)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(src), "n"(kBytes),
                 "r"(on ? kBytes : 0)
                 : "memory");
}
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
template <class T>
__device__ __forceinline__ F4 staged4(const char* src) {
  if constexpr (sizeof(T) == 4)
    return make4(*reinterpret_cast<const float4*>(src));
  else
    return halves4<T>(*reinterpret_cast<const uint2*>(src));
}
// The rows of the calling thread in a picture: their offsets from the picture's first element, with
// the lane's four positions, and of their exponents from the picture's first (held rows: 32 bits
// do). kWhole: a multiple of 16 channels and of 32 positions, every row and position there.
constexpr int kStagedRows = 4;
template <bool kWhole>
struct StagedRows {
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

// How c channels at p positions are taken. staged: rows held and copied ahead, where vector accesses
// are possible; else kRows rows of a thread held in registers, or (0) read again. Sixteen warps an
// SM are resident at the registers that __launch_bounds__ leaves, so blocks of few warps come in
// numbers.
struct Shape {
  bool staged, whole;
  int rows, warps, per_sm;
};
Shape shape_of(int c, int p, bool vec, bool backward) {
  // held rows are addressed by 32-bit offsets from their picture
  const bool held = c <= kHeldC && (long long)c * p < (1LL << 32) - 64;
  // without vector accesses the backward pass takes two rows a thread where the warps allow it
  const int rows = !held ? 0 : !vec && backward && c <= kHeldC / 2 ? 2 : kStagedRows;
  const int warps = rows ? (c + 4 * rows - 1) / (4 * rows) : kMaxWarps;
  return {held && vec, c % (4 * kStagedRows) == 0 && p % kTapeGroup == 0, rows, warps,
          kMaxWarps / warps};
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
