// The residual step of a block with its norms, gate and scale in one kernel, and its backward pass
// (zjai_gated_residual_norm, zjai_gated_residual_norm_backward).
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
#include <algorithm>
#include <type_traits>

#include "train.h"

namespace zjai {
namespace {

constexpr float kEps = 1e-5f;
constexpr int kMaxC = 8192;  // the parameter sums of a block sit in shared memory, 20 B a channel
constexpr int kMaxWarps = 16;
constexpr int kVecs = 4;  // positions of a lane

template <class T>
struct FwdArgs {
  const T *x, *f, *gate;
  int gate_c, c, p;
  long long tiles;
  zjai_residual_params prm;
  T *y, *z;
  zjai_residual_tapes tp;
};

template <class T>
struct BwdArgs {
  const T *dy, *dz, *f, *gate, *y;
  zjai_residual_tapes tp;  // taped f, gate, y
  int gate_c, c, p;
  long long tiles;
  zjai_residual_params prm;
  T *dx, *df, *dgate;
  float* sums;  // [blocks][5][c]: scale, post_weight, post_bias, pre_weight, pre_bias
};

// Four neighbouring positions, as two packed pairs.
struct F4 {
  float2 a, b;
};
__device__ __forceinline__ F4 operator+(F4 x, F4 y) {
  return {__fadd2_rn(x.a, y.a), __fadd2_rn(x.b, y.b)};
}
__device__ __forceinline__ F4 operator*(F4 x, F4 y) {
  return {__fmul2_rn(x.a, y.a), __fmul2_rn(x.b, y.b)};
}
__device__ __forceinline__ F4 fma4(F4 x, F4 y, F4 z) {
  return {__ffma2_rn(x.a, y.a, z.a), __ffma2_rn(x.b, y.b, z.b)};
}
__device__ __forceinline__ F4 all(float v) {
  return {make_float2(v, v), make_float2(v, v)};
}
__device__ __forceinline__ F4 operator-(F4 x) {
  return {make_float2(-x.a.x, -x.a.y), make_float2(-x.b.x, -x.b.y)};
}
__device__ __forceinline__ F4 operator-(F4 x, F4 y) { return x + (-y); }
__device__ __forceinline__ F4 make4(float4 v) {
  return {make_float2(v.x, v.y), make_float2(v.z, v.w)};
}
__device__ __forceinline__ float4 flat(F4 v) { return make_float4(v.a.x, v.a.y, v.b.x, v.b.y); }

// four positions from row pointer + at, zeros behind the row's end; kVec: all in or out, aligned
template <bool kVec, class T>
__device__ __forceinline__ F4 load4(const T* row, int at, int p) {
  if constexpr (kVec) {
    if (at >= p) return all(0.f);
    if constexpr (sizeof(T) == 4) {
      return make4(__ldg(reinterpret_cast<const float4*>(row + at)));
    } else {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + at));
      if constexpr (std::is_same<T, __half>::value)
        return {__half22float2(reinterpret_cast<const __half2&>(w.x)),
                __half22float2(reinterpret_cast<const __half2&>(w.y))};
      else
        return {make_float2(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u)),
                make_float2(__uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u))};
    }
  } else {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = at + i < p ? to_f32(row[at + i]) : 0.f;
    return {make_float2(v[0], v[1]), make_float2(v[2], v[3])};
  }
}
template <bool kVec, class T>
__device__ __forceinline__ void store4(T* row, int at, int p, F4 v) {
  if constexpr (kVec) {
    if (at >= p) return;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row + at) = flat(v);
    } else {
      uint2 w;
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 x = __float22half2_rn(v.a), y = __float22half2_rn(v.b);
        w = make_uint2(reinterpret_cast<const uint32_t&>(x), reinterpret_cast<const uint32_t&>(y));
      } else {
        const __nv_bfloat162 x = __float22bfloat162_rn(v.a), y = __float22bfloat162_rn(v.b);
        w = make_uint2(reinterpret_cast<const uint32_t&>(x), reinterpret_cast<const uint32_t&>(y));
      }
      *reinterpret_cast<uint2*>(row + at) = w;
    }
  } else {
    const float f[4] = {v.a.x, v.a.y, v.b.x, v.b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < p) row[at + i] = from_f32<T>(f[i]);
  }
}
// codes of four positions as a word, and back to values
template <bool kVec>
__device__ __forceinline__ uint32_t load_codes(const int8_t* row, int at, int p) {
  if constexpr (kVec) return at < p ? __ldg(reinterpret_cast<const uint32_t*>(row + at)) : 0u;
  uint32_t w = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < p) w |= (uint32_t)(uint8_t)__ldg(row + at + i) << (8 * i);
  return w;
}
__device__ __forceinline__ F4 taped4(uint32_t codes, int e) {
  const uint32_t w = codes ^ 0x80808080u;
  const F4 off = all(-8388736.f);  // see tape_value
  const F4 v = {make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)),
                            __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441))),
                make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)),
                            __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)))};
  return (v + off) * all(tape_scale(e));
}

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

// Hold four positions of a row (zeros behind its end) as part of a tape's group; the row's eight
// lanes call together (`on`: the row exists).
template <bool kVec>
__device__ __forceinline__ void tape_store4(const zjai_tape& t, long long row, int groups, int g,
                                            int at, int p, F4 v, bool on) {
  const uint32_t b[4] = {__float_as_uint(v.a.x), __float_as_uint(v.a.y), __float_as_uint(v.b.x),
                         __float_as_uint(v.b.y)};
  uint32_t m = max(max(b[0] & 0x7fffffffu, b[1] & 0x7fffffffu),
                   max(b[2] & 0x7fffffffu, b[3] & 0x7fffffffu));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (!on) return;
  const int e = tape_exp(m);
  uint32_t w;
  // only the largest 1 / 128 of magnitudes can round to 128, and only a marked group has no codes
  if ((m & 0x7fffffu) < 0x7f0000u && m < 0x7f800000u) {
    const F4 c = fma4(v, all(tape_inv_scale(e)), all(12582912.f));
    w = __byte_perm(__byte_perm(__float_as_uint(c.a.x), __float_as_uint(c.a.y), 0x0040),
                    __byte_perm(__float_as_uint(c.b.x), __float_as_uint(c.b.y), 0x0040), 0x5410);
  } else {
    w = 0u;
    if (e != kTapeNan) {
      const float inv = tape_inv_scale(e);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w |= (tape_code_bits(__uint_as_float(b[i]), inv) & 0xffu) << (8 * i);
    }
  }
  int8_t* codes = t.codes + row * p;
  if constexpr (kVec) {
    if (at < p) *reinterpret_cast<uint32_t*>(codes + at) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < p) codes[at + i] = (int8_t)(w >> (8 * i) & 0xffu);
  }
  if ((threadIdx.x & 7) == 0) t.exps[row * groups + g] = (int8_t)e;
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

// threads a block may have, and blocks an SM holds of the largest
constexpr int kThreadsMost = 32 * kMaxWarps;
template <int kRows>
constexpr int blocks_least() {
  return kRows == 4 ? 1 : 2;
}

// value of positions behind the row's end set to zero
template <bool kVec>
__device__ __forceinline__ F4 clip4(F4 v, int at, int p) {
  if (kVec) return at < p ? v : all(0.f);
  return {make_float2(at < p ? v.a.x : 0.f, at + 1 < p ? v.a.y : 0.f),
          make_float2(at + 2 < p ? v.b.x : 0.f, at + 3 < p ? v.b.y : 0.f)};
}
__device__ __forceinline__ float sum4(F4 v) {
  const float2 t = __fadd2_rn(v.a, v.b);
  return t.x + t.y;
}

template <int kRows, bool kVec, class T>
__global__ void __launch_bounds__(kThreadsMost, blocks_least<kRows>())
    residual_norm_kernel(const FwdArgs<T> a) {
  __shared__ Exchange<2> ex;
  const int warps = blockDim.x >> 5, wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Rows<kRows> rows(a.c, warps);
  constexpr int kHeld = kRows ? kRows : 1;
  const int groups = (int)tape_groups(a.p);
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, per_row = a.gate_c > 1;
  for (long long tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const long long img = tile / groups, base = img * a.c;
    const int g = (int)(tile - img * groups), at = g * kTapeGroup + (lane & 7) * kVecs;
    F4 f[kHeld], x[kHeld], q[kHeld];  // branch, input (then y), gate logits
    auto load = [&](const T* v, int j) {
      return rows.on(j) ? load4<kVec>(v + (base + rows.row(j)) * a.p, at, a.p) : all(0.f);
    };
    if (kRows) {
      FOR_ROWS(j) f[j % kHeld] = load(a.f, j);
      FOR_ROWS(j) x[j % kHeld] = load(a.x, j);
      if (per_row) FOR_ROWS(j) q[j % kHeld] = load(a.gate, j);
    }
    auto f_of = [&](int j) { return kRows ? f[j % kHeld] : load(a.f, j); };
    auto gate_of = [&](int j) { return kRows ? q[j % kHeld] : load(a.gate, j); };
    F4 gate1 = all(0.f), sg1 = all(1.f), unused;
    if (a.gate_c == 1) {
      gate1 = load4<kVec>(a.gate + img * a.p, at, a.p);
      sigmoid4(gate1, &sg1, &unused);
    }
    F4 m = all(0.f), r = all(1.f);
    auto exchange = [&](auto v) {
      stats_part(rows, v, ex, 0);
      __syncthreads();
      if (wp == 0) stats_join<kRows>(ex, 0, a.c, warps);
      __syncthreads();
      m = total4(ex, 0);
      r = total4(ex, 1);
    };
    if (post) exchange(f_of);
    const F4 m1 = m, r1 = r;
    auto y_of = [&](int j) {
      const int ch = rows.param(j);
      F4 u = f_of(j), s = sg1;
      if (post)
        u = fma4((u - m1) * r1, all(__ldg(a.prm.post_weight + ch)), all(__ldg(a.prm.post_bias + ch)));
      if (per_row) sigmoid4(gate_of(j), &s, &unused);
      if (a.prm.scale) s = s * all(__ldg(a.prm.scale + ch));
      return fma4(s, u, kRows ? x[j % kHeld] : load(a.x, j));
    };
    // y and the tapes of f, gate and y (whole warps call)
    auto emit = [&](int j, F4 y) {
      const bool on = rows.on(j);
      const long long row = base + rows.row(j);
      if (on) store4<kVec>(a.y + row * a.p, at, a.p, y);
      if (a.tp.f.codes) tape_store4<kVec>(a.tp.f, row, groups, g, at, a.p, f_of(j), on);
      if (per_row && a.tp.gate.codes)
        tape_store4<kVec>(a.tp.gate, row, groups, g, at, a.p, gate_of(j), on);
      if (a.tp.y.codes)
        tape_store4<kVec>(a.tp.y, row, groups, g, at, a.p, clip4<kVec>(y, at, a.p), on);
    };
    if (a.gate_c == 1 && a.tp.gate.codes && wp == 0)
      tape_store4<kVec>(a.tp.gate, img, groups, g, at, a.p, gate1, lane < 8);
    if (kRows) {
      FOR_ROWS(j) {
        const F4 y = y_of(j);
        emit(j, y);
        x[j % kHeld] = y;
      }
    }
    auto done_y = [&](int j) { return kRows ? x[j % kHeld] : y_of(j); };
    if (pre) exchange(done_y);
    if (kRows && !pre) continue;
    FOR_ROWS(j) {
      const F4 y = done_y(j);
      if (!kRows) emit(j, y);
      if (!pre) continue;
      const int ch = rows.param(j);
      const F4 z = fma4((y - m) * r, all(__ldg(a.prm.pre_weight + ch)), all(__ldg(a.prm.pre_bias + ch)));
      const long long row = base + rows.row(j);
      if (rows.on(j)) store4<kVec>(a.z + row * a.p, at, a.p, z);
      if (a.tp.z.codes)
        tape_store4<kVec>(a.tp.z, row, groups, g, at, a.p, clip4<kVec>(z, at, a.p), rows.on(j));
    }
  }
}

// A row's four positions of a kept map: codes and exponent of a tape, or values.
template <bool kTaped, bool kVec, class T>
struct Kept {
  F4 v;
  __device__ __forceinline__ void load(const T* map, const zjai_tape&, long long row, int, int,
                                       int at, int p) {
    v = load4<kVec>(map + row * p, at, p);
  }
  __device__ __forceinline__ F4 get() const { return v; }
};
template <bool kVec, class T>
struct Kept<true, kVec, T> {
  uint32_t w;
  int e;
  __device__ __forceinline__ void load(const T*, const zjai_tape& t, long long row, int groups,
                                       int g, int at, int p) {
    w = load_codes<kVec>(t.codes + row * p, at, p);
    e = __ldg(t.exps + row * groups + g);
  }
  __device__ __forceinline__ F4 get() const { return taped4(w, e); }
};

// The parameter gradients are summed over a block's tiles (in registers, or per channel in shared
// memory where rows are not held) and written out per block.
template <int kRows, bool kTaped, bool kVec, class T>
__global__ void __launch_bounds__(kThreadsMost, 1)
    residual_norm_bwd_kernel(const BwdArgs<T> a) {
  __shared__ Exchange<4> ex;
  extern __shared__ float acc_c[];  // [5][c] where rows are not held
  const int warps = blockDim.x >> 5, wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Rows<kRows> rows(a.c, warps);
  constexpr int kHeld = kRows ? kRows : 1;
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, per_row = a.gate_c > 1;
  const bool need_f = post || a.gate_c || a.prm.scale;
  const int second = warps > 1 ? 1 : 0;  // warp that joins the second of two sums
  float acc[kHeld][5];
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
#pragma unroll
    for (int i = 0; i < 5; ++i) acc[j][i] = 0.f;
  if (!kRows) {
    for (int i = threadIdx.x; i < 5 * a.c; i += blockDim.x) acc_c[i] = 0.f;
    __syncthreads();
  }
  for (long long tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const long long img = tile / groups, base = img * a.c;
    const int g = (int)(tile - img * groups), at = g * kTapeGroup + (lane & 7) * kVecs;
    using K = Kept<kTaped, kVec, T>;
    F4 dy[kHeld], dz[kHeld];
    K f[kHeld], y[kHeld], q[kHeld];
    auto grad = [&](const T* v, int j) {
      return rows.on(j) ? load4<kVec>(v + (base + rows.row(j)) * a.p, at, a.p) : all(0.f);
    };
    auto kept = [&](const T* v, const zjai_tape& t, int j) {
      K k;
      k.load(v, t, base + rows.param(j), groups, g, at, a.p);
      return k;
    };
    if (kRows) {
      if (pre) FOR_ROWS(j) y[j % kHeld] = kept(a.y, a.tp.y, j);
      if (need_f) FOR_ROWS(j) f[j % kHeld] = kept(a.f, a.tp.f, j);
      if (pre) FOR_ROWS(j) dz[j % kHeld] = grad(a.dz, j);
      FOR_ROWS(j) dy[j % kHeld] = grad(a.dy, j);
      if (per_row) FOR_ROWS(j) q[j % kHeld] = kept(a.gate, a.tp.gate, j);
    }
    auto f_of = [&](int j) { return kRows ? f[j % kHeld].get() : kept(a.f, a.tp.f, j).get(); };
    auto y_of = [&](int j) { return kRows ? y[j % kHeld].get() : kept(a.y, a.tp.y, j).get(); };
    auto gate_of = [&](int j) {
      return kRows ? q[j % kHeld].get() : kept(a.gate, a.tp.gate, j).get();
    };
    auto dz_of = [&](int j) { return kRows ? dz[j % kHeld] : grad(a.dz, j); };
    F4 sg1 = all(1.f), os1 = all(0.f);
    if (a.gate_c == 1) {
      K k;
      k.load(a.gate, a.tp.gate, img, groups, g, at, a.p);
      sigmoid4(k.get(), &sg1, &os1);
    }
    F4 m1 = all(0.f), r1 = all(1.f), m2 = all(0.f), r2 = all(1.f), am = all(0.f), ay = all(0.f);
    if (post) stats_part(rows, f_of, ex, 0);
    if (pre) stats_part(rows, y_of, ex, 2);
    if (post || pre) {
      __syncthreads();
      if (post && wp == 0) stats_join<kRows>(ex, 0, a.c, warps);
      if (pre && wp == second) stats_join<kRows>(ex, 2, a.c, warps);
      __syncthreads();
      if (post) m1 = total4(ex, 0), r1 = total4(ex, 1);
      if (pre) m2 = total4(ex, 2), r2 = total4(ex, 3);
    }
    if (pre) {
      F4 s0 = all(0.f), s1 = all(0.f);
      FOR_ROWS(j) if (rows.on(j)) {
        const F4 t = dz_of(j) * all(__ldg(a.prm.pre_weight + rows.param(j)));
        s0 = s0 + t;
        s1 = fma4(t, (y_of(j) - m2) * r2, s1);
      }
      sum_part(s0, ex, 0);
      sum_part(s1, ex, 1);
      __syncthreads();
      if (wp == 0) sum_join(ex, 0, warps);
      if (wp == second) sum_join(ex, 1, warps);
      __syncthreads();
      am = total4(ex, 0) * all(inv_c);
      ay = total4(ex, 1) * all(inv_c);
    }
    // everything of a row but d_f's projection
    struct Row {
      F4 d, du, fn, u, sg, os, sc, yn, dz;
    };
    auto row_of = [&](int j) {
      const int ch = rows.param(j);
      Row k;
      k.d = kRows ? dy[j % kHeld] : grad(a.dy, j);
      k.yn = k.dz = all(0.f);
      if (pre) {
        k.dz = dz_of(j);
        k.yn = (y_of(j) - m2) * r2;
        const F4 t = k.dz * all(__ldg(a.prm.pre_weight + ch));
        k.d = fma4(fma4(-k.yn, ay, t - am), r2, k.d);
      }
      k.fn = k.u = all(0.f);
      if (need_f) {
        k.u = f_of(j);
        k.fn = (k.u - m1) * r1;
        if (post)
          k.u = fma4(k.fn, all(__ldg(a.prm.post_weight + ch)), all(__ldg(a.prm.post_bias + ch)));
      }
      k.sg = sg1;
      k.os = os1;
      if (per_row) sigmoid4(gate_of(j), &k.sg, &k.os);
      k.sc = all(a.prm.scale ? __ldg(a.prm.scale + ch) : 1.f);
      k.du = k.d * k.sc * k.sg;
      return k;
    };
    F4 t0 = all(0.f), t1 = all(0.f), t2 = all(0.f);
    FOR_ROWS(j) {
      const Row k = row_of(j);
      const int ch = rows.param(j);
      const long long e = (base + ch) * a.p;
      F4 b = k.du;
      if (post) b = b * all(__ldg(a.prm.post_weight + ch));
      if (rows.on(j)) {
        store4<kVec>(a.dx + e, at, a.p, k.d);
        if (!post && a.df) store4<kVec>(a.df + e, at, a.p, k.du);
        if (per_row) store4<kVec>(a.dgate + e, at, a.p, k.du * k.u * k.os);
        t0 = t0 + b;
        t1 = fma4(b, k.fn, t1);
        t2 = fma4(k.d * k.sc, k.u, t2);
      }
      const float v[5] = {sum4(k.d * k.sg * k.u), sum4(k.du * k.fn), sum4(k.du), sum4(k.dz * k.yn),
                          sum4(k.dz)};
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        if (kRows) {
          acc[j % kHeld][i] += v[i];
        } else {
          float s = v[i];
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
          if ((lane & 7) == 0 && rows.on(j)) acc_c[i * a.c + ch] += s;
        }
      }
      if (kRows) {
        dy[j % kHeld] = b;  // from here on b
      }
    }
    if (post || a.gate_c == 1) {
      if (post) sum_part(t0, ex, 0), sum_part(t1, ex, 1);
      if (a.gate_c == 1) sum_part(t2, ex, 2);
      __syncthreads();
      if (post && wp == 0) sum_join(ex, 0, warps);
      if (post && wp == second) sum_join(ex, 1, warps);
      if (a.gate_c == 1 && wp == warps - 1) sum_join(ex, 2, warps);
      __syncthreads();
      if (a.gate_c == 1 && threadIdx.x < 8)
        store4<kVec>(a.dgate + img * a.p, at, a.p, total4(ex, 2) * sg1 * os1);
      if (post) {
        const F4 bm = total4(ex, 0) * all(inv_c), bf = total4(ex, 1) * all(inv_c);
        FOR_ROWS(j) if (rows.on(j)) {
          const int ch = rows.param(j);
          F4 b = dy[j % kHeld], fn;
          if (kRows) {
            fn = (f_of(j) - m1) * r1;
          } else {
            const Row k = row_of(j);
            fn = k.fn;
            b = k.du * all(__ldg(a.prm.post_weight + ch));
          }
          store4<kVec>(a.df + (base + ch) * a.p, at, a.p, fma4(-fn, bf, b - bm) * r1);
        }
      }
    }
  }
  float* out = a.sums + (long long)blockIdx.x * 5 * a.c;
  if (kRows) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        float s = acc[j][i];
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((lane & 7) == 0 && rows.on(j)) out[i * a.c + rows.row(j)] = s;
      }
  } else {
    __syncthreads();
    for (int i = threadIdx.x; i < 5 * a.c; i += blockDim.x) out[i] = acc_c[i];
  }
}

struct SumOut {
  float* p[5];
};

// out[k][ch] = sum over the blocks of sums[block][k][ch], in a fixed order
__global__ void __launch_bounds__(256) residual_sums_kernel(const float* __restrict__ sums,
                                                            int blocks, int c, SumOut out) {
  __shared__ float red[8][33];
  const int k = blockIdx.y, ch = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
  float s = 0.f;
  if (ch < c)
    for (int b = r; b < blocks; b += 8) s += sums[((long long)b * 5 + k) * c + ch];
  red[r][threadIdx.x & 31] = s;
  __syncthreads();
  if (r == 0 && ch < c && out.p[k]) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x & 31];
    out.p[k][ch] = s;
  }
}

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

using namespace zjai;

extern "C" {

int zjai_gated_residual_norm(zjai_ctx* ctx, const void* x, const void* f, const void* gate,
                             int gate_channels, int dtype, int n, int c, int h, int w,
                             const zjai_residual_params* prm, void* y, void* z,
                             const zjai_residual_tapes* tapes, int mem) {
  return guarded([&]() -> int {
    const char* me = "gated_residual_norm";
    ZJAI_TRY(ctx_enter(ctx));
    ZJAI_TRY(check_map(me, dtype, n, c, h, w));
    ZJAI_TRY(check_mem(mem));
    ZJAI_TRY(check_step(me, c, gate_channels, prm));
    if (!x || !f || !y || (gate_channels && !gate) || (prm->pre_weight && !z))
      return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": null buffer");
    const zjai_residual_tapes none = {};
    const zjai_residual_tapes& want = tapes ? *tapes : none;
    if ((want.gate.codes && !gate_channels) || (want.z.codes && !prm->pre_weight))
      return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": tape of a part the step lacks");
    const zjai_tape* wt[4] = {&want.f, &want.gate, &want.y, &want.z};
    for (const zjai_tape* t : wt)
      if (t->codes && !t->exps)
        return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": tape without exponents");
    ArenaScope scope(ctx);
    const int p = h * w;
    const size_t es = dtype_size(dtype), rows = (size_t)n * c, groups = tape_groups(p);
    const size_t bytes = rows * p * es, grows = (size_t)n * gate_channels;
    const char *dx, *df, *dg;
    char *dyo, *dzo;
    zjai_residual_params dp = {};
    ZJAI_TRY(stage_bytes_in(ctx, (const char*)x, bytes, es, mem, "x", &dx));
    ZJAI_TRY(stage_bytes_in(ctx, (const char*)f, bytes, es, mem, "f", &df));
    ZJAI_TRY(stage_bytes_in(ctx, gate_channels ? (const char*)gate : nullptr, grows * p * es, es,
                            mem, "gate", &dg));
    ZJAI_TRY(stage_params(ctx, *prm, c, mem, &dp));
    ZJAI_TRY(stage_bytes_out(ctx, (char*)y, bytes, es, mem, "y", &dyo));
    ZJAI_TRY(stage_bytes_out(ctx, prm->pre_weight ? (char*)z : nullptr, bytes, es, mem, "z", &dzo));
    zjai_residual_tapes dt = {};
    zjai_tape* tt[4] = {&dt.f, &dt.gate, &dt.y, &dt.z};
    const size_t tr[4] = {rows, grows, rows, rows};
    for (int i = 0; i < 4; ++i) {
      if (!wt[i]->codes) continue;
      ZJAI_TRY(stage_bytes_out(ctx, wt[i]->codes, tr[i] * p, 1, mem, "codes", &tt[i]->codes));
      ZJAI_TRY(stage_bytes_out(ctx, wt[i]->exps, tr[i] * groups, 1, mem, "exps", &tt[i]->exps));
    }
    const Shape sh = shape_of(c);
    VecCheck vec(p);
    vec.map(dx, es).map(df, es).map(dg, es).map(dyo, es).map(dzo, es);
    for (zjai_tape* t : tt) vec.map(t->codes, 1);
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      return by_rows(sh.rows, [&](auto r) -> int {
        constexpr int kRows = decltype(r)::value;
        FwdArgs<T> a = {(const T*)dx, (const T*)df, (const T*)dg, gate_channels, c, p,
                        (long long)n * (long long)groups, dp, (T*)dyo, (T*)dzo, dt};
        const int blocks = (int)std::min<long long>(a.tiles, (long long)ctx->sms * sh.per_sm);
        auto k = vec.ok ? residual_norm_kernel<kRows, true, T> : residual_norm_kernel<kRows, false, T>;
        k<<<blocks, sh.warps * 32, 0, ctx->stream>>>(a);
        return cuda_check(cudaGetLastError(), "gated_residual_norm");
      });
    }));
    ctx->launches++;
    ZJAI_TRY(finish_bytes_out(ctx, y, dyo, bytes, mem));
    if (dzo) ZJAI_TRY(finish_bytes_out(ctx, z, dzo, bytes, mem));
    for (int i = 0; i < 4; ++i) {
      if (!wt[i]->codes) continue;
      ZJAI_TRY(finish_bytes_out(ctx, wt[i]->codes, tt[i]->codes, tr[i] * p, mem));
      ZJAI_TRY(finish_bytes_out(ctx, wt[i]->exps, tt[i]->exps, tr[i] * groups, mem));
    }
    return finish_call(ctx, mem);
  });
}

int zjai_gated_residual_norm_backward(zjai_ctx* ctx, const void* dy, const void* dz, const void* f,
                                      const void* gate, int gate_channels, const void* y,
                                      const zjai_residual_tapes* tapes, int dtype, int n, int c,
                                      int h, int w, const zjai_residual_params* prm,
                                      const zjai_residual_grads* grads, int mem) {
  return guarded([&]() -> int {
    const char* me = "gated_residual_norm_backward";
    ZJAI_TRY(ctx_enter(ctx));
    ZJAI_TRY(check_map(me, dtype, n, c, h, w));
    ZJAI_TRY(check_mem(mem));
    ZJAI_TRY(check_step(me, c, gate_channels, prm));
    const bool post = prm->post_weight, pre = prm->pre_weight, taped = tapes != nullptr;
    const bool need_f = post || prm->scale || gate_channels;
    if (!dy || !grads || !grads->x || (pre && !dz) || (need_f && !grads->f) ||
        (gate_channels && !grads->gate) || (post && (!grads->post_weight || !grads->post_bias)) ||
        (prm->scale && !grads->scale) || (pre && (!grads->pre_weight || !grads->pre_bias)))
      return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": null buffer");
    if (taped && (f || gate || y))
      return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": either tapes or maps");
    auto have = [&](const void* map, const zjai_tape* t) {
      return taped ? t->codes && t->exps : map != nullptr;
    };
    const zjai_residual_tapes none = {};
    const zjai_residual_tapes& kept = taped ? *tapes : none;
    if ((need_f && !have(f, &kept.f)) || (gate_channels && !have(gate, &kept.gate)) ||
        (pre && !have(y, &kept.y)))
      return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": f, gate or y missing");
    ArenaScope scope(ctx);
    const int p = h * w;
    const size_t es = dtype_size(dtype), rows = (size_t)n * c, groups = tape_groups(p);
    const size_t bytes = rows * p * es, grows = (size_t)n * gate_channels;
    const char *ddy, *ddz, *df = nullptr, *dg = nullptr, *dyy = nullptr;
    zjai_residual_tapes dt = {};
    zjai_residual_params dp = {};
    ZJAI_TRY(stage_bytes_in(ctx, (const char*)dy, bytes, es, mem, "dy", &ddy));
    ZJAI_TRY(stage_bytes_in(ctx, pre ? (const char*)dz : nullptr, bytes, es, mem, "dz", &ddz));
    if (!taped) {
      ZJAI_TRY(stage_bytes_in(ctx, need_f ? (const char*)f : nullptr, bytes, es, mem, "f", &df));
      ZJAI_TRY(stage_bytes_in(ctx, gate_channels ? (const char*)gate : nullptr, grows * p * es, es,
                              mem, "gate", &dg));
      ZJAI_TRY(stage_bytes_in(ctx, pre ? (const char*)y : nullptr, bytes, es, mem, "y", &dyy));
    } else {
      const zjai_tape* in[3] = {need_f ? &kept.f : nullptr, gate_channels ? &kept.gate : nullptr,
                                pre ? &kept.y : nullptr};
      zjai_tape* out[3] = {&dt.f, &dt.gate, &dt.y};
      const size_t tr[3] = {rows, grows, rows};
      for (int i = 0; i < 3; ++i) {
        if (!in[i]) continue;
        const int8_t *cd, *ex;
        ZJAI_TRY(stage_bytes_in(ctx, (const int8_t*)in[i]->codes, tr[i] * p, 1, mem, "codes", &cd));
        ZJAI_TRY(
            stage_bytes_in(ctx, (const int8_t*)in[i]->exps, tr[i] * groups, 1, mem, "exps", &ex));
        *out[i] = {const_cast<int8_t*>(cd), const_cast<int8_t*>(ex)};
      }
    }
    ZJAI_TRY(stage_params(ctx, *prm, c, mem, &dp));
    char *gx, *gf, *gg;
    ZJAI_TRY(stage_bytes_out(ctx, (char*)grads->x, bytes, es, mem, "d_x", &gx));
    ZJAI_TRY(stage_bytes_out(ctx, (char*)grads->f, bytes, es, mem, "d_f", &gf));
    ZJAI_TRY(stage_bytes_out(ctx, gate_channels ? (char*)grads->gate : nullptr, grows * p * es, es,
                             mem, "d_gate", &gg));
    float* host[5] = {prm->scale ? grads->scale : nullptr, post ? grads->post_weight : nullptr,
                      post ? grads->post_bias : nullptr, pre ? grads->pre_weight : nullptr,
                      pre ? grads->pre_bias : nullptr};
    SumOut so;
    for (int i = 0; i < 5; ++i)
      ZJAI_TRY(stage_bytes_out(ctx, host[i], (size_t)c * 4, 4, mem, "parameter gradient", &so.p[i]));
    const long long tiles = (long long)n * (long long)groups;
    const Shape sh = shape_of(c);
    const int blocks = (int)std::min<long long>(tiles, (long long)ctx->sms * sh.per_sm);
    float* sums = static_cast<float*>(ctx->arena.alloc((size_t)blocks * 5 * c * sizeof(float)));
    if (!sums) return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (parameter sums)");
    VecCheck vec(p);
    vec.map(ddy, es).map(ddz, es).map(df, es).map(dg, es).map(dyy, es);
    vec.map(gx, es).map(gf, es).map(gg, es);
    vec.map(dt.f.codes, 1).map(dt.gate.codes, 1).map(dt.y.codes, 1);
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      return by_rows(sh.rows, [&](auto r) -> int {
        constexpr int kRows = decltype(r)::value;
        BwdArgs<T> a = {(const T*)ddy, (const T*)ddz, (const T*)df, (const T*)dg, (const T*)dyy, dt,
                        gate_channels, c, p, tiles, dp, (T*)gx, (T*)gf, (T*)gg, sums};
        auto k = taped ? (vec.ok ? residual_norm_bwd_kernel<kRows, true, true, T>
                                 : residual_norm_bwd_kernel<kRows, true, false, T>)
                       : (vec.ok ? residual_norm_bwd_kernel<kRows, false, true, T>
                                 : residual_norm_bwd_kernel<kRows, false, false, T>);
        const size_t smem = kRows ? 0 : (size_t)5 * c * sizeof(float);
        if (!kRows)
          ZJAI_TRY(cuda_check(cudaFuncSetAttribute((const void*)k,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   5 * kMaxC * (int)sizeof(float)),
                              "gated_residual_norm_backward"));
        k<<<blocks, sh.warps * 32, smem, ctx->stream>>>(a);
        return cuda_check(cudaGetLastError(), "gated_residual_norm_backward");
      });
    }));
    residual_sums_kernel<<<dim3((c + 31) / 32, 5), 256, 0, ctx->stream>>>(sums, blocks, c, so);
    ctx->launches += 2;
    ZJAI_TRY(cuda_check(cudaGetLastError(), "parameter sums"));
    ZJAI_TRY(finish_bytes_out(ctx, grads->x, gx, bytes, mem));
    if (gf) ZJAI_TRY(finish_bytes_out(ctx, grads->f, gf, bytes, mem));
    if (gg) ZJAI_TRY(finish_bytes_out(ctx, grads->gate, gg, grows * p * es, mem));
    for (int i = 0; i < 5; ++i)
      if (host[i]) ZJAI_TRY(finish_bytes_out(ctx, host[i], so.p[i], (size_t)c * 4, mem));
    return finish_call(ctx, mem);
  });
}

}  // extern "C"
