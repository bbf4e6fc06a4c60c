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
// Maps are planar: a channel row holds a picture's positions. A block takes a tile of 32
// consecutive positions of one picture, which are one group of each row's 8-bit tape: lane =
// position, the channels spread over the warps, a position's sums gathered over the warps in
// shared memory. Variances are two-pass (the mean first; one pass would cancel), and the second pass
// also sums the deviations, which corrects the mean's own rounding: a normalised value near zero
// keeps its relative precision. The products in a - mean a and b - mean b are the ones that were
// summed (no fused multiply-add): with one channel they cancel to zero.
#include <algorithm>

#include "train.h"

namespace zjai {
namespace {

constexpr float kEps = 1e-5f;
constexpr int kMaxC = 8192;  // the parameter sums of a block sit in shared memory, 20 B a channel
constexpr int kWarps = 8;

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

// sigmoid(g) and 1 - sigmoid(g), neither by cancellation and both finite for every g but NaN
__device__ __forceinline__ void sigmoid2(float g, float* s, float* one_minus) {
  const float a = expf(-fabsf(g)), r = 1.f / (1.f + a), ar = a * r;
  *s = g >= 0.f ? r : (g < 0.f ? ar : g);
  *one_minus = g >= 0.f ? ar : (g < 0.f ? r : g);
}

// A position's mean over the channels (m, and what its rounding left, dm) and 1 / sigma.
struct Stats {
  float m = 0.f, dm = 0.f, r = 1.f;
  // from the means of v - m and (v - m)^2
  __device__ __forceinline__ void finish(float d, float sq) {
    dm = d;
    r = 1.f / sqrtf(fmaxf(sq - d * d, 0.f) + kEps);
  }
  __device__ __forceinline__ float norm(float v) const { return ((v - m) - dm) * r; }
};

// Sum of v over the block's warps, per lane, in warp order.
__device__ __forceinline__ float over_warps(float v, float (*red)[32]) {
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  __syncthreads();
  red[wp][lane] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) s += red[k][lane];
  return s;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Hold a value per lane (0 beyond the row's end) as the group of a tape: row, group index.
__device__ __forceinline__ void tape_group_store(const zjai_tape& t, long long row, int groups,
                                                 int g, int p, float v, bool in) {
  const int lane = threadIdx.x & 31;
  const int e = tape_exp(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
  const uint32_t code = e == kTapeNan ? 0u : tape_code_bits(v, tape_inv_scale(e));
  if (in) t.codes[row * p + g * kTapeGroup + lane] = (int8_t)(code & 0xffu);
  if (lane == 0) t.exps[row * groups + g] = (int8_t)e;
}

template <bool kTaped, class T>
__device__ __forceinline__ float load_kept(const T* v, const zjai_tape& t, long long row,
                                           int groups, int g, int p, bool in) {
  const long long at = row * p + g * kTapeGroup + (threadIdx.x & 31);
  if (!in) return 0.f;
  if (kTaped) return (float)t.codes[at] * tape_scale(t.exps[row * groups + g]);
  return to_f32(v[at]);
}

// Any channel count: a tile's channels are read again for each of the step's sums.
template <class T>
__global__ void __launch_bounds__(kWarps * 32) residual_norm_kernel(FwdArgs<T> a) {
  __shared__ float red[kWarps][32];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  for (long long tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const long long img = tile / groups;
    const int g = (int)(tile - img * groups), at = g * kTapeGroup + lane;
    const bool in = at < a.p;
    const long long base = img * a.c;
    const T* gate = a.gate ? a.gate + img * a.gate_c * a.p + at : nullptr;
    auto value = [&](const T* v, int ch) { return in ? to_f32(v[(base + ch) * a.p + at]) : 0.f; };
    // mean, its correction and 1 / sigma of v(ch) over the channels
    auto stats = [&](auto v) {
      float s = 0.f, t = 0.f;
      for (int ch = wp; ch < a.c; ch += kWarps) s += v(ch);
      Stats st;
      st.m = over_warps(s, red) * inv_c;
      s = 0.f;
      for (int ch = wp; ch < a.c; ch += kWarps) {
        const float d = v(ch) - st.m;
        s += d * d;
        t += d;
      }
      st.finish(over_warps(t, red) * inv_c, over_warps(s, red) * inv_c);
      return st;
    };
    Stats s1, s2;
    if (a.prm.post_weight) s1 = stats([&](int ch) { return value(a.f, ch); });
    float sg1 = 1.f, unused;
    if (a.gate && a.gate_c == 1) sigmoid2(in ? to_f32(gate[0]) : 0.f, &sg1, &unused);
    auto y_of = [&](int ch) {
      float u = value(a.f, ch), q = sg1;
      if (a.prm.post_weight)
        u = s1.norm(u) * __ldg(a.prm.post_weight + ch) + __ldg(a.prm.post_bias + ch);
      if (a.gate && a.gate_c != 1)
        sigmoid2(in ? to_f32(gate[(long long)ch * a.p]) : 0.f, &q, &unused);
      if (a.prm.scale) q *= __ldg(a.prm.scale + ch);
      return value(a.x, ch) + q * u;
    };
    if (a.prm.pre_weight) s2 = stats(y_of);
    for (int ch = wp; ch < a.c; ch += kWarps) {
      const long long row = base + ch;
      const float y = y_of(ch);
      if (in) a.y[row * a.p + at] = from_f32<T>(y);
      if (a.tp.f.codes) tape_group_store(a.tp.f, row, groups, g, a.p, value(a.f, ch), in);
      if (a.tp.gate.codes && (a.gate_c != 1 || ch == 0))
        tape_group_store(a.tp.gate, img * a.gate_c + (a.gate_c == 1 ? 0 : ch), groups, g, a.p,
                         in ? to_f32(gate[a.gate_c == 1 ? 0 : (long long)ch * a.p]) : 0.f, in);
      if (a.tp.y.codes) tape_group_store(a.tp.y, row, groups, g, a.p, in ? y : 0.f, in);
      if (a.prm.pre_weight) {
        const float z = s2.norm(y) * __ldg(a.prm.pre_weight + ch) + __ldg(a.prm.pre_bias + ch);
        if (in) a.z[row * a.p + at] = from_f32<T>(z);
        if (a.tp.z.codes) tape_group_store(a.tp.z, row, groups, g, a.p, in ? z : 0.f, in);
      }
    }
  }
}

// Backward, any channel count: as the forward kernel, and a block's parameter sums in shared
// memory, a channel's by the warp that owns it, written out per block when the block ends.
template <bool kTaped, class T>
__global__ void __launch_bounds__(kWarps * 32) residual_norm_bwd_kernel(BwdArgs<T> a) {
  __shared__ float red[kWarps][32];
  extern __shared__ float acc[];  // [5][c]
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, gated = a.gate_c != 0;
  const bool need_f = post || gated || a.prm.scale;
  for (int i = threadIdx.x; i < 5 * a.c; i += blockDim.x) acc[i] = 0.f;
  __syncthreads();
  for (long long tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const long long img = tile / groups;
    const int g = (int)(tile - img * groups), at = g * kTapeGroup + lane;
    const bool in = at < a.p;
    const long long base = img * a.c;
    auto grad = [&](const T* v, int ch) { return in ? to_f32(v[(base + ch) * a.p + at]) : 0.f; };
    auto f_of = [&](int ch) {
      return load_kept<kTaped>(a.f, a.tp.f, base + ch, groups, g, a.p, in);
    };
    auto y_of = [&](int ch) {
      return load_kept<kTaped>(a.y, a.tp.y, base + ch, groups, g, a.p, in);
    };
    auto gate_of = [&](int ch) {
      return load_kept<kTaped>(a.gate, a.tp.gate, img * a.gate_c + ch, groups, g, a.p, in);
    };
    auto stats = [&](auto v) {
      float s = 0.f, t = 0.f;
      for (int ch = wp; ch < a.c; ch += kWarps) s += v(ch);
      Stats st;
      st.m = over_warps(s, red) * inv_c;
      s = 0.f;
      for (int ch = wp; ch < a.c; ch += kWarps) {
        const float d = v(ch) - st.m;
        s += d * d;
        t += d;
      }
      st.finish(over_warps(t, red) * inv_c, over_warps(s, red) * inv_c);
      return st;
    };
    Stats s1, s2;
    float am = 0.f, ay = 0.f;
    if (post) s1 = stats(f_of);
    if (pre) {
      s2 = stats(y_of);
      float t0 = 0.f, t1 = 0.f;
      for (int ch = wp; ch < a.c; ch += kWarps) {
        const float t = __fmul_rn(grad(a.dz, ch), __ldg(a.prm.pre_weight + ch));
        t0 += t;
        t1 += t * s2.norm(y_of(ch));
      }
      am = over_warps(t0, red) * inv_c;
      ay = over_warps(t1, red) * inv_c;
    }
    float sg1 = 1.f, os1 = 0.f;
    if (a.gate_c == 1) sigmoid2(gate_of(0), &sg1, &os1);
    // D, fn, u, sigma(g), 1 - sigma(g), s of one channel
    struct Chan {
      float d, fn, u, sg, os, sc, yn, dz;
    };
    auto chan = [&](int ch) {
      Chan k;
      k.d = grad(a.dy, ch);
      k.yn = k.dz = 0.f;
      if (pre) {
        k.dz = grad(a.dz, ch);
        k.yn = s2.norm(y_of(ch));
        k.d += (__fmul_rn(k.dz, __ldg(a.prm.pre_weight + ch)) - am - k.yn * ay) * s2.r;
      }
      k.fn = k.u = 0.f;
      if (need_f) {
        const float f = f_of(ch);
        k.fn = s1.norm(f);
        k.u = post ? k.fn * __ldg(a.prm.post_weight + ch) + __ldg(a.prm.post_bias + ch) : f;
      }
      k.sg = sg1;
      k.os = os1;
      if (gated && a.gate_c != 1) sigmoid2(gate_of(ch), &k.sg, &k.os);
      k.sc = a.prm.scale ? __ldg(a.prm.scale + ch) : 1.f;
      return k;
    };
    float bm = 0.f, bf = 0.f;
    if (post || a.gate_c == 1) {
      float t0 = 0.f, t1 = 0.f, t2 = 0.f;
      for (int ch = wp; ch < a.c; ch += kWarps) {
        const Chan k = chan(ch);
        if (post) {
          const float t = __fmul_rn(k.d * k.sc * k.sg, __ldg(a.prm.post_weight + ch));
          t0 += t;
          t1 += t * k.fn;
        }
        t2 += k.d * k.sc * k.u;
      }
      bm = over_warps(t0, red) * inv_c;
      bf = over_warps(t1, red) * inv_c;
      if (a.gate_c == 1) {
        t2 = over_warps(t2, red);
        if (wp == 0 && in) a.dgate[img * a.p + at] = from_f32<T>(t2 * sg1 * os1);
      }
    }
    for (int ch = wp; ch < a.c; ch += kWarps) {
      const Chan k = chan(ch);
      const long long e = (base + ch) * a.p + at;
      const float du = k.d * k.sc * k.sg;
      if (in) {
        a.dx[e] = from_f32<T>(k.d);
        if (a.df)
          a.df[e] = from_f32<T>(
              post ? (__fmul_rn(du, __ldg(a.prm.post_weight + ch)) - bm - k.fn * bf) * s1.r : du);
        if (a.gate_c > 1)
          a.dgate[e] = from_f32<T>(k.d * k.sc * k.u * k.sg * k.os);
      }
      float v[5] = {k.d * k.sg * k.u, du * k.fn, du, k.dz * k.yn, k.dz};
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const float s = warp_sum(in ? v[i] : 0.f);
        if (lane == 0) acc[i * a.c + ch] += s;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 5 * a.c; i += blockDim.x)
    a.sums[(long long)blockIdx.x * 5 * a.c + i] = acc[i];
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
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      FwdArgs<T> a = {(const T*)dx, (const T*)df, (const T*)dg, gate_channels, c, p,
                      (long long)n * (long long)groups, dp, (T*)dyo, (T*)dzo, dt};
      const int blocks = (int)std::min<long long>(a.tiles, (long long)ctx->sms * 8);
      residual_norm_kernel<T><<<blocks, kWarps * 32, 0, ctx->stream>>>(a);
      return cuda_check(cudaGetLastError(), "gated_residual_norm");
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
    const int blocks = (int)std::min<long long>(tiles, (long long)ctx->sms * 4);
    float* sums = static_cast<float*>(ctx->arena.alloc((size_t)blocks * 5 * c * sizeof(float)));
    if (!sums) return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (parameter sums)");
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      BwdArgs<T> a = {(const T*)ddy, (const T*)ddz, (const T*)df, (const T*)dg, (const T*)dyy, dt,
                      gate_channels, c, p, tiles, dp, (T*)gx, (T*)gf, (T*)gg, sums};
      const size_t smem = (size_t)5 * c * sizeof(float);
      auto k = taped ? residual_norm_bwd_kernel<true, T> : residual_norm_bwd_kernel<false, T>;
      ZJAI_TRY(cuda_check(cudaFuncSetAttribute((const void*)k,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               5 * kMaxC * (int)sizeof(float)),
                          "gated_residual_norm_backward"));
      k<<<blocks, kWarps * 32, smem, ctx->stream>>>(a);
      return cuda_check(cudaGetLastError(), "gated_residual_norm_backward");
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
