// Parameter gradients of a 1x1 convolution from the 8-bit tape of its input
// (zjai_conv1x1_weight_grad): dw[o][i] = sum over pictures and positions of d_out[o] x[i],
// db[o] = sum of d_out[o].
//
// A matrix product whose long axis K is the positions, along which both operands are contiguous
// (planar maps): dw = D X^T on tcgen05.mma, M = 128 output channels, N = up to 128 input channels,
// K = 16 positions an instruction. Read once, the operands bound it (HBM) up to about 500 channels
// a side; above that the tensor cores do.
//
// Exactness. A taped value code 2^e has at most 7 significant bits: exact in bf16. d_out in bf16
// goes in as it is; in f16 as the sum of two bf16 numbers, in f32 of three, each the truncation of
// what the ones before left (8 + 8 + 8 bits: exact), so every product is exact and the result has
// the error of its f32 sums alone, like an f32 product of the f32 operands. The tensor core's own
// accumulation truncates, a bias that grows with the length of the chain: the first terms have an
// accumulator of their own, and both are drained every kWindow positions and added, rounding to
// nearest, to f32 sums in registers.
//
// One CTA per SM takes a 128 x N tile of dw over a range of positions:
//  - 8 loader warps read both operands into registers a chunk ahead, convert, and store them in the
//    128-byte-swizzled K-major layout the tensor core reads (16-byte piece j of row r at j ^ (r & 7));
//    no TMA: its boxes cannot start at the odd row strides of planar maps, and all but bf16 d_out
//    passes through registers anyway. They also sum d_out's rows for db;
//  - one thread issues the MMAs of a chunk, alternating between two accumulator sets in TMEM;
//  - 8 warps drain a finished set while the next one fills.
// Ranges of one tile are summed in order by a second kernel (no atomics). Every wait is bounded.
#include <algorithm>

#include "ptx.cuh"
#include "train.h"

namespace zjai {
namespace {

constexpr int kM = 128, kN = 128;       // tile of dw
constexpr int kWindow = 256;            // positions between drains
constexpr int kLoaderWarp = 8, kMmaWarp = 16;
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr int kBlock = kM * 64 * 2;     // 64 positions of 128 rows in bf16

// bf16 terms of a d_out element, positions per pipeline stage, stages
template <class T>
struct Form;
template <>
struct Form<float> {
  static constexpr int kTerms = 3, kChunk = 64, kStages = 3;
};
template <>
struct Form<__half> {
  static constexpr int kTerms = 2, kChunk = 128, kStages = 2;
};
template <>
struct Form<__nv_bfloat16> {
  static constexpr int kTerms = 1, kChunk = 128, kStages = 3;
};

struct WgArgs {
  const void* dout;
  const int8_t *codes, *exps;
  int oc, c, p, groups;
  int nb;          // N of the MMA: rows of the input tile, a multiple of 16
  int m_tiles;
  int chunks_img;  // chunks per picture
  long long chunks;
  int splits;
  int vec_d, vec_x;  // rows start on 16-byte boundaries
  float *dw, *db;    // [split][oc][c], [split][oc] (db null: not wanted)
  int* err;
  long long limit;
};

__device__ __forceinline__ uint32_t bf2(float lo, float hi) {  // truncated: the upper halves
  return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
}
__device__ __forceinline__ float trunc_bf(float v) {
  return __uint_as_float(__float_as_uint(v) & 0xffff0000u);
}
// what truncation to bf16 left of v (none of an infinity; NaN stays NaN)
__device__ __forceinline__ float rest_bf(float v) {
  const float r = v - trunc_bf(v);
  return fabsf(v) == __uint_as_float(0x7f800000u) ? 0.f : r;
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// 8 positions of a d_out row, raw
template <class T>
struct Raw {
  uint4 v[sizeof(T) == 4 ? 2 : 1];
};
template <class T>
__device__ __forceinline__ Raw<T> load_d(const T* row, int at, int p, bool ok, bool vec) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.v[i] = make_uint4(0u, 0u, 0u, 0u);
  if (!ok || at >= p) return r;
  if (vec) {  // p is a multiple of 8 elements here: all eight are in
    const uint4* q = reinterpret_cast<const uint4*>(row + at);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.v[i] = __ldg(q + i);
    return r;
  }
  uint32_t e[8];
  if constexpr (sizeof(T) == 4) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = at + i < p ? __ldg(q + at + i) : 0u;
    r.v[0] = make_uint4(e[0], e[1], e[2], e[3]);
    r.v[sizeof(T) / 2 - 1] = make_uint4(e[4], e[5], e[6], e[7]);
  } else {
    const unsigned short* q = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = at + i < p ? __ldg(q + at + i) : 0u;
    r.v[0] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
  }
  return r;
}

// 16 codes of an input row and their exponent
struct RawX {
  uint4 v;
  int e;
};
__device__ __forceinline__ RawX load_x(const int8_t* row, const int8_t* exps, int at, int p, bool ok,
                                       bool vec) {
  RawX r = {make_uint4(0u, 0u, 0u, 0u), 0};
  if (!ok || at >= p) return r;
  r.e = __ldg(exps + at / kTapeGroup);
  if (vec) {
    r.v = __ldg(reinterpret_cast<const uint4*>(row + at));
    return r;
  }
  const uint8_t* q = reinterpret_cast<const uint8_t*>(row);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + 4 * i + j < p) w[i] |= (uint32_t)__ldg(q + at + 4 * i + j) << (8 * j);
  }
  r.v = make_uint4(w[0], w[1], w[2], w[3]);
  return r;
}

// 4 codes -> 4 bf16 values code 2^e: the low 7 bits and the sign bit of a code, each as the low
// mantissa bits of 128 (bf16 0x4300), give code = (128 + low7) - (128 + 128 sign); the subtraction
// and the scaling are exact.
__device__ __forceinline__ uint2 taped_bf16(uint32_t w, __nv_bfloat162 scale) {
  uint2 out;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t t = __byte_perm(w, 0u, h ? 0x4342 : 0x4140);
    const uint32_t a = (t & 0x007f007fu) | 0x43004300u, b = (t & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 v = __hmul2(
        __hsub2(reinterpret_cast<const __nv_bfloat162&>(a), reinterpret_cast<const __nv_bfloat162&>(b)),
        scale);
    (h ? out.y : out.x) = reinterpret_cast<const uint32_t&>(v);
  }
  return out;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 1) weight_grad_kernel(const WgArgs a) {
  using F = Form<T>;
  constexpr int kTerms = F::kTerms, kSub = F::kChunk / 64, kStages = F::kStages;
  constexpr int kStageBytes = (kTerms + 1) * kSub * kBlock;
  constexpr int kPerWindow = kWindow / F::kChunk;
  constexpr int kSets = kTerms > 1 ? 2 : 1;  // accumulators of a set: first terms, the others
  extern __shared__ char smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 4 + 1];
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x, split = blockIdx.y;
  const int o0 = (tile % a.m_tiles) * kM, i0 = (tile / a.m_tiles) * kN;
  const long long q0 = a.chunks * split / a.splits, q1 = a.chunks * (split + 1) / a.splits;
  const int count = (int)(q1 - q0), windows = (count + kPerWindow - 1) / kPerWindow;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, acc_full = empty + 8 * kStages,
                 acc_empty = acc_full + 16, drain = acc_empty + 16;
  volatile int* abort = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, 8);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, 8);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&tmem_at), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;

  if (warp == kMmaWarp) {
    if (lane == 0) {
      const uint32_t idesc = idesc_f16((uint32_t)a.nb) | (1u << 7) | (1u << 10);  // bf16 operands
      bool ok = true;
      for (int k = 0; k < count && ok; ++k) {
        const int st = k % kStages, win = k / kPerWindow, buf = win & 1;
        const bool first = k % kPerWindow == 0;
        if (first && win >= 2) {
          ok = mbar_wait(acc_empty + 8 * buf, ((win >> 1) - 1) & 1, abort, a.err,
                         DEV_TIMEOUT_ACC_EMPTY, a.limit);
          if (!ok) break;
        }
        ok = mbar_wait(full + 8 * st, (k / kStages) & 1, abort, a.err, DEV_TIMEOUT_FULL, a.limit);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * kSets * kN;
#pragma unroll
        for (int s = 0; s < kSub; ++s) {
          const uint32_t at = smem + st * kStageBytes + s * (kTerms + 1) * kBlock;
          const uint64_t db = smem_desc(at + kTerms * kBlock, 128u);
#pragma unroll
          for (int t = 0; t < kTerms; ++t) {
            const uint64_t da = smem_desc(at + t * kBlock, 128u);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 16 positions: 32 bytes along the row
              umma_f16(d + (t ? kN : 0), da + 2 * kk, db + 2 * kk, idesc,
                       first && s == 0 && t < 2 && kk == 0 ? 0u : 1u);
          }
        }
        umma_commit(empty + 8 * st);
        if (k % kPerWindow == kPerWindow - 1 || k == count - 1) umma_commit(acc_full + 8 * buf);
      }
      // all MMAs done before TMEM goes, also after a wait that gave up
      umma_commit(drain);
      mbar_wait_drain(drain, 0, a.err);
    }
    __syncwarp();
  } else if (warp >= kLoaderWarp) {
    const int tid = threadIdx.x - kLoaderWarp * 32;
    constexpr int kUd = 4 * kSub, kUx = 2 * kSub;
    const T* dout = static_cast<const T*>(a.dout);
    const int dr = tid >> 3, dj = tid & 7;  // d_out: row (of 32), 8 positions
    const int xr = tid >> 2, xj = tid & 3;  // input: row (of 64), 16 positions
    Raw<T> rd[kUd];
    RawX rx[kUx];
    float bsum[4] = {}, btot[4] = {};
    const bool want_db = a.db && i0 == 0;
    // the chunk being loaded: its picture and first position
    long long img = q0 / a.chunks_img;
    int at0 = (int)(q0 - img * a.chunks_img) * F::kChunk;
    const T* pd = dout + (img * a.oc + o0 + dr) * (long long)a.p;
    const int8_t* px = a.codes + (img * a.c + i0 + xr) * (long long)a.p;
    const int8_t* pe = a.exps + (img * a.c + i0 + xr) * (long long)a.groups;
    const long long d32 = 32LL * a.p, x64 = 64LL * a.p, e64 = 64LL * a.groups;
    const int x_rows = min(a.nb, a.c - i0);
    auto load_du = [&](int u) {
      return load_d(pd + (u & 3) * d32, at0 + (u >> 2) * 64 + dj * 8, a.p,
                    o0 + (u & 3) * 32 + dr < a.oc, a.vec_d);
    };
    auto load_xu = [&](int u) {
      return load_x(px + (u & 1) * x64, pe + (u & 1) * e64, at0 + (u >> 1) * 64 + xj * 16, a.p,
                    (u & 1) * 64 + xr < x_rows, a.vec_x);
    };
    auto advance = [&]() {
      at0 += F::kChunk;
      if (at0 >= a.p) {
        at0 = 0;
        pd += (long long)a.oc * a.p;
        px += (long long)a.c * a.p;
        pe += (long long)a.c * a.groups;
      }
    };
#pragma unroll
    for (int u = 0; u < kUd; ++u) rd[u] = load_du(u);
#pragma unroll
    for (int u = 0; u < kUx; ++u) rx[u] = load_xu(u);
    for (int k = 0; k < count; ++k) {
      const int st = k % kStages;
      if (k >= kStages &&
          !mbar_wait(empty + 8 * st, (k / kStages - 1) & 1, abort, a.err, DEV_TIMEOUT_EMPTY, a.limit))
        break;
      const uint32_t stage = smem + st * kStageBytes;
      const bool more = k + 1 < count;
      advance();
#pragma unroll
      for (int u = 0; u < kUd; ++u) {
        const int r = (u & 3) * 32 + dr;
        const uint32_t at = stage + (u >> 2) * (kTerms + 1) * kBlock + r * 128 + ((dj ^ (r & 7)) << 4);
        float s = 0.f;
        if constexpr (kTerms == 1) {
          st_shared16(at, rd[u].v[0]);
          const uint32_t w[4] = {rd[u].v[0].x, rd[u].v[0].y, rd[u].v[0].z, rd[u].v[0].w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s += __uint_as_float(w[i] << 16) + __uint_as_float(w[i] & 0xffff0000u);
        } else {
          float f[8];
          if constexpr (kTerms == 2) {
            const uint32_t w[4] = {rd[u].v[0].x, rd[u].v[0].y, rd[u].v[0].z, rd[u].v[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 t = __half22float2(reinterpret_cast<const __half2&>(w[i]));
              f[2 * i] = t.x;
              f[2 * i + 1] = t.y;
            }
          } else {
            const uint4 v0 = rd[u].v[0], v1 = rd[u].v[sizeof(T) / 2 - 1];
            const uint32_t w[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
          }
#pragma unroll
          for (int i = 0; i < 8; i += 2) s += f[i] + f[i + 1];
#pragma unroll
          for (int t = 0; t < kTerms; ++t) {
            st_shared16(at + t * kBlock, make_uint4(bf2(f[0], f[1]), bf2(f[2], f[3]), bf2(f[4], f[5]),
                                                    bf2(f[6], f[7])));
            if (t + 1 < kTerms)
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = rest_bf(f[i]);
          }
        }
        bsum[u & 3] += s;
        if (more) rd[u] = load_du(u);
      }
#pragma unroll
      for (int u = 0; u < kUx; ++u) {
        const int r = (u & 1) * 64 + xr;
        const uint32_t row = stage + ((u >> 1) * (kTerms + 1) + kTerms) * kBlock + r * 128;
        const uint32_t sb = rx[u].e == kTapeNan ? 0x7fc0u : (uint32_t)(max(rx[u].e, -126) + 127) << 7;
        const uint32_t s2 = sb | sb << 16;
        const __nv_bfloat162 sc = reinterpret_cast<const __nv_bfloat162&>(s2);
        const uint2 v0 = taped_bf16(rx[u].v.x, sc), v1 = taped_bf16(rx[u].v.y, sc);
        const uint2 v2 = taped_bf16(rx[u].v.z, sc), v3 = taped_bf16(rx[u].v.w, sc);
        if (r < a.nb) {
          st_shared16(row + (((2 * xj) ^ (r & 7)) << 4), make_uint4(v0.x, v0.y, v1.x, v1.y));
          st_shared16(row + (((2 * xj + 1) ^ (r & 7)) << 4), make_uint4(v2.x, v2.y, v3.x, v3.y));
        }
        if (more) rx[u] = load_xu(u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + 8 * st);
      if ((k & 31) == 31)  // two levels: chains of 32 chunks, and of the chains
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          btot[i] += bsum[i];
          bsum[i] = 0.f;
        }
    }
    if (want_db) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s = btot[i] + bsum[i];
#pragma unroll
        for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const int row = o0 + i * 32 + dr;
        if (dj == 0 && row < a.oc) a.db[(long long)split * a.oc + row] = s;
      }
    }
  } else {
    // warp w: rows 32 (w % 4) + lane of the tile, columns 64 (w / 4) ..
    float acc[64];
#pragma unroll
    for (int j = 0; j < 64; ++j) acc[j] = 0.f;
    const int c0 = (warp >> 2) * 64;
    const uint32_t base = tmem + ((uint32_t)(warp & 3) * 32u << 16) + c0;
    bool ok = true;
    for (int w = 0; w < windows && ok; ++w) {
      const int buf = w & 1;
      ok = mbar_wait_sleep(acc_full + 8 * buf, (w >> 1) & 1, abort, a.err, DEV_TIMEOUT_ACC_FULL,
                           a.limit);
      if (!ok) break;
      tc_fence_after();
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c0 + j * 16 < a.nb) {
          const uint32_t at = base + buf * kSets * kN + j * 16;
#pragma unroll
          for (int set = kSets - 1; set >= 0; --set) {
            float v[16];
            tmem_ld16(at + set * kN, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j * 16 + i] += v[i];
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + 8 * buf);
    }
    const int o = o0 + (warp & 3) * 32 + lane;
    if (o < a.oc) {
      float* out = a.dw + ((long long)split * a.oc + o) * a.c + i0 + c0;
#pragma unroll
      for (int j = 0; j < 64; ++j)
        if (i0 + c0 + j < a.c) out[j] = acc[j];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

// out[e] = sum over the splits of part[split][e], in a fixed order
__global__ void __launch_bounds__(256) split_sum_kernel(const float* __restrict__ part, int splits,
                                                        long long n, float* __restrict__ out) {
  __shared__ float red[8][33];
  const int l = threadIdx.x & 31, r = threadIdx.x >> 5;
  for (long long e0 = (long long)blockIdx.x * 32; e0 < n; e0 += (long long)gridDim.x * 32) {
    float s = 0.f;
    if (e0 + l < n)
      for (int k = r; k < splits; k += 8) s += part[k * n + e0 + l];
    __syncthreads();
    red[r][l] = s;
    __syncthreads();
    if (r == 0 && e0 + l < n) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += red[i][l];
      out[e0 + l] = s;
    }
  }
}

// Ranges per tile: the fewest rounds of CTAs over the SMs times the chunks of a range, with a few
// chunks' time for what a CTA does once (start, write its partial tile).
int choose_splits(long long tiles, long long chunks, int sms) {
  long long best = 1;
  double cost = 1e300;
  const long long most = std::min<long long>({chunks, std::max<long long>(1, 4LL * sms / tiles), 1024});
  for (long long s = 1; s <= most; ++s) {
    const double rounds = (double)((tiles * s + sms - 1) / sms);
    const double t = rounds * ((double)((chunks + s - 1) / s) + 4.0) + (s > 1 ? 2.0 : 0.0);
    if (t < cost) cost = t, best = s;
  }
  return (int)best;
}

}  // namespace
}  // namespace zjai

using namespace zjai;

extern "C" int zjai_conv1x1_weight_grad(zjai_ctx* ctx, const void* dout, int dtype, int n, int oc,
                                        int c, int h, int w, const zjai_tape* tape, float* dw,
                                        float* db, int mem) {
  return guarded([&]() -> int {
    const char* me = "conv1x1_weight_grad";
    ZJAI_TRY(ctx_enter(ctx));
    ZJAI_TRY(check_map(me, dtype, n, c, h, w));
    ZJAI_TRY(check_map(me, dtype, n, oc, h, w));
    ZJAI_TRY(check_mem(mem));
    if (!dout || !tape || !tape->codes || !tape->exps || !dw)
      return fail(ZJAI_INVALID_ARGUMENT, std::string(me) + ": null buffer");
    ArenaScope scope(ctx);
    const int p = h * w;
    const size_t es = dtype_size(dtype), groups = tape_groups(p), nw = (size_t)oc * c;
    const char* dd;
    const int8_t *dc, *de;
    float *ow, *ob;
    ZJAI_TRY(stage_bytes_in(ctx, (const char*)dout, (size_t)n * oc * p * es, es, mem, "dout", &dd));
    ZJAI_TRY(stage_bytes_in(ctx, (const int8_t*)tape->codes, (size_t)n * c * p, 1, mem, "codes",
                            &dc));
    ZJAI_TRY(stage_bytes_in(ctx, (const int8_t*)tape->exps, (size_t)n * c * groups, 1, mem, "exps",
                            &de));
    ZJAI_TRY(stage_bytes_out(ctx, dw, nw * 4, 4, mem, "dw", &ow));
    ZJAI_TRY(stage_bytes_out(ctx, db, (size_t)oc * 4, 4, mem, "db", &ob));
    const long long m_tiles = (oc + kM - 1) / kM, n_tiles = (c + kN - 1) / kN;
    const long long tiles = m_tiles * n_tiles;
    if (tiles > 0x7fffffffLL) return fail(ZJAI_LIMIT_EXCEEDED, std::string(me) + ": too many channels");
    auto aligned = [&](const void* q, size_t row) {
      return reinterpret_cast<uintptr_t>(q) % 16 == 0 && row % 16 == 0;
    };
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      using F = Form<T>;
      WgArgs a = {};
      a.dout = dd;
      a.codes = dc;
      a.exps = de;
      a.oc = oc;
      a.c = c;
      a.p = p;
      a.groups = (int)groups;
      a.nb = c >= kN ? kN : (c + 15) / 16 * 16;
      a.m_tiles = (int)m_tiles;
      a.chunks_img = (p + F::kChunk - 1) / F::kChunk;
      a.chunks = (long long)n * a.chunks_img;
      a.splits = choose_splits(tiles, a.chunks, ctx->sms);
      // eight elements at a time: rows of 16 bytes and of eight elements
      a.vec_d = aligned(dd, (size_t)p * es) && p % 8 == 0;
      a.vec_x = aligned(dc, (size_t)p);
      a.dw = ow;
      a.db = ob;
      a.err = ctx->d_err;
      a.limit = ctx->wait_cycles > 0 ? ctx->wait_cycles : kWaitCycles;
      if (a.splits > 1) {
        a.dw = static_cast<float*>(ctx->arena.alloc(a.splits * nw * sizeof(float)));
        if (ob) a.db = static_cast<float*>(ctx->arena.alloc((size_t)a.splits * oc * sizeof(float)));
        if (!a.dw || (ob && !a.db))
          return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (weight gradient)");
      }
      const int smem = 1024 + F::kStages * (F::kTerms + 1) * (F::kChunk / 64) * kBlock;
      ZJAI_TRY(cuda_check(cudaFuncSetAttribute((const void*)weight_grad_kernel<T>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                          me));
      weight_grad_kernel<T><<<dim3((unsigned)tiles, a.splits), kThreads, smem, ctx->stream>>>(a);
      ctx->launches++;
      if (a.splits > 1) {
        auto sum = [&](const float* part, long long e, float* out) {
          const int blocks = (int)std::min<long long>((e + 31) / 32, ctx->sms * 8LL);
          split_sum_kernel<<<blocks, 256, 0, ctx->stream>>>(part, a.splits, e, out);
          ctx->launches++;
        };
        sum(a.dw, (long long)nw, ow);
        if (ob) sum(a.db, oc, ob);
      }
      return cuda_check(cudaGetLastError(), me);
    }));
    ZJAI_TRY(finish_bytes_out(ctx, dw, ow, nw * 4, mem));
    if (ob) ZJAI_TRY(finish_bytes_out(ctx, db, ob, (size_t)oc * 4, mem));
    return finish_call(ctx, mem);
  });
}
