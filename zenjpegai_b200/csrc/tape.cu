// 8-bit activation tapes (zjai_tape_pack, zjai_tape_unpack): the format is in tape.cuh. Both
// directions are one pass over the map, bound by HBM: per element the map's 4 or 2 bytes plus
// 1 + 1/32 for the tape. 28 x 1024 x 128^2 f16, packed and unpacked: 429 to 439 us, 6.5 TB/s and more,
// the speed of a plain copy.
//
// Groups lie one behind the other in memory. Where all are whole (rows of a multiple of 32
// positions) a thread has eight neighbouring positions (four lanes a group) and several such pieces
// in flight, all accesses 8 or 16 bytes (the flat kernels). Other rows end in a short group and start
// anywhere. Packing, a block copies its run of groups to shared memory by aligned 16 bytes, works on
// it with eight lanes a group, and stores the codes by 16 bytes again. Unpacking, a lane has four
// neighbouring elements, whatever groups they are of. (With eight lanes a group at global memory
// both calls together took 51 us on f32, 8 x 128 x 127 x 129, and 52 us on f16; now 46 and 43, of which
// the kernels take 24 and 18 in either type: instructions bound them, not the bytes' 26 and 16 us.)
#include <algorithm>

#include "quad.cuh"
#include "train.h"

namespace zjai {
namespace {

constexpr int kPieces = 4;  // of 8 positions per thread of the flat kernels
constexpr int kFlatBlock = 256 * kPieces;

// eight positions, as two quads, from aligned memory
template <class T>
__device__ __forceinline__ void load8(const T* q, F4* lo, F4* hi) {
  if constexpr (sizeof(T) == 4) {
    *lo = make4(__ldg(reinterpret_cast<const float4*>(q)));
    *hi = make4(__ldg(reinterpret_cast<const float4*>(q) + 1));
  } else {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q));
    *lo = halves4<T>(make_uint2(w.x, w.y));
    *hi = halves4<T>(make_uint2(w.z, w.w));
  }
}
template <class T>
__device__ __forceinline__ void store8(T* q, F4 lo, F4 hi) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(q)[0] = flat(lo);
    reinterpret_cast<float4*>(q)[1] = flat(hi);
  } else {
    const uint2 a = words2<T>(lo), b = words2<T>(hi);
    *reinterpret_cast<uint4*>(q) = make_uint4(a.x, a.y, b.x, b.y);
  }
}

template <class T>
__global__ void __launch_bounds__(256) tape_pack_flat_kernel(const T* __restrict__ x,
                                                             long long pieces,
                                                             int8_t* __restrict__ codes,
                                                             int8_t* __restrict__ exps) {
  const long long i0 = (long long)blockIdx.x * kFlatBlock + threadIdx.x;
  F4 v[kPieces][2];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long i = i0 + k * 256;
    v[k][0] = v[k][1] = all(0.f);
    if (i < pieces) load8(x + i * 8, &v[k][0], &v[k][1]);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long i = i0 + k * 256;
    uint32_t m = max(amax4(v[k][0]), amax4(v[k][1]));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint2 w = make_uint2(codes4(v[k][0], m), codes4(v[k][1], m));
    if (i >= pieces) continue;
    *reinterpret_cast<uint2*>(codes + i * 8) = w;
    if ((threadIdx.x & 3) == 0) exps[i >> 2] = (int8_t)tape_exp(m);
  }
}

template <class T>
__global__ void __launch_bounds__(256) tape_unpack_flat_kernel(const int8_t* __restrict__ codes,
                                                               const int8_t* __restrict__ exps,
                                                               long long pieces,
                                                               T* __restrict__ x) {
  const long long i0 = (long long)blockIdx.x * kFlatBlock + threadIdx.x;
  uint2 w[kPieces];
  int e[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long i = i0 + k * 256;
    if (i >= pieces) continue;
    w[k] = __ldg(reinterpret_cast<const uint2*>(codes + i * 8));
    e[k] = __ldg(exps + (i >> 2));
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long i = i0 + k * 256;
    if (i < pieces) store8(x + i * 8, taped4(w[k].x, e[k]), taped4(w[k].y, e[k]));
  }
}

// n / d for n < 2^31, by a multiplication (Granlund and Montgomery, "Division by invariant integers
// using multiplication", 1994: the quotient's multiplier has 33 bits, its top one added as n)
struct Div {
  uint32_t magic, shift, d;
  explicit Div(uint32_t d_) : shift(0), d(d_) {
    while ((1ull << shift) < d) ++shift;
    magic = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const {
    return (__umulhi(n, magic) + n) >> shift;
  }
};

constexpr int kRunGroups = 128;  // of a block
// Rows of any length, bases of any alignment. The aligned 16 bytes that hold the run's first and
// last elements may reach beyond the map, but lie in one granule of memory with them.
template <class T>
__global__ void __launch_bounds__(256) tape_pack_kernel(const T* __restrict__ x, long long total,
                                                        int p, Div groups, zjai_tape t) {
  constexpr int kMost = kRunGroups * kTapeGroup;
  __shared__ __align__(16) char xs[kMost * sizeof(T) + 32];
  __shared__ __align__(16) char cs[kMost + 32];
  const long long q0 = (long long)blockIdx.x * kRunGroups, q1 = min(q0 + kRunGroups, total);
  auto start = [&](long long q) {
    const long long row = q / groups.d;
    return row * p + (q - row * groups.d) * kTapeGroup;
  };
  const long long s0 = start(q0);
  const int n = (int)(start(q1) - s0);  // elements
  const uint32_t g0 = (uint32_t)(q0 % groups.d);
  const int xhead = (int)(reinterpret_cast<uintptr_t>(x + s0) & 15);
  const int chead = (int)(reinterpret_cast<uintptr_t>(t.codes + s0) & 15);
  const char* from = reinterpret_cast<const char*>(x + s0) - xhead;
  for (int i = threadIdx.x * 16; i < xhead + n * (int)sizeof(T); i += 256 * 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(xs + i)),
                 "l"(from + i)
                 : "memory");
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  const T* mine = reinterpret_cast<const T*>(xs + xhead);
#pragma unroll
  for (int k = 0; k < kRunGroups / 32; ++k) {
    const int lq = k * 32 + (threadIdx.x >> 3), at = (threadIdx.x & 7) * 4;
    const uint32_t r = groups.of(g0 + lq), g = g0 + lq - r * groups.d;
    const int left = q0 + lq < q1 ? p - (int)g * kTapeGroup : 0;  // of the row, from the group on
    const int first = (int)r * p + ((int)g - (int)g0) * kTapeGroup + at;
    // the four groups of a warp take their lanes' elements in turned orders: no bank is met twice
    float v[4];
    const int turn = (threadIdx.x >> 3) & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = (i + turn) & 3;
      v[i] = u + at < left ? to_f32(mine[first + u]) : 0.f;
    }
    const F4 f = {make_float2(v[0], v[1]), make_float2(v[2], v[3])};
    uint32_t m = amax4(f);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t w = codes4(f, m);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = (i + turn) & 3;
      if (u + at < left) cs[chead + first + u] = (char)(w >> 8 * i);
    }
    if ((threadIdx.x & 7) == 0 && left > 0) t.exps[q0 + lq] = (int8_t)tape_exp(m);
  }
  __syncthreads();
  char* to = reinterpret_cast<char*>(t.codes + s0) - chead;
  for (int i = threadIdx.x * 16; i < chead + n; i += 256 * 16) {
    if (i >= chead && i + 16 <= chead + n) {
      *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(cs + i);
    } else {
      for (int b = max(i, chead); b < min(i + 16, chead + n); ++b) to[b] = cs[b];
    }
  }
}

// Rows of any length, x aligned to four elements, codes to four bytes.
template <class T>
__global__ void __launch_bounds__(256) tape_unpack_quads_kernel(const zjai_tape t, long long ne,
                                                                long long total, int p, Div by_p,
                                                                T* __restrict__ x) {
  const long long b0 = (long long)blockIdx.x * (256 * 4 * kPieces);
  const long long row0 = b0 / p;
  const uint32_t pos0 = (uint32_t)(b0 - row0 * p);
  const uint32_t groups = (uint32_t)tape_groups(p);
  const int8_t* exps = t.exps + row0 * groups;
  uint32_t w[kPieces];
  int e0[kPieces], e1[kPieces], nb[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const uint32_t i = (k * 256 + threadIdx.x) * 4;
    const uint32_t r = by_p.of(pos0 + i), pos = pos0 + i - r * (uint32_t)p, g = pos / kTapeGroup;
    const long long left = ne - b0 - i;
    nb[k] = min(kTapeGroup - (int)(pos % kTapeGroup), p - (int)pos);  // in the first one's group
    const long long q = (long long)r * groups + g;
    w[k] = 0, e0[k] = e1[k] = 0;
    if (left >= 4) w[k] = __ldg(reinterpret_cast<const uint32_t*>(t.codes + b0 + i));
    if (left > 0) e0[k] = __ldg(exps + q);
    if (left > 0 && nb[k] < 4 && row0 * groups + q + 1 < total) e1[k] = __ldg(exps + q + 1);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const uint32_t i = (k * 256 + threadIdx.x) * 4;
    const long long left = ne - b0 - i;
    F4 v = taped4(w[k], e0[k]);
    if (nb[k] < 4) {
      const F4 u = taped4(w[k], e1[k]);
      if (nb[k] <= 1) v.a.y = u.a.y;
      if (nb[k] <= 2) v.b.x = u.b.x;
      v.b.y = u.b.y;
    }
    // a third group (a short last one between), or the map's end: each element by itself
    const uint32_t r = by_p.of(pos0 + i);
    const int pos = (int)(pos0 + i - r * (uint32_t)p) + nb[k];  // behind the first group
    const int second = pos == p ? min(p, kTapeGroup) : min(p - pos, kTapeGroup);
    if (left >= 4 && nb[k] + second >= 4) {
      store4_in(x + b0 + i, v);
    } else {
      for (int j = 0; j < 4 && j < left; ++j) {
        const uint32_t rj = by_p.of(pos0 + i + j), pj = pos0 + i + j - rj * (uint32_t)p;
        const int ej = __ldg(exps + (long long)rj * groups + pj / kTapeGroup);
        const uint32_t c = (uint8_t)__ldg(t.codes + b0 + i + j);
        x[b0 + i + j] = from_f32<T>(taped4(c, ej).a.x);
      }
    }
  }
}

// Any alignment: the group of eight lanes.
template <class T>
__global__ void __launch_bounds__(256) tape_unpack_kernel(const zjai_tape t, long long rows, int p,
                                                          T* __restrict__ x) {
  const int groups = (int)tape_groups(p);
  const long long total = rows * groups;
  for (long long q = (long long)blockIdx.x * 32 + (threadIdx.x >> 3); q < total;
       q += (long long)gridDim.x * 32) {
    const long long row = q / groups;
    const int g = (int)(q - row * groups), at = g * kTapeGroup + (threadIdx.x & 7) * 4;
    const uint32_t w = load_codes<false>(t.codes + row * p, at, p);
    store4<false>(x + row * p, at, p, taped4(w, __ldg(t.exps + q)));
  }
}

int row_blocks(Ctx* ctx, long long groups) {
  return (int)std::max<long long>(1,
                                  std::min<long long>((groups + 31) / 32, (long long)ctx->sms * 8));
}
bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace zjai

using namespace zjai;

extern "C" {

int zjai_tape_pack(zjai_ctx* ctx, const void* x, int dtype, int n, int c, int h, int w,
                   const zjai_tape* tape, int mem) {
  return guarded([&]() -> int {
    ZJAI_TRY(ctx_enter(ctx));
    ZJAI_TRY(check_map("tape_pack", dtype, n, c, h, w));
    ZJAI_TRY(check_mem(mem));
    if (!x || !tape || !tape->codes || !tape->exps)
      return fail(ZJAI_INVALID_ARGUMENT, "tape_pack: null buffer");
    ArenaScope scope(ctx);
    const int p = h * w;
    const size_t rows = (size_t)n * c, ne = rows * p, ng = rows * tape_groups(p);
    const size_t es = dtype_size(dtype);
    const char* dx;
    int8_t *dc, *de;
    ZJAI_TRY(stage_bytes_in(ctx, static_cast<const char*>(x), ne * es, es, mem, "x", &dx));
    ZJAI_TRY(stage_bytes_out(ctx, tape->codes, ne, 1, mem, "codes", &dc));
    ZJAI_TRY(stage_bytes_out(ctx, tape->exps, ng, 1, mem, "exps", &de));
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      const T* tx = reinterpret_cast<const T*>(dx);
      const long long pieces = (long long)(ne / 8);
      if (p % kTapeGroup == 0 && aligned_to(dx, 16) && aligned_to(dc, 8)) {
        const unsigned blocks = (unsigned)((pieces + kFlatBlock - 1) / kFlatBlock);
        tape_pack_flat_kernel<T><<<blocks, 256, 0, ctx->stream>>>(tx, pieces, dc, de);
      } else {
        const unsigned blocks = (unsigned)((ng + kRunGroups - 1) / kRunGroups);
        tape_pack_kernel<T><<<blocks, 256, 0, ctx->stream>>>(
            tx, (long long)ng, p, Div((uint32_t)tape_groups(p)), zjai_tape{dc, de});
      }
      return cuda_check(cudaGetLastError(), "tape_pack");
    }));
    ctx->launches++;
    ZJAI_TRY(finish_bytes_out(ctx, tape->codes, dc, ne, mem));
    ZJAI_TRY(finish_bytes_out(ctx, tape->exps, de, ng, mem));
    return finish_call(ctx, mem);
  });
}

int zjai_tape_unpack(zjai_ctx* ctx, const zjai_tape* tape, int n, int c, int h, int w, void* x,
                     int dtype, int mem) {
  return guarded([&]() -> int {
    ZJAI_TRY(ctx_enter(ctx));
    ZJAI_TRY(check_map("tape_unpack", dtype, n, c, h, w));
    ZJAI_TRY(check_mem(mem));
    if (!x || !tape || !tape->codes || !tape->exps)
      return fail(ZJAI_INVALID_ARGUMENT, "tape_unpack: null buffer");
    ArenaScope scope(ctx);
    const int p = h * w;
    const size_t rows = (size_t)n * c, ne = rows * p, ng = rows * tape_groups(p);
    const size_t es = dtype_size(dtype);
    const int8_t *dc, *de;
    char* dx;
    ZJAI_TRY(stage_bytes_in(ctx, (const int8_t*)tape->codes, ne, 1, mem, "codes", &dc));
    ZJAI_TRY(stage_bytes_in(ctx, (const int8_t*)tape->exps, ng, 1, mem, "exps", &de));
    ZJAI_TRY(stage_bytes_out(ctx, static_cast<char*>(x), ne * es, es, mem, "x", &dx));
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      const zjai_tape t8 = {const_cast<int8_t*>(dc), const_cast<int8_t*>(de)};
      T* tx = reinterpret_cast<T*>(dx);
      const long long pieces = (long long)(ne / 8);
      if (p % kTapeGroup == 0 && aligned_to(dx, 16) && aligned_to(dc, 8)) {
        const unsigned blocks = (unsigned)((pieces + kFlatBlock - 1) / kFlatBlock);
        tape_unpack_flat_kernel<T><<<blocks, 256, 0, ctx->stream>>>(dc, de, pieces, tx);
      } else if (aligned_to(dx, 4 * es) && aligned_to(dc, 4)) {
        const unsigned blocks = (unsigned)((ne + 1024 * kPieces - 1) / (1024 * kPieces));
        tape_unpack_quads_kernel<T><<<blocks, 256, 0, ctx->stream>>>(
            t8, (long long)ne, (long long)ng, p, Div((uint32_t)p), tx);
      } else {
        tape_unpack_kernel<T>
            <<<row_blocks(ctx, (long long)ng), 256, 0, ctx->stream>>>(t8, (long long)rows, p, tx);
      }
      return cuda_check(cudaGetLastError(), "tape_unpack");
    }));
    ctx->launches++;
    ZJAI_TRY(finish_bytes_out(ctx, x, dx, ne * es, mem));
    return finish_call(ctx, mem);
  });
}

int zjai_ctx_wait_stream(zjai_ctx* ctx, void* cuda_stream) {
  ZJAI_TRY(ctx_enter(ctx));
  cudaStream_t s = cuda_stream ? static_cast<cudaStream_t>(cuda_stream) : cudaStreamLegacy;
  if (s == ctx->stream) return ZJAI_OK;
  ZJAI_TRY(cuda_check(cudaEventRecord(ctx->ev_caller, s), "caller stream"));
  return cuda_check(cudaStreamWaitEvent(ctx->stream, ctx->ev_caller, 0), "caller stream");
}

int zjai_ctx_release_stream(zjai_ctx* ctx, void* cuda_stream) {
  ZJAI_TRY(ctx_enter(ctx));
  cudaStream_t s = cuda_stream ? static_cast<cudaStream_t>(cuda_stream) : cudaStreamLegacy;
  if (s == ctx->stream) return ZJAI_OK;
  ZJAI_TRY(cuda_check(cudaEventRecord(ctx->ev_caller, ctx->stream), "caller stream"));
  return cuda_check(cudaStreamWaitEvent(s, ctx->ev_caller, 0), "caller stream");
}

}  // extern "C"
