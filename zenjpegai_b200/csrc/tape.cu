// 8-bit activation tapes (zjai_tape_pack, zjai_tape_unpack): the format is in tape.cuh. Both
// directions are one pass over the map, bound by HBM: per element the map's 4 or 2 bytes plus
// 1 + 1/32 for the tape.
//
// Rows of whole groups lie one behind the other, so the map is one run of groups: a thread has eight
// neighbouring positions (four lanes a group) and several such pieces in flight, all accesses 8 or
// 16 bytes (the flat kernels). Other rows end in a short group and start anywhere: eight lanes a
// group, four positions each (the row kernels).
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

// the group of eight lanes: rows of any length
template <bool kVec, class T>
__global__ void __launch_bounds__(256) tape_pack_kernel(const T* __restrict__ x, long long rows,
                                                        int p, zjai_tape t) {
  const int groups = (int)tape_groups(p);
  const long long total = rows * groups;
  const long long first = (long long)blockIdx.x * 32 + (threadIdx.x >> 5) * 4;  // of the warp
  for (long long q0 = first; q0 < total; q0 += (long long)gridDim.x * 32) {
    const long long q = q0 + ((threadIdx.x & 31) >> 3);
    const bool on = q < total;
    const long long row = on ? q / groups : 0;
    const int g = on ? (int)(q - row * groups) : 0, at = g * kTapeGroup + (threadIdx.x & 7) * 4;
    const F4 v = on ? load4<kVec>(x + row * p, at, p) : all(0.f);
    tape_store4<kVec>(t, row * p, q, at, p, v, on);
  }
}

template <bool kVec, class T>
__global__ void __launch_bounds__(256) tape_unpack_kernel(const zjai_tape t, long long rows, int p,
                                                          T* __restrict__ x) {
  const int groups = (int)tape_groups(p);
  const long long total = rows * groups;
  for (long long q = (long long)blockIdx.x * 32 + (threadIdx.x >> 3); q < total;
       q += (long long)gridDim.x * 32) {
    const long long row = q / groups;
    const int g = (int)(q - row * groups), at = g * kTapeGroup + (threadIdx.x & 7) * 4;
    const uint32_t w = load_codes<kVec>(t.codes + row * p, at, p);
    store4<kVec>(x + row * p, at, p, taped4(w, __ldg(t.exps + q)));
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
        const bool vec = p % 4 == 0 && aligned_to(dx, 4 * es) && aligned_to(dc, 4);
        auto k = vec ? tape_pack_kernel<true, T> : tape_pack_kernel<false, T>;
        k<<<row_blocks(ctx, (long long)ng), 256, 0, ctx->stream>>>(tx, (long long)rows, p,
                                                                   zjai_tape{dc, de});
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
      T* tx = reinterpret_cast<T*>(dx);
      const long long pieces = (long long)(ne / 8);
      if (p % kTapeGroup == 0 && aligned_to(dx, 16) && aligned_to(dc, 8)) {
        const unsigned blocks = (unsigned)((pieces + kFlatBlock - 1) / kFlatBlock);
        tape_unpack_flat_kernel<T><<<blocks, 256, 0, ctx->stream>>>(dc, de, pieces, tx);
      } else {
        const bool vec = p % 4 == 0 && aligned_to(dx, 4 * es) && aligned_to(dc, 4);
        auto k = vec ? tape_unpack_kernel<true, T> : tape_unpack_kernel<false, T>;
        k<<<row_blocks(ctx, (long long)ng), 256, 0, ctx->stream>>>(
            zjai_tape{const_cast<int8_t*>(dc), const_cast<int8_t*>(de)}, (long long)rows, p, tx);
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
