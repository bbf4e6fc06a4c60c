// 8-bit activation tapes (zjai_tape_pack, zjai_tape_unpack): the format is in tape.cuh. Both
// directions are one pass over the map, bound by HBM: per element the map's 4 or 2 bytes plus
// 1 + 1/32 for the tape.
#include <algorithm>

#include "train.h"

namespace zjai {
namespace {

// One warp per group: a lane's position, the group's largest magnitude by one warp reduction.
template <class T>
__global__ void __launch_bounds__(256) tape_pack_kernel(const T* __restrict__ x, long long rows,
                                                        int p, int8_t* __restrict__ codes,
                                                        int8_t* __restrict__ exps) {
  const int lane = threadIdx.x & 31;
  const long long groups = tape_groups(p), total = rows * groups;
  for (long long g = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); g < total;
       g += (long long)gridDim.x * 8) {
    const long long row = g / groups;
    const int at = (int)(g - row * groups) * kTapeGroup + lane;
    const bool in = at < p;
    const float v = in ? to_f32(x[row * p + at]) : 0.f;
    const int e = tape_exp(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
    const uint32_t code = e == kTapeNan ? 0u : tape_code_bits(v, tape_inv_scale(e));
    if (in) codes[row * p + at] = (int8_t)(code & 0xffu);
    if (lane == 0) exps[g] = (int8_t)e;
  }
}

template <class T>
__global__ void __launch_bounds__(256) tape_unpack_kernel(const int8_t* __restrict__ codes,
                                                          const int8_t* __restrict__ exps,
                                                          long long rows, int p,
                                                          T* __restrict__ x) {
  const int lane = threadIdx.x & 31;
  const long long groups = tape_groups(p), total = rows * groups;
  for (long long g = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); g < total;
       g += (long long)gridDim.x * 8) {
    const long long row = g / groups;
    const int at = (int)(g - row * groups) * kTapeGroup + lane;
    if (at < p) x[row * p + at] = from_f32<T>((float)codes[row * p + at] * tape_scale(exps[g]));
  }
}

int row_blocks(Ctx* ctx, long long total) {
  return (int)std::max<long long>(1, std::min<long long>((total + 7) / 8, (long long)ctx->sms * 16));
}

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
      tape_pack_kernel<T><<<row_blocks(ctx, (long long)ng), 256, 0, ctx->stream>>>(
          reinterpret_cast<const T*>(dx), (long long)rows, p, dc, de);
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
      tape_unpack_kernel<T><<<row_blocks(ctx, (long long)ng), 256, 0, ctx->stream>>>(
          dc, de, (long long)rows, p, reinterpret_cast<T*>(dx));
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
