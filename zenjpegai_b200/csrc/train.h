// Shared by the entries of the training operators (tape.cu, residual_norm.cu, weight_grad.cu):
// checks of maps, staging of host and device buffers of any element type, dispatch on the type.
#pragma once
#include <new>
#include <string>

#include "api_common.h"
#include "tape.cuh"

namespace zjai {

inline size_t dtype_size(int dtype) { return dtype == ZJAI_F32 ? 4 : 2; }

// n, c, h, w >= 1 and small enough that rows (n c) and positions (h w, rounded up to groups and
// tiles) fit an int; the element count fits 2^40.
inline int check_map(const char* what, int dtype, int n, int c, int h, int w) {
  if (dtype != ZJAI_F32 && dtype != ZJAI_F16 && dtype != ZJAI_BF16)
    return fail(ZJAI_INVALID_ARGUMENT, std::string(what) + ": dtype must be f32, f16 or bf16");
  if (n <= 0 || c <= 0 || h <= 0 || w <= 0)
    return fail(ZJAI_INVALID_ARGUMENT, std::string(what) + ": extents must be positive");
  const long long p = (long long)h * w, rows = (long long)n * c;
  if (p > 0x7fffffffLL - 64 || rows > 0x7fffffffLL || p > (1LL << 40) / rows)
    return fail(ZJAI_LIMIT_EXCEEDED, std::string(what) + ": map too large");
  return ZJAI_OK;
}
inline int check_mem(int mem) {
  if (mem != ZJAI_MEM_HOST && mem != ZJAI_MEM_DEVICE)
    return fail(ZJAI_INVALID_ARGUMENT, "mem must be HOST or DEVICE");
  return ZJAI_OK;
}
// A caller's device buffer: addressable by the context's GPU and aligned to its element.
inline int check_aligned(Ctx* ctx, const void* p, size_t align, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) % align)
    return fail(ZJAI_INVALID_ARGUMENT, std::string(what) + ": not aligned to its element");
  return check_device_buffer(ctx, p, what);
}
// Device pointer of `bytes` of a caller's input. NULL stays NULL (the caller has checked that it
// may be).
template <class T>
int stage_bytes_in(Ctx* ctx, const T* p, size_t bytes, size_t align, int mem, const char* what,
                   const T** out) {
  *out = nullptr;
  if (!p) return ZJAI_OK;
  if (mem == ZJAI_MEM_DEVICE) {
    ZJAI_TRY(check_aligned(ctx, p, align, what));
    *out = p;
    return ZJAI_OK;
  }
  void* d = ctx->arena.alloc(bytes);
  if (!d) return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (input staging)");
  ZJAI_TRY(cuda_check(cudaMemcpyAsync(d, p, bytes, cudaMemcpyHostToDevice, ctx->stream), "H2D"));
  *out = static_cast<const T*>(d);
  return ZJAI_OK;
}
template <class T>
int stage_bytes_out(Ctx* ctx, T* p, size_t bytes, size_t align, int mem, const char* what,
                    T** dev) {
  *dev = nullptr;
  if (!p) return ZJAI_OK;
  if (mem == ZJAI_MEM_DEVICE) {
    ZJAI_TRY(check_aligned(ctx, p, align, what));
    *dev = p;
    return ZJAI_OK;
  }
  *dev = static_cast<T*>(ctx->arena.alloc(bytes));
  if (!*dev) return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (output staging)");
  return ZJAI_OK;
}
inline int finish_bytes_out(Ctx* ctx, void* host, const void* dev, size_t bytes, int mem) {
  if (mem == ZJAI_MEM_DEVICE || !host) return ZJAI_OK;
  return cuda_check(cudaMemcpyAsync(host, dev, bytes, cudaMemcpyDeviceToHost, ctx->stream), "D2H");
}

// f(T()) with the element type of `dtype` (checked before)
template <class F>
int by_dtype(int dtype, F&& f) {
  if (dtype == ZJAI_F32) return f(float());
  if (dtype == ZJAI_F16) return f(__half());
  return f(__nv_bfloat16());
}

// No C++ exception leaves a C entry: host allocations of messages and the like are all that throw.
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return ZJAI_LIMIT_EXCEEDED;
  } catch (...) {
    return ZJAI_DEVICE;
  }
}

}  // namespace zjai
