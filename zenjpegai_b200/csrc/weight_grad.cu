// Parameter gradients of a 1x1 convolution from the 8-bit tape of its input
// (zjai_conv1x1_weight_grad): dw[o][i] = sum over pictures and positions of d_out[o] x[i],
// db[o] = sum of d_out[o].
#include <algorithm>

#include "train.h"

namespace zjai {
namespace {

constexpr int kTile = 64;

// One 64 x 64 tile of dw over the split's groups of 32 positions; partial sums per split.
template <class T>
__global__ void __launch_bounds__(256) weight_grad_kernel(const T* __restrict__ dout,
                                                          const int8_t* __restrict__ codes,
                                                          const int8_t* __restrict__ exps, int oc,
                                                          int c, int p, long long groups_all,
                                                          float* __restrict__ dw,
                                                          float* __restrict__ db) {
  __shared__ float ds[kTapeGroup][kTile + 1], xs[kTapeGroup][kTile + 1];
  const int o0 = blockIdx.x * kTile, i0 = blockIdx.y * kTile;
  const int splits = gridDim.z, lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int to = threadIdx.x >> 4, ti = threadIdx.x & 15;
  const int groups = (int)tape_groups(p);
  float acc[4][4] = {}, bacc[4] = {};
  for (long long q = blockIdx.z; q < groups_all; q += splits) {
    const long long img = q / groups;
    const int g = (int)(q - img * groups), at = g * kTapeGroup + lane;
    const bool in = at < p;
    __syncthreads();
    for (int r = wp; r < kTile; r += 8) {
      const long long orow = img * oc + o0 + r, irow = img * c + i0 + r;
      ds[lane][r] = in && o0 + r < oc ? to_f32(dout[orow * p + at]) : 0.f;
      xs[lane][r] = in && i0 + r < c ? (float)codes[irow * p + at] * tape_scale(exps[irow * groups + g])
                                     : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < kTapeGroup; ++k) {
      float d[4], x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d[j] = ds[k][to * 4 + j];
        x[j] = xs[k][ti * 4 + j];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bacc[j] += d[j];
#pragma unroll
        for (int l = 0; l < 4; ++l) acc[j][l] = fmaf(d[j], x[l], acc[j][l]);
      }
    }
  }
  float* w = dw + (long long)blockIdx.z * oc * c;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int o = o0 + to * 4 + j;
    if (o >= oc) continue;
#pragma unroll
    for (int l = 0; l < 4; ++l)
      if (i0 + ti * 4 + l < c) w[(long long)o * c + i0 + ti * 4 + l] = acc[j][l];
    if (blockIdx.y == 0 && ti == 0) db[(long long)blockIdx.z * oc + o] = bacc[j];
  }
}

// out[e] = sum over the splits of part[split][e], in order
__global__ void __launch_bounds__(256) split_sum_kernel(const float* __restrict__ part, int splits,
                                                        long long n, float* __restrict__ out) {
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < n;
       e += (long long)gridDim.x * blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += part[k * n + e];
    out[e] = s;
  }
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
    const int mt = (oc + kTile - 1) / kTile, nt = (c + kTile - 1) / kTile;
    if (nt > 65535) return fail(ZJAI_UNSUPPORTED, std::string(me) + ": too many channels");
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
    const long long groups_all = (long long)n * (long long)groups;
    const long long tiles = (long long)mt * nt;
    const int splits = (int)std::max<long long>(
        1, std::min<long long>({groups_all, (4LL * ctx->sms + tiles - 1) / tiles, 65535LL}));
    float* part = static_cast<float*>(ctx->arena.alloc(splits * nw * sizeof(float)));
    float* bpart = static_cast<float*>(ctx->arena.alloc((size_t)splits * oc * sizeof(float)));
    if (!part || !bpart) return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (weight gradient)");
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      weight_grad_kernel<T><<<dim3(mt, nt, splits), 256, 0, ctx->stream>>>(
          (const T*)dd, dc, de, oc, c, p, groups_all, part, bpart);
      return cuda_check(cudaGetLastError(), me);
    }));
    auto blocks = [&](long long e) { return (int)std::min<long long>((e + 255) / 256, ctx->sms * 8LL); };
    split_sum_kernel<<<blocks((long long)nw), 256, 0, ctx->stream>>>(part, splits, (long long)nw, ow);
    if (ob) split_sum_kernel<<<blocks(oc), 256, 0, ctx->stream>>>(bpart, splits, oc, ob);
    ctx->launches += ob ? 3 : 2;
    ZJAI_TRY(cuda_check(cudaGetLastError(), me));
    ZJAI_TRY(finish_bytes_out(ctx, dw, ow, nw * 4, mem));
    if (ob) ZJAI_TRY(finish_bytes_out(ctx, db, ob, (size_t)oc * 4, mem));
    return finish_call(ctx, mem);
  });
}
