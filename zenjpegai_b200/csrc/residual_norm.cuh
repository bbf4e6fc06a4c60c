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
// three times the instructions, and issue slots bounded the kernels, not HBM). A block takes up to
// 256 channels, four rows a thread, and a cluster of up to eight blocks up to 2048, reading the
// partial sums of each other's shared memory. Everything is read once, copied to shared memory a
// tile ahead (the staged kernels). More channels are read again for each pass. A position's sums go
// over the warps' shared-memory partials, gathered by four lanes each. Statistics: a mean and sum of
// squared deviations per warp, joined by their exact update formula (sums of squares would cancel).
// The products in a - mean a and b - mean b are the ones that were summed (not fused): with one
// channel they cancel to zero.
// Measured at 28 x 128 x 128^2 with a full gate, kernels alone: f32 forward with four tapes 285 us,
// 5.0 TB/s, and backward from tapes 428 us, 3.2 TB/s: the sixteen warps an SM that the registers
// leave issue every other cycle, each waiting on its own latencies between the exchanges. So bf16,
// with half of the bytes and the same instructions, is hardly faster: forward without tapes 173 us
// (f32 195), backward 383 us.
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
constexpr int kBlockC = kMaxWarps * 4 * kStagedRows;  // channels of a block
constexpr int kMaxCluster = 8;

// sigmoid(g) and sigmoid(g) (1 - sigmoid(g)), an even function of g: with a = exp(-|g|) and
// r = 1 / (1 + a), sigmoid is r or a r and the product a r^2, nothing by cancellation and both finite
// for every g but NaN. __expf's documented error is 2 + floor(1.16 |g|) units in the last place: where
// it grows, at large |g|, what carries it (sigmoid's small side, the slope) is as small as exp(-|g|)
// itself: at |g| = 20 some 25 units, 3e-6 of values of 2e-9. expf took 2 to 6 % longer (28 x 128 x
// 128^2, full gate, a call: f32 forward with tapes read back 402 and 412 us, backward 437 and 449; bf16
// forward 171 and 182, backward 384 and 402). __fdividef's two units are as many as the sums' own.
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

// A cluster of blocks that share a tile's channels (one block: no cluster instruction runs).
struct Cluster {
  int size, rank;
  __device__ __forceinline__ explicit Cluster(int size_) : size(size_), rank(0) {
    if (size > 1) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  }
  __device__ __forceinline__ void sync() const {
    if (size > 1)
      asm volatile(
          "barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
              : "memory");
    else
      __syncthreads();
  }
  // *q of the block with this rank (kMany: a cluster of more than one)
  template <bool kMany>
  static __device__ __forceinline__ float read(const float* q, int of) {
    if (!kMany) return *q;
    float v;
    asm volatile(
        "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\t"
        "ld.shared::cluster.f32 %0, [a];\n\t}"
        : "=f"(v)
        : "r"((uint32_t)__cvta_generic_to_shared(q)), "r"(of)
        : "memory");
    return v;
  }
};

// The block's partial sums per warp and position, and their totals: written by the warps, cl.sync(),
// joined, cl.sync() (no block sums them any more). Then a warp may use its own as scratch.
constexpr int kScratchBytes = 256;  // of a warp, from at(0, warp) on: 128 halves
template <int kVals>
struct Exchange {
  static constexpr int kPitch = kVals * 32 + 8;  // per warp; the lanes of a join meet no bank twice
  static_assert(kScratchBytes <= kPitch * (int)sizeof(float), "scratch reaches the next warp's sums");
  float *part, *totals;
  __device__ __forceinline__ float* at(int val, int w) const { return part + w * kPitch + val * 32; }
  __device__ __forceinline__ float* total(int val) const { return totals + val * 32; }
};

// Rows of the calling thread among its block's channels: row(j) for j < n, a warp's consecutive
// groups of four. kRows > 0: as many, held; 0: as many as c takes. kAll: all rows exist. The same
// rows to the same warps either way (up to 2048 channels), so that results do not depend on
// alignment.
template <int kRows, bool kAll = false>
struct Rows {
  int c, first, n, share, all_c;
  // c of the block; channels of every block but the last one of a cluster; channels
  __device__ __forceinline__ Rows(int c_, int share_, int all_c_, int warps)
      : c(c_), share(share_), all_c(all_c_) {
    n = kRows ? kRows : max(kStagedRows, (share + 4 * warps - 1) / (4 * warps));
    first = (threadIdx.x >> 5) * 4 * n + ((threadIdx.x & 31) >> 3);
  }
  __device__ __forceinline__ int row(int j) const { return first + j * 4; }
  __device__ __forceinline__ bool on(int j) const { return kAll || row(j) < c; }
  // a row that exists, to read for one that does not
  __device__ __forceinline__ int param(int j) const { return min(row(j), c - 1); }
  // rows of a warp of a block
  __device__ __forceinline__ int of_warp(int w, int rank) const {
    return kAll ? 4 * kRows : max(0, min(all_c - rank * share - w * 4 * n, 4 * n));
  }
};
#define FOR_ROWS(j) _Pragma("unroll") for (int j = 0; j < (kRows ? kRows : rows.n); ++j)

// Per warp the sum and the squared deviations from the warp's own mean of v(j), to the partials at
// val, val + 1.
template <int kRows, bool kAll, int kVals, class V>
__device__ __forceinline__ void stats_part(const Rows<kRows, kAll>& rows, V&& v,
                                           const Exchange<kVals>& ex, int val, int rank) {
  const int wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  F4 s = all(0.f), q = all(0.f);
  FOR_ROWS(j) if (rows.on(j)) s = s + v(j);
  s = over_rows(s);
  const int n = rows.of_warp(wp, rank);
  const F4 nm = s * all(kAll ? -1.f / (4 * kRows) : n ? __fdividef(-1.f, (float)n) : 0.f);
  FOR_ROWS(j) if (rows.on(j)) {
    const F4 d = v(j) + nm;
    q = fma4(d, d, q);
  }
  if (lane < 8) *reinterpret_cast<float4*>(ex.at(val, wp) + lane * 4) = flat(s);
  rows_to_part(q, ex.at(val + 1, wp));
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
// f of every warp's partials that the caller's lanes join: (warp, block of the cluster)
template <bool kMany, class F>
__device__ __forceinline__ void each_part(int sub, int warps, const Cluster& cl, F&& f) {
#pragma unroll 1
  for (int r = 0; r < (kMany ? cl.size : 1); ++r)
#pragma unroll
    for (int i = 0; i < kMaxWarps / 4; ++i)
      if (i * 4 + sub < warps) f(i * 4 + sub, r);
}
// Joined: the totals at to, to + 1 are the negated mean and 1 / sigma. Partials' means are joined by
// M2 = sum of M2_w + n_w (mean_w - mean)^2.
template <bool kMany, int kRows, bool kAll, int kVals>
__device__ __forceinline__ void stats_join_of(const Rows<kRows, kAll>& rows,
                                              const Exchange<kVals>& ex, int val, int to,
                                              float inv_c, int warps, const Cluster& cl, int nth,
                                              int of) {
  by_position(nth, of, [&](int pos, int sub) {
    float sum = 0.f, q = 0.f;
    each_part<kMany>(sub, warps, cl,
                     [&](int w, int r) { sum += Cluster::read<kMany>(ex.at(val, w) + pos, r); });
    // products rounded on their own: the same bits wherever this is compiled in
    const float m = __fmul_rn(over_subs(sum), inv_c);
    each_part<kMany>(sub, warps, cl, [&](int w, int r) {
      const int n = rows.of_warp(w, r);
      if (!n) return;
      const float s = Cluster::read<kMany>(ex.at(val, w) + pos, r);
      // (whole warps: by a constant)
      const float mean = kAll ? __fmul_rn(s, 1.f / (4 * kRows)) : __fdividef(s, (float)n);
      const float d = __fsub_rn(mean, m);
      q = __fadd_rn(q, fmaf(__fmul_rn((float)n, d), d,
                            Cluster::read<kMany>(ex.at(val + 1, w) + pos, r)));
    });
    q = over_subs(q);
    if (sub == 0) {
      ex.total(to)[pos] = -m;
      ex.total(to + 1)[pos] = rsqrtf(fmaf(q, inv_c, kEps));
    }
  });
}
template <int kRows, bool kAll, int kVals>
__device__ __forceinline__ void stats_join(const Rows<kRows, kAll>& rows,
                                           const Exchange<kVals>& ex, int val, int to, float inv_c,
                                           int warps, const Cluster& cl, int nth, int of) {
  if (cl.size == 1)
    stats_join_of<false>(rows, ex, val, to, inv_c, warps, cl, nth, of);
  else
    stats_join_of<true>(rows, ex, val, to, inv_c, warps, cl, nth, of);
}
template <int kVals>
__device__ __forceinline__ F4 total4(const Exchange<kVals>& ex, int val) {
  return make4(*reinterpret_cast<const float4*>(ex.total(val) + (threadIdx.x & 7) * 4));
}
// Sums over the warps of the partials at val, times k, to the total at to.
template <bool kMany, int kVals>
__device__ __forceinline__ void sum_join_of(const Exchange<kVals>& ex, int val, int to, float k,
                                            int warps, const Cluster& cl, int nth, int of) {
  by_position(nth, of, [&](int pos, int sub) {
    float s = 0.f;
    each_part<kMany>(sub, warps, cl,
                     [&](int w, int r) { s += Cluster::read<kMany>(ex.at(val, w) + pos, r); });
    s = over_subs(s);
    if (sub == 0) ex.total(to)[pos] = s * k;
  });
}
template <int kVals>
__device__ __forceinline__ void sum_join(const Exchange<kVals>& ex, int val, int to, float k,
                                         int warps, const Cluster& cl, int nth, int of) {
  if (cl.size == 1)
    sum_join_of<false>(ex, val, to, k, warps, cl, nth, of);
  else
    sum_join_of<true>(ex, val, to, k, warps, cl, nth, of);
}

// The parameters of a channel in all four positions: doubled in shared memory where rows are held,
// else from global memory. Absent ones are those of the identity.
enum { kPostW, kPostB, kScale, kPreW, kPreB, kParams };
template <int kRows>
struct Params {
  float2* v;  // [kParams][share], where rows are held
  int share;
  static __device__ __forceinline__ const float* of(const zjai_residual_params& p, int k) {
    return k == kPostW ? p.post_weight : k == kPostB ? p.post_bias : k == kScale ? p.scale
           : k == kPreW ? p.pre_weight : p.pre_bias;
  }
  static __device__ __forceinline__ float one(const zjai_residual_params& p, int k, int ch) {
    const float* q = of(p, k);
    return q ? __ldg(q + ch) : (k == kPostB || k == kPreB ? 0.f : 1.f);
  }
  // of c channels from ch0 on
  __device__ __forceinline__ void load(const zjai_residual_params& p, int ch0, int c) {
    for (int i = threadIdx.x; i < kParams * c; i += blockDim.x) {
      const float x = one(p, i / c, ch0 + i % c);
      v[i / c * share + i % c] = make_float2(x, x);
    }
  }
  __device__ __forceinline__ F4 get(const zjai_residual_params& p, int k, int ch) const {
    if (!kRows) return all(one(p, k, ch));
    const float2 x = v[k * share + ch];
    return {x, x};
  }
};

constexpr int kThreadsMost = 32 * kMaxWarps;
// The shared memory behind the slots of a staged kernel: parameters and partial sums.
template <int kVals>
constexpr int tail_bytes(int share, int warps) {
  return kParams * share * (int)sizeof(float2) +
         warps * Exchange<kVals>::kPitch * (int)sizeof(float);
}
template <int kVals>
__device__ __forceinline__ void take_tail(char* tail, int share, float2** params,
                                          Exchange<kVals>* ex) {
  *params = reinterpret_cast<float2*>(tail);
  ex->part = reinterpret_cast<float*>(*params + kParams * share);
}
// The tiles of a block or cluster, one after the other: picture and group of positions, without a
// division.
struct Tiles {
  int img, g, groups, step_img, step_g;
  long long left;  // tiles from the current one on, of the whole grid
  unsigned step;
  __device__ __forceinline__ Tiles(long long tiles, int groups_, int cluster) : groups(groups_) {
    const unsigned first = blockIdx.x / (unsigned)cluster;
    step = gridDim.x / (unsigned)cluster;
    img = (int)(first / (unsigned)groups);
    g = (int)(first - (unsigned)img * groups);
    step_img = (int)(step / (unsigned)groups);
    step_g = (int)(step - (unsigned)step_img * groups);
    left = tiles - first;
  }
  __device__ __forceinline__ bool on() const { return left > 0; }
  __device__ __forceinline__ void next() {
    left -= step;
    img += step_img;
    g += step_g;
    if (g >= groups) g -= groups, ++img;
  }
};

// Staged loads (rows held): a warp copies what it will itself read of the next tile to its own
// regions in shared memory (cp.async, no warp waits for another) while it works on the current one.
// A region holds 32 positions of four rows of a map. By alignment:
//   kWholeTiles: a multiple of 16 channels and of 32 positions, all aligned: no bounds to check;
//   kAligned: rows of a multiple of four positions on aligned bases: a lane's four positions are all
//     in the row or behind it. In both each lane copies the four positions that it reads;
//   kAnywhere: rows start anywhere. f32: a lane copies and stores its own positions one by one. Halves
//     and codes: a row's 32 positions come as the aligned 8 bytes that hold them (9, 5; of memory
//     before or behind the tensor no more than an aligned 8 bytes' rest is touched, never a whole
//     one), neighbouring ones by neighbouring lanes, are shifted into place when read, and go through
//     shared memory to whole rows. (For f32 that takes more instructions than it saves sectors:
//     backward, 8 x 128 x 127 x 129 taped, 248 us so and 223 one by one, 200 with the L1 cache that one
//     slot leaves; bf16 190 us so and 220 one by one.)
enum { kWholeTiles, kAligned, kAnywhere };
// the first `bytes` (1 to 4) of an aligned word, zeros behind them
__device__ __forceinline__ void stage_copy_some(char* dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void stage_copy_two(char* dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src), "r"(on ? 8 : 0)
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
// The rows of the calling thread in a block's channels: their offsets from the block's first element
// of a picture, with the lane's four positions, and of their exponents (held rows: 32 bits do).
template <int kMode>
struct StagedRows {
  static constexpr bool kWhole = kMode == kWholeTiles;
  uint32_t e0, x0, e4, x4;
  int ch0, c, p;
  __device__ __forceinline__ StagedRows(int c_, int p_, int groups) : c(c_), p(p_) {
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
  // Of the 16 rows of the warp: a bit each that exists; the first one's offset.
  __device__ __forceinline__ uint32_t warp_rows() const {
    const int n = c - (int)(threadIdx.x >> 5) * 4 * kStagedRows;
    return n >= 16 ? 0xffffu : n > 0 ? (1u << n) - 1u : 0u;
  }
  __device__ __forceinline__ uint32_t warp_e() const {
    return (threadIdx.x >> 5) * (uint32_t)(4 * kStagedRows) * (uint32_t)p;
  }
  // the rows whose position `lane` of the tile exists; nv: positions from the lane's first on
  __device__ __forceinline__ uint32_t in_tile(int nv) const {
    const int lane = threadIdx.x & 31;
    return lane < nv + (lane & 7) * 4 ? warp_rows() : 0u;
  }
};
static_assert(4 * kStagedRows == 16, "the rows of a warp have a bit each");

// Regions of E (float, __half, __nv_bfloat16, or int8_t for codes). map: the block's first element of
// the tile; nv: how many positions of the row there are from the lane's first on; end: behind the
// tensor's last element.
template <int kMode, class E>
struct Region {
  static constexpr int kSize = (int)sizeof(E);
  static constexpr int kChunks = 4 * kSize + 1;  // of 8 bytes (kShifted)
  static constexpr bool kShifted = kMode == kAnywhere && kSize < 4;
  static constexpr int kRowBytes = kShifted ? 8 * kChunks : 32 * kSize;
  static constexpr int kBytes = 4 * kRowBytes;                     // per warp
  // the warp's rows, step j's to the j-th region
  static __device__ __forceinline__ void copy(char* to, const E* map, const StagedRows<kMode>& row,
                                              int nv, const E* end) {
    const int lane = threadIdx.x & 31;
    if constexpr (kMode != kAnywhere) {
#pragma unroll
      for (int j = 0; j < kStagedRows; ++j)
        stage_copy_all<4 * kSize>(to + j * kBytes + lane * 4 * kSize, map + row.e(j),
                                  kMode == kWholeTiles || (row.on(j) && nv > 0));
    } else if constexpr (kSize == 4) {
#pragma unroll
      for (int j = 0; j < kStagedRows; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          stage_copy_some(to + j * kBytes + lane * 16 + i * 4, map + row.e(j) + i,
                          row.on(j) && nv > i ? 4 : 0);
    } else {
      // the 8 bytes from the ones that hold the map's first element on; what would begin behind the
      // tensor is replaced by its last ones, of which nothing is used; zeros for rows that do not
      // exist
      const uint32_t sub = (uint32_t)reinterpret_cast<uintptr_t>(map) & 7u, on = row.warp_rows();
      const char* from = reinterpret_cast<const char*>(map) - sub;
      const uint32_t last =
          (uint32_t)min((long long)(reinterpret_cast<const char*>(end) - 1 - from), 0xffffffffLL);
      // (offsets run on by additions; as products, each costs a shift and a multiplication more)
      constexpr int kLanes = kChunks - 1, kRowsAtOnce = 32 / kLanes;
      const uint32_t step = (uint32_t)row.p * kSize;
      uint32_t o = row.warp_e() * kSize + sub;
      auto chunk = [&](uint32_t at, int r, int k) {
        stage_copy_two(to + r * kRowBytes + k * 8, from + (min(at, last) & ~7u), on >> r & 1);
      };
      if (lane < 4 * kStagedRows) chunk(o + lane * step + 8u * kLanes, lane, kLanes);
      o += lane / kLanes * step + 8u * (lane % kLanes);
#pragma unroll
      for (int i = 0; i < 4 * kStagedRows; i += kRowsAtOnce, o += kRowsAtOnce * step)
        chunk(o, i + lane / kLanes, lane % kLanes);
    }
  }
  // the word with the lane's first position, and the bits that are before it there (kShifted)
  static __device__ __forceinline__ const uint32_t* first_word(const char* from, const E* map,
                                                               const StagedRows<kMode>& row, int j,
                                                               uint32_t* bits) {
    const int lane = threadIdx.x & 31;
    const uint32_t sub =
        ((uint32_t)reinterpret_cast<uintptr_t>(map) + (row.e0 + row.e4 * j) * kSize) &
        7u;  // of the lane's first position: as of the row's, 4 kSize apart
    const uint32_t row_sub = kSize == 1 ? (sub - (lane & 1) * 4) & 7u : sub;
    *bits = (row_sub & 3u) * 8u;
    return reinterpret_cast<const uint32_t*>(from + (lane >> 3) * kRowBytes + (lane & 7) * 4 * kSize +
                                             (row_sub & 4u));
  }
  // two words (halves) or one (codes) of the lane's four positions, zeros behind the row
  static __device__ __forceinline__ uint2 words(const char* from, const E* map,
                                                const StagedRows<kMode>& row, int j, int nv) {
    if constexpr (!kShifted) {
      const char* q = from + (threadIdx.x & 31) * 4 * kSize;
      if constexpr (kSize == 2) return *reinterpret_cast<const uint2*>(q);
      else return make_uint2(*reinterpret_cast<const uint32_t*>(q), 0u);
    } else {
      uint32_t sh;
      const uint32_t* q = first_word(from, map, row, j, &sh);
      if constexpr (kSize == 2) {
        const uint32_t lo = nv >= 2 ? ~0u : nv == 1 ? 0xffffu : 0u;
        const uint32_t hi = nv >= 4 ? ~0u : nv == 3 ? 0xffffu : 0u;
        const uint32_t w1 = q[1];
        return make_uint2(__funnelshift_r(q[0], w1, sh) & lo, __funnelshift_r(w1, q[2], sh) & hi);
      } else {
        const uint32_t in = nv >= 4 ? ~0u : nv <= 0 ? 0u : ~0u >> (32 - 8 * nv);
        return make_uint2(__funnelshift_r(q[0], q[1], sh) & in, 0u);
      }
    }
  }
  static __device__ __forceinline__ F4 get(const char* from, const E* map,
                                           const StagedRows<kMode>& row, int j, int nv) {
    if constexpr (kSize == 4) {
      return make4(*reinterpret_cast<const float4*>(from + (threadIdx.x & 31) * 16));
    } else {
      return halves4<E>(words(from, map, row, j, nv));
    }
  }
};
// A predicated store: the compiler put a branch and its join around each.
template <class T>
__device__ __forceinline__ void store_if(T* to, T v, uint32_t on) {
  if constexpr (sizeof(T) == 4)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.f32 [%0], %1;\n\t}" ::
                     "l"(to), "f"(v), "r"(on) : "memory");
  else if constexpr (sizeof(T) == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u16 [%0], %1;\n\t}" ::
                     "l"(to), "h"(reinterpret_cast<const uint16_t&>(v)), "r"(on) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p st.global.u8 [%0], %1;\n\t}" ::
                     "l"(to), "r"((uint32_t)(uint8_t)v), "r"(on) : "memory");
}
// What put writes for the lane's four positions, by rows.
template <class T, class F>
__device__ __forceinline__ void scatter(T* map, F&& put, const StagedRows<kAnywhere>& row, int j, int nv,
                                        float* scratch) {
  static_assert(4 * 32 * sizeof(T) <= kScratchBytes, "four rows of halves or codes");
  const int lane = threadIdx.x & 31;
  const uint32_t in = row.in_tile(nv);
  T* s = reinterpret_cast<T*>(scratch);
  T* to = map + (row.warp_e() + lane + 4u * j * (uint32_t)row.p);
  __syncwarp();
  put(s + lane * 4);
  __syncwarp();
#pragma unroll
  for (int r = 0; r < 4; ++r, to += row.p) store_if(to, s[r * 32 + lane], in & 1u << (4 * j + r));
}
// four positions of the rows of step j to a map (scratch: kScratchBytes of the warp, for halves of
// kAnywhere)
template <int kMode, class T>
__device__ __forceinline__ void staged_store(T* map, F4 v, const StagedRows<kMode>& row, int j, int nv,
                                             float* scratch) {
  if constexpr (kMode == kWholeTiles) {
    store4_in(map + row.e(j), v);
  } else if constexpr (kMode == kAligned) {
    if (row.on(j) && nv > 0) store4_in(map + row.e(j), v);
  } else if constexpr (sizeof(T) == 4) {
    const float x[4] = {v.a.x, v.a.y, v.b.x, v.b.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) store_if(map + row.e(j) + i, x[i], row.on(j) && nv > i);
  } else {
    scatter(map, [&](T* s) { store4_in(s, v); }, row, j, nv, scratch);
  }
}
// and as part of a tape: the group's codes and exponents (whole warps call)
template <int kMode>
__device__ __forceinline__ void staged_hold(int8_t* codes, int8_t* exps, F4 v,
                                            const StagedRows<kMode>& row, int j, int nv,
                                            float* scratch) {
  const int lane = threadIdx.x & 31;
  uint32_t m = amax4(v);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  const uint32_t w = codes4(v, m);
  if constexpr (kMode != kAnywhere) {
    if (kMode == kWholeTiles || (row.on(j) && nv > 0))
      *reinterpret_cast<uint32_t*>(codes + row.e(j)) = w;
  } else {
    scatter(codes, [&](int8_t* s) { *reinterpret_cast<uint32_t*>(s) = w; }, row, j, nv, scratch);
  }
  if ((lane & 7) == 0 && row.on(j)) exps[row.x(j)] = (int8_t)tape_exp(m);
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

// How c channels at p positions are taken: staged (rows held) in a mode, or read again for each
// pass (mode -1); blocks of a cluster, and channels of a block (the last one's may be fewer); warps of
// a block.
struct Shape {
  int mode, cluster, share, warps;
};
Shape shape_of(int c, int p, bool vec) {
  // held rows are addressed by 32-bit byte offsets from their block's first
  const bool split = c <= kMaxCluster * kBlockC;
  const bool held = split && 4LL * std::min(c, kBlockC) * p < (1LL << 32) - 256;
  constexpr int kWarpC = 4 * kStagedRows;
  Shape sh;
  sh.mode = !held                                          ? -1
            : vec && c % kWarpC == 0 && p % kTapeGroup == 0 ? kWholeTiles
            : vec                                          ? kAligned
                                                           : kAnywhere;
  sh.cluster = split ? (c + kBlockC - 1) / kBlockC : 1;
  sh.share = ((c + sh.cluster - 1) / sh.cluster + kWarpC - 1) / kWarpC * kWarpC;
  if (sh.mode == kWholeTiles && sh.share * sh.cluster != c) sh.mode = kAligned;
  sh.warps = std::min(kMaxWarps, sh.share / kWarpC);
  return sh;
}
cudaLaunchConfig_t launch_of(const Shape& sh, int smem, int count, cudaStream_t stream,
                             cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(count * sh.cluster));
  cfg.blockDim = dim3((unsigned)(sh.warps * 32));
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = (unsigned)sh.cluster;
  attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = sh.cluster > 1 ? 1 : 0;
  return cfg;
}
// Blocks (or clusters) for the tiles: as many as are resident at once, each taking several tiles.
template <class A>
cudaError_t blocks_of(const Shape& sh, void (*k)(A), int smem, long long tiles, int sms, int* count) {
  *count = (int)std::min<long long>(tiles, std::max(1, sms / sh.cluster));
  cudaError_t e =
      cudaFuncSetAttribute((const void*)k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess || tiles <= *count) return e;
  int n = 0;
  if (sh.cluster == 1) {
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, k, sh.warps * 32, smem);
    n *= sms;
  } else {
    cudaLaunchAttribute attr;
    const cudaLaunchConfig_t cfg = launch_of(sh, smem, 1, nullptr, &attr);
    e = cudaOccupancyMaxActiveClusters(&n, k, &cfg);
  }
  if (n > 0) *count = (int)std::min<long long>(tiles, n);
  return e;
}
template <class A>
cudaError_t launch(const Shape& sh, void (*k)(A), int smem, int count, cudaStream_t stream,
                   const A& a) {
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = launch_of(sh, smem, count, stream, &attr);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, a);
  return e == cudaSuccess ? cudaGetLastError() : e;
}
// f(std::integral_constant) with a staged mode
template <class F>
auto by_mode(int mode, F&& f) {
  if (mode == kWholeTiles) return f(std::integral_constant<int, kWholeTiles>());
  if (mode == kAligned) return f(std::integral_constant<int, kAligned>());
  return f(std::integral_constant<int, kAnywhere>());
}
// ok: four neighbouring positions can be loaded and stored at once (rows of a multiple of four
// positions, maps aligned to four elements and codes to four bytes).
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
