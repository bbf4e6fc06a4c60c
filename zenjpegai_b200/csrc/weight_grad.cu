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
// accumulator of their own, and both are drained every 256 or 512 positions and added, rounding to
// nearest, to f32 sums in registers.
//
// One CTA per SM takes a 128 x N tile of dw over a share of the positions, every so many chunks of 64
// (the CTAs of a tile work on neighbouring chunks at a time: rows are far apart in memory, and with
// ranges of their own they kept opening DRAM pages for 128 bytes):
//  - the operands come to shared memory some chunks ahead: by TMA where all rows start on 16 bytes
//    (kVec; bf16 d_out, which needs no conversion, straight into the operand), else by cp.async:
//    rows of odd length start anywhere, which a TMA box cannot, so a warp copies the aligned 16
//    bytes that hold the rows it will itself convert, and shifts them into place as it reads them;
//  - 16 converter warps, in groups that take turns, turn a chunk into bf16 in the 128-byte-swizzled
//    K-major layout that the tensor core reads (16-byte piece j of row r at j ^ (r & 7)), and drain
//    the accumulators, half a window after they are complete;
//  - one thread issues the MMAs of a chunk, alternating between two accumulator sets in TMEM;
//  - db comes from the converters' registers, or, where d_out does not pass through them, from a
//    row of ones below the input's rows in the operand: one more column of the product.
// At 28 x 128 x 128^2, the kernel alone: f32 to 384 channels 210 us (3.6 TB/s; its copies alone take
// 154), f16 164 us, bf16 to 1024 241 us (4.1 TB/s; 198): what is left is a chunk's way through
// conversion while its places in shared memory are taken. The sums of the shares take 12 to 14 us
// more (f32 224 us a call, bf16 258). Call after call for seconds f32 settles at 245 us and bf16 at 290:
// the card is at its 1000 W limit then, and the SMs at 1.6 GHz of 1.965.
// Shares of one tile are summed in order by a second kernel (no atomics). Every wait is bounded
// (zjai_ctx_set_wait_limit); a role whose time is up has the others give up too, and the CTA ends once
// its copies and MMAs in flight have.
#include <algorithm>
#include <type_traits>

#include "ptx.cuh"
#include "train.h"

namespace zjai {
namespace {

constexpr int kM = 128, kN = 128;       // tile of dw
constexpr int kWorkers = 16, kMmaWarp = kWorkers, kTmaWarp = kWorkers + 1;
constexpr int kWorkThreads = 32 * kWorkers;
constexpr int kThreads = 32 * (kTmaWarp + 1);
constexpr int kChunk = 64;                 // positions of a pipeline stage
constexpr int kBlock = kM * kChunk * 2;    // a chunk of 128 rows in bf16
constexpr int kOnes = 16 * kChunk * 2;     // and of the 16 rows with the ones
constexpr int kBufCols = 256;              // TMEM columns of an accumulator set

// Per element type and alignment: bf16 terms of a d_out element; groups of converter warps, which
// take every kGroups-th chunk; stages of converted operands and chunks copied ahead of them; chunks
// between drains. A chunk has a fixed cost of waits and hand-offs per warp, which groups hide where
// there are chunks enough in shared memory (28 x 128 x 128^2, the kernel alone: f16 to 384 channels
// 163 us with two groups, 171 with one; bf16 to 1024 242 us with four, a tenth more with one); f32's
// few and large ones are done with sooner by all warps at once (to 384: a ninth sooner than by two
// groups).
template <bool kVec, class T>
struct Form;
template <>
struct Form<true, float> {
  static constexpr int kTerms = 3, kGroups = 1, kStages = 2, kAhead = 2, kPerWindow = 4;
  static constexpr int kRaw = 2 * kBlock + kBlock / 2;
};
template <>
struct Form<true, __half> {
  static constexpr int kTerms = 2, kGroups = 2, kStages = 2, kAhead = 4, kPerWindow = 4;
  static constexpr int kRaw = kBlock + kBlock / 2;
};
template <>
struct Form<true, __nv_bfloat16> {  // kRaw: the codes alone
  static constexpr int kTerms = 1, kGroups = 4, kStages = 5, kAhead = 4, kPerWindow = 8;
  static constexpr int kRaw = kBlock / 2;
};
template <class T>
struct Form<false, T> {
  static constexpr int kTerms = sizeof(T) == 4 ? 3 : std::is_same<T, __half>::value ? 2 : 1;
  static constexpr int kGroups = 1, kStages = kTerms == 1 ? 3 : 2, kAhead = kTerms == 3 ? 2 : 4;
  static constexpr int kPerWindow = 4;
  static constexpr int kPitchD = kChunk * (int)sizeof(T) + 16, kPitchX = kChunk + 16;  // of a row
  static constexpr int kRaw = kM * kPitchD + kN * kPitchX;
};
template <bool kVec, class T>
constexpr bool direct() {  // d_out is copied into the operand, the ones row gives db
  return kVec && std::is_same<T, __nv_bfloat16>::value;
}
template <bool kVec, class T>
constexpr int stage_bytes() {
  return (Form<kVec, T>::kTerms + 1) * kBlock + (direct<kVec, T>() ? kOnes : 0);
}
template <bool kVec, class T>
constexpr int smem_bytes() {
  return 1024 + Form<kVec, T>::kStages * stage_bytes<kVec, T>() +
         Form<kVec, T>::kAhead * Form<kVec, T>::kRaw;
}

struct WgArgs {
  const void* dout;
  const int8_t *codes, *exps;
  int oc, c, p, groups;
  int nb;          // N of the MMA: rows of the input tile, a multiple of 16
  int m_tiles;
  long long d_elems, x_elems;  // of d_out and the codes
  int chunks_img;  // chunks per picture
  long long chunks;
  int splits;
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
__device__ __forceinline__ float rest_bf_any(float v) {
  return fabsf(v) == __uint_as_float(0x7f800000u) ? 0.f : v - trunc_bf(v);
}

__device__ __forceinline__ void st_shared16(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

__device__ __forceinline__ void ld_shared16(uint32_t at, uint32_t* w) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t ld_shared4(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
// 16 bytes from src, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int kNewer>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kNewer) : "memory");
}

// Rows that start anywhere: a chunk's kBytes of kRows rows, `first` and those behind it, of a map
// whose chunk starts at `at` in row 0, rows `row_bytes` apart, to rows of kBytes + 16 in shared
// memory, by the aligned 16 bytes that hold them: of memory outside the map none but the rest of an
// aligned 16 bytes with a byte of it is touched (what would begin behind the map is replaced by its
// last). Rows from `rows` on do not exist: zeros. (Copies of the map's last bytes in their place, from
// every block, took the kernel from 37 to 67 us at 64 x 64 channels in bf16.)
template <int kRows, int kBytes>
__device__ __forceinline__ void copy_rows(uint32_t to, const char* at, long long row_bytes, int first,
                                          int rows, const char* last) {
  constexpr int kLanes = kBytes / 16, kAtOnce = 32 / kLanes;
  const int lane = threadIdx.x & 31;
  auto piece = [&](int r, int j) {
    const uintptr_t q = (reinterpret_cast<uintptr_t>(at + r * row_bytes) & ~(uintptr_t)15) + 16 * j;
    copy16(to + r * (kBytes + 16) + 16 * j,
           reinterpret_cast<const void*>(min(q, reinterpret_cast<uintptr_t>(last))), r < rows);
  };
#pragma unroll
  for (int r = 0; r < kRows; r += kAtOnce) piece(first + r + lane / kLanes, lane % kLanes);
  if (lane < kRows) piece(first + lane, kLanes);
}
// Words of 4 kWords bytes from the byte `from` of shared memory on.
template <int kWords>
__device__ __forceinline__ void ld_shifted(uint32_t from, uint32_t* w) {
  const uint32_t at = from & ~3u, sh = (from & 3u) * 8u;
  uint32_t v[kWords + 1];
#pragma unroll
  for (int i = 0; i <= kWords; ++i) v[i] = ld_shared4(at + 4 * i);
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], sh);
}
// bytes from `valid` on zero
template <int kWords>
__device__ __forceinline__ void clip_words(uint32_t* w, int valid) {
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const int left = valid - 4 * i;
    if (left < 4) w[i] = left <= 0 ? 0u : w[i] & (0xffffffffu >> (32 - 8 * left));
  }
}

// Before a slot is given to the next copy: the registers of each vector that was read from it have
// their values, in all lanes. (Arriving at the slot's barrier does not say so: the next chunk's copy
// was seen to land before reads issued ahead of the arrival.) `seen` combines a register of each.
// One answer for the whole warp: whether `ok` holds in all lanes.
__device__ __forceinline__ bool wait_read(uint32_t seen, bool ok) {
  if (!__all_sync(0xffffffffu, ok && seen != 0x9e3779b9u)) {
    if (!__all_sync(0xffffffffu, ok)) return false;
    __nanosleep(1);  // any use of `seen` will do
  }
  return true;
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

// A chunk's picture and place in it, of a sequence with a fixed step.
struct Chunk {
  int img, in, step_img, step_in, of;
  __device__ __forceinline__ Chunk(int first, int step, int chunks_img) : of(chunks_img) {
    img = first / of;
    in = first - img * of;
    step_img = step / of;
    step_in = step - step_img * of;
  }
  __device__ __forceinline__ void next() {
    img += step_img;
    in += step_in;
    if (in >= of) in -= of, ++img;
  }
};

template <bool kVec, class T>
__global__ void __launch_bounds__(kThreads, 1)
    weight_grad_kernel(const __grid_constant__ CUtensorMap map_d,
                       const __grid_constant__ CUtensorMap map_x, const WgArgs a) {
  using F = Form<kVec, T>;
  constexpr int kTerms = F::kTerms, kStages = F::kStages, kAhead = F::kAhead, kRaw = F::kRaw;
  constexpr int kGroups = F::kGroups, kPerWindow = F::kPerWindow;
  // a slot is always read by the same group: another one's parity test would take the phase before
  // the last for the one it waits for
  static_assert(kAhead % kGroups == 0, "slots change groups");
  // and with fewer stages than groups, of a stage
  static_assert(kStages >= kGroups, "a group may be two phases behind");
  constexpr int kGroupWarps = kWorkers / kGroups, kGroupThreads = kWorkThreads / kGroups;
  constexpr int kStageBytes = stage_bytes<kVec, T>();
  constexpr bool kDirect = direct<kVec, T>();
  constexpr int kSets = kTerms > 1 ? 2 : 1;  // accumulators of a set: first terms, the others
  extern __shared__ char smem_raw[];
  // full / empty: operand stages; d_full: a stage's directly copied d_out; raw_*: copied chunks
  __shared__ __align__(8) uint64_t bars[3 * kStages + 2 * kAhead + 4 + 1];
  __shared__ uint32_t tmem_at;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x, split = blockIdx.y;
  const int o0 = (tile % a.m_tiles) * kM, i0 = (tile / a.m_tiles) * kN;
  // chunks split, split + splits, ..
  const int count = (int)((a.chunks - split + a.splits - 1) / a.splits);
  const int windows = (count + kPerWindow - 1) / kPerWindow;
  const bool want_db = a.db && i0 == 0;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t raw_base = smem + kStages * kStageBytes;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, d_full = empty + 8 * kStages,
                 raw_full = d_full + 8 * kStages, raw_empty = raw_full + 8 * kAhead,
                 acc_full = raw_empty + 8 * kAhead, acc_empty = acc_full + 16,
                 drain = acc_empty + 16;
  volatile int* abort = &abort_flag;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, kGroupWarps);
      mbar_init(empty + 8 * i, 1);
      mbar_init(d_full + 8 * i, 1);
    }
    for (int i = 0; i < kAhead; ++i) {
      mbar_init(raw_full + 8 * i, 1);
      mbar_init(raw_empty + 8 * i, kGroupWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, kWorkers);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (kDirect && want_db) {
    // the ones: row nb of each stage's input rows, the 15 rows behind it zero
    for (int i = threadIdx.x; i < kStages * kOnes / 16; i += kThreads) {
      const int st = i / (kOnes / 16), e = i % (kOnes / 16);
      const uint32_t v = e < 8 ? 0x3f803f80u : 0u;
      st_shared16(smem + st * kStageBytes + kTerms * kBlock + a.nb * 128 + e * 16,
                  make_uint4(v, v, v, v));
    }
    fence_proxy_async_smem();
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
      const int n = kDirect && want_db ? a.nb + 16 : a.nb;
      const uint32_t idesc = idesc_f16((uint32_t)n) | (1u << 7) | (1u << 10);  // bf16 operands
      bool ok = true;
      for (int k = 0; k < count && ok; ++k) {
        const int st = k % kStages, win = k / kPerWindow, buf = win & 1;
        const bool first = k % kPerWindow == 0;
        if (first && win >= 2) {
          ok = mbar_wait(acc_empty + 8 * buf, ((win >> 1) - 1) & 1, abort, a.err,
                         DEV_TIMEOUT_ACC_EMPTY, a.limit);
          if (!ok) break;
        }
        if (kDirect) {
          ok = mbar_wait(d_full + 8 * st, (k / kStages) & 1, abort, a.err, DEV_TIMEOUT_FULL, a.limit);
          if (!ok) break;
        }
        ok = mbar_wait(full + 8 * st, (k / kStages) & 1, abort, a.err, DEV_TIMEOUT_FULL, a.limit);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * kBufCols, at = smem + st * kStageBytes;
        const uint64_t db = smem_desc(at + kTerms * kBlock, 128u);
#pragma unroll
        for (int t = 0; t < kTerms; ++t) {
          const uint64_t da = smem_desc(at + t * kBlock, 128u);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 positions: 32 bytes along the row
            umma_f16(d + (t ? kN : 0), da + 2 * kk, db + 2 * kk, idesc,
                     first && t < 2 && kk == 0 ? 0u : 1u);
        }
        umma_commit(empty + 8 * st);
        if (k % kPerWindow == kPerWindow - 1 || k == count - 1) umma_commit(acc_full + 8 * buf);
      }
      // all MMAs done before TMEM goes, also after a wait that gave up
      umma_commit(drain);
      mbar_wait_drain(drain, 0, a.err);
    }
    __syncwarp();
  } else if (warp == kTmaWarp) {
    if (kVec && lane == 0) {
      tma_prefetch_desc(&map_d);
      tma_prefetch_desc(&map_x);
      Chunk q(split, a.splits, a.chunks_img);
      int k = 0;
      for (; k < count; ++k) {
        const int sl = k % kAhead, st = k % kStages;
        if (k >= kAhead &&
            !mbar_wait(raw_empty + 8 * sl, (k / kAhead - 1) & 1, abort, a.err, DEV_TIMEOUT_EMPTY,
                       a.limit))
          break;
        if (kDirect && k >= kStages &&
            !mbar_wait(empty + 8 * st, (k / kStages - 1) & 1, abort, a.err, DEV_TIMEOUT_EMPTY,
                       a.limit))
          break;
        const uint32_t raw = raw_base + sl * kRaw, bar = raw_full + 8 * sl;
        const int img = q.img, at = q.in * kChunk;
        mbar_arrive_expect_tx(bar, kRaw);
        if constexpr (kDirect) {
          mbar_arrive_expect_tx(d_full + 8 * st, kBlock);
          tma_load_3d(smem + st * kStageBytes, &map_d, d_full + 8 * st, at, o0, img);
        } else {
          tma_load_3d(raw, &map_d, bar, at, o0, img);
          if constexpr (sizeof(T) == 4) tma_load_3d(raw + kBlock, &map_d, bar, at + 32, o0, img);
        }
        tma_load_3d(raw + kRaw - kBlock / 2, &map_x, bar, at, i0, img);
        q.next();
      }
      // all copies landed before the CTA goes, also after a wait that gave up
      for (int j = max(0, k - kAhead); j < k; ++j)
        mbar_wait_drain(raw_full + 8 * (j % kAhead), (j / kAhead) & 1, a.err);
      if (kDirect)
        for (int j = max(0, k - kStages); j < k; ++j)
          mbar_wait_drain(d_full + 8 * (j % kStages), (j / kStages) & 1, a.err);
    }
    __syncwarp();
  } else {
    // this thread's group of converters takes the chunks `group`, group + kGroups, ..; pieces of a
    // chunk: d_out rows dr + u kRowsD, positions 8 dj .. (f32 from TMA: of each half of the chunk,
    // rows spread over a warp's lanes such that eight lanes' 16 bytes lie in different banks both as
    // read, two pieces of four of a half row, and as stored); input rows xr + u kRowsX, positions
    // 16 xj ..
    const int group = warp / kGroupWarps, tid = threadIdx.x % kGroupThreads;
    constexpr bool kHalves = kVec && sizeof(T) == 4;
    constexpr int kRowsD = kHalves ? kGroupThreads / 4 : kGroupThreads / 8, kUnitsD = kM / kRowsD;
    constexpr int kRowsX = kGroupThreads / 4, kUnitsX = kN / kRowsX;
    const int l8 = lane >> 2;
    const int dr = kHalves ? (tid >> 5) * 8 + ((l8 >> 1) ^ (l8 & 1 ? 5 : 0)) : tid >> 3;
    const int dj = kHalves ? lane & 3 : tid & 7;
    const int xr = tid >> 2, xj = tid & 3;
    const int x_rows = min(a.nb, a.c - i0);
    auto swizzled = [](uint32_t base, int r, int j) { return base + r * 128 + ((j ^ (r & 7)) << 4); };

    // cp.async: the group's chunk being copied, and the one being converted
    const char* d_lo = static_cast<const char*>(a.dout);
    const char* x_lo = reinterpret_cast<const char*>(a.codes);
    const long long d_row = (long long)a.p * (int)sizeof(T);
    auto last_of = [](const char* hi) {  // the aligned 16 bytes with the byte before hi
      return reinterpret_cast<const char*>((reinterpret_cast<uintptr_t>(hi) - 1) & ~(uintptr_t)15);
    };
    const char *d_last = last_of(d_lo + a.d_elems * (int)sizeof(T)), *x_last = last_of(x_lo + a.x_elems);
    Chunk next(split + group * a.splits, kGroups * a.splits, a.chunks_img), cur = next;
    auto at_d = [&](const Chunk& q) {
      return d_lo + (((long long)q.img * a.oc + o0) * a.p + q.in * kChunk) * (int)sizeof(T);
    };
    auto at_x = [&](const Chunk& q) {
      return x_lo + ((long long)q.img * a.c + i0) * a.p + q.in * kChunk;
    };
    int copied = group;
    auto copy_chunk = [&]() {
      if constexpr (!kVec) {
        if (copied < count) {
          const uint32_t raw = raw_base + copied % kAhead * kRaw;
#pragma unroll
          for (int u = 0; u < kUnitsD; ++u)
            copy_rows<4, kChunk * (int)sizeof(T)>(raw, at_d(next), d_row,
                                                  u * kRowsD + (tid >> 5) * 4, a.oc - o0, d_last);
#pragma unroll
          for (int u = 0; u < kUnitsX; ++u)
            copy_rows<8, kChunk>(raw + kM * F::kPitchD, at_x(next), a.p,
                                 u * kRowsX + (tid >> 5) * 8, x_rows, x_last);
          copied += kGroups;
          next.next();
        }
        copy_commit();
      }
    };
    // the exponents of the group's next chunk, loaded while it converts the current one
    Chunk ahead(split + group * a.splits, kGroups * a.splits, a.chunks_img);
    int eb[kUnitsX];
    auto load_exps = [&](bool on) {
      const int8_t* pe = a.exps + ((long long)ahead.img * a.c + i0 + xr) * a.groups;
      const int g = 2 * ahead.in + (xj >> 1);
#pragma unroll
      for (int u = 0; u < kUnitsX; ++u)
        eb[u] = on && g < a.groups && u * kRowsX + xr < x_rows
                    ? __ldg(pe + (long long)(u * kRowsX) * a.groups + g)
                    : 0;
      ahead.next();
    };

    // A warp's wait, with one answer for all its lanes: a warp whose time is up leaves as a whole, and
    // no lane of it is left alone in a vote, a warp barrier or a TMEM load. (The wait for a copied
    // chunk gets its answer from wait_read's vote.)
    auto wait = [&](uint32_t bar, int phase, int code) {
      return __all_sync(0xffffffffu,
                        mbar_wait_sleep(bar, phase & 1, abort, a.err, code, a.limit)) != 0;
    };

    // accumulator rows 32 (warp % 4) + lane, columns 32 (warp / 4) ..
    float acc[32], acc_db = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] = 0.f;
    const int c0 = (warp >> 2) * 32;
    int drained = 0;
    auto drain_window = [&]() {
      const int buf = drained & 1;
      if (!wait(acc_full + 8 * buf, drained >> 1, DEV_TIMEOUT_ACC_FULL)) return false;
      tc_fence_after();
      const uint32_t base = tmem + ((uint32_t)(warp & 3) * 32u << 16) + buf * kBufCols;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (c0 + j * 16 < a.nb) {
#pragma unroll
          for (int set = kSets - 1; set >= 0; --set) {
            float v[16];
            tmem_ld16(base + set * kN + c0 + j * 16, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j * 16 + i] += v[i];
          }
        }
      }
      if (kDirect && want_db && c0 == 0) {
        float v[16];
        tmem_ld16(base + a.nb, v);
        acc_db += v[0];
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + 8 * buf);
      ++drained;
      return true;
    };
    float2 bsum[kUnitsD] = {};
    float btot[kUnitsD] = {};

#pragma unroll
    for (int j = 0; j < kAhead / kGroups; ++j) copy_chunk();
    load_exps(group < count);
    bool ok = true;
    for (int k = group, turn = 0; k < count && ok; k += kGroups, ++turn) {
      const int st = k % kStages, sl = k % kAhead;
      const uint32_t stage = smem + st * kStageBytes;
      const uint32_t raw = raw_base + sl * kRaw;
      int e[kUnitsX];
#pragma unroll
      for (int u = 0; u < kUnitsX; ++u) e[u] = eb[u];
      load_exps(k + kGroups < count);
      // read all of it, so that the slot is free for the next copy while this one is converted
      constexpr int kParts = kDirect ? 0 : kUnitsD * (kHalves ? 2 : 1);  // f32: part i of half i & 1
      uint32_t wx[kUnitsX][4], wd[kParts ? kParts : 1][2 * sizeof(T)];
      auto read_all = [&](bool copied_in) {
        uint32_t seen = 0;
#pragma unroll
        for (int u = 0; u < kUnitsX; ++u) seen += wx[u][0] ^ wx[u][3];
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
          for (int q = 0; q < 2 * (int)sizeof(T); q += kVec ? 4 : 1) seen += wd[i][q];
        if constexpr (!kVec)
#pragma unroll
          for (int u = 0; u < kUnitsX; ++u) seen += wx[u][1] ^ wx[u][2];
        return wait_read(seen, copied_in);
      };
      if constexpr (kVec) {
        const bool here = mbar_wait_sleep(raw_full + 8 * sl, (k / kAhead) & 1, abort, a.err,
                                          DEV_TIMEOUT_FULL, a.limit);
#pragma unroll
        for (int u = 0; u < kUnitsX; ++u)
          ld_shared16(raw + kRaw - kBlock / 2 + (u * kRowsX + xr) * 64 + xj * 16, wx[u]);
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          if constexpr (kHalves) {
            const uint32_t at = raw + (i & 1) * kBlock;
            ld_shared16(swizzled(at, (i >> 1) * kRowsD + dr, 2 * dj), wd[i]);
            ld_shared16(swizzled(at, (i >> 1) * kRowsD + dr, 2 * dj + 1), wd[i] + 4);
          } else {
            ld_shared16(swizzled(raw, i * kRowsD + dr, dj), wd[i]);
          }
        }
        ok = read_all(here);
        if (!ok) break;
        __syncwarp();
        if (lane == 0) mbar_arrive(raw_empty + 8 * sl);
      } else {
        copy_wait<kAhead / kGroups - 1>();
        __syncwarp();
        const uint32_t d_sub = (uint32_t)reinterpret_cast<uintptr_t>(at_d(cur));
        const uint32_t x_sub = (uint32_t)reinterpret_cast<uintptr_t>(at_x(cur));
#pragma unroll
        for (int u = 0; u < kUnitsX; ++u) {
          const int r = u * kRowsX + xr;
          ld_shifted<4>(raw + kM * F::kPitchD + r * F::kPitchX + ((x_sub + r * (uint32_t)a.p) & 15u) +
                            xj * 16,
                        wx[u]);
        }
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          const int r = i * kRowsD + dr;
          const uint32_t from = raw + r * F::kPitchD + ((d_sub + r * (uint32_t)d_row) & 15u) +
                                dj * 8 * (int)sizeof(T);
          if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int q = 0; q < 8; ++q) wd[i][q] = ld_shared4(from + 4 * q);
          } else {
            ld_shifted<4>(from, wd[i]);
          }
        }
        read_all(true);
        __syncwarp();
        copy_chunk();
        if (cur.in * kChunk + kChunk > a.p) {  // a row's last chunk
          const int left = a.p - cur.in * kChunk;
#pragma unroll
          for (int u = 0; u < kUnitsX; ++u) clip_words<4>(wx[u], left - xj * 16);
#pragma unroll
          for (int i = 0; i < kParts; ++i)
            clip_words<2 * (int)sizeof(T)>(wd[i], (left - dj * 8) * (int)sizeof(T));
        }
        cur.next();
      }
      if (k >= kStages) {
        ok = wait(empty + 8 * st, k / kStages - 1, DEV_TIMEOUT_EMPTY);
        if (!ok) break;
      }
#pragma unroll
      for (int u = 0; u < kUnitsX; ++u) {
        const uint32_t sb = e[u] == kTapeNan ? 0x7fc0u : (uint32_t)(max(e[u], -126) + 127) << 7;
        const uint32_t s2 = sb | sb << 16;
        const __nv_bfloat162 sc = reinterpret_cast<const __nv_bfloat162&>(s2);
        const uint2 v0 = taped_bf16(wx[u][0], sc), v1 = taped_bf16(wx[u][1], sc);
        const uint2 v2 = taped_bf16(wx[u][2], sc), v3 = taped_bf16(wx[u][3], sc);
        const int r = u * kRowsX + xr;
        if (r < a.nb) {
          const uint32_t to = stage + kTerms * kBlock;
          st_shared16(swizzled(to, r, 2 * xj), make_uint4(v0.x, v0.y, v1.x, v1.y));
          st_shared16(swizzled(to, r, 2 * xj + 1), make_uint4(v2.x, v2.y, v3.x, v3.y));
        }
      }
      if constexpr (!kDirect) {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          const int u = kHalves ? i >> 1 : i, r = u * kRowsD + dr;
          const uint32_t at = kHalves ? swizzled(stage, r, 4 * (i & 1) + dj) : swizzled(stage, r, dj);
          const uint32_t* w = wd[i];
          float2 f[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (sizeof(T) == 4)
              f[q] = make_float2(__uint_as_float(w[2 * q]), __uint_as_float(w[2 * q + 1]));
            else if constexpr (kTerms == 2)
              f[q] = __half22float2(reinterpret_cast<const __half2&>(w[q]));
            else
              f[q] = make_float2(__uint_as_float(w[q] << 16), __uint_as_float(w[q] & 0xffff0000u));
          }
          const float2 s = __fadd2_rn(__fadd2_rn(f[0], f[1]), __fadd2_rn(f[2], f[3]));
          bsum[u] = __fadd2_rn(bsum[u], s);
          if constexpr (kTerms == 1) {
            st_shared16(at, make_uint4(w[0], w[1], w[2], w[3]));
          } else {
            // an infinity or NaN anywhere makes the sum one: then each rest is looked at
            const bool finite =
                __all_sync(0xffffffffu, fabsf(s.x + s.y) < __uint_as_float(0x7f800000u));
#pragma unroll
            for (int t = 0; t < kTerms; ++t) {
              st_shared16(at + t * kBlock, make_uint4(bf2(f[0].x, f[0].y), bf2(f[1].x, f[1].y),
                                                      bf2(f[2].x, f[2].y), bf2(f[3].x, f[3].y)));
              if (t + 1 == kTerms) continue;
              if (finite) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  f[q] = __fadd2_rn(f[q], make_float2(-trunc_bf(f[q].x), -trunc_bf(f[q].y)));
              } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  f[q] = make_float2(rest_bf_any(f[q].x), rest_bf_any(f[q].y));
              }
            }
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + 8 * st);
      if (!kDirect && (turn & 31) == 31) {  // two levels: chains of 32 chunks, and of the chains
#pragma unroll
        for (int i = 0; i < kUnitsD; ++i) {
          btot[i] += bsum[i].x + bsum[i].y;
          bsum[i] = make_float2(0.f, 0.f);
        }
      }
      if (k % kPerWindow >= kPerWindow / 2 && drained < k / kPerWindow) ok = drain_window();
    }
    if (!kVec) copy_wait<0>();
    while (ok && drained < windows) ok = drain_window();
    // the operands' stages are free now
    float* stage_f = reinterpret_cast<float*>(smem_raw + (smem - smem_u32(smem_raw)));
    const int o = o0 + (warp & 3) * 32 + lane;
    if (want_db) {
      float* db = a.db + (long long)split * a.oc;
      if constexpr (kDirect) {
        if (c0 == 0 && o < a.oc) db[o] = acc_db;
      } else {
        // each group's sums of the rows, then their sum
        float* rows = stage_f + kWorkers * 32 * 33;
#pragma unroll
        for (int i = 0; i < kUnitsD; ++i) {
          float s = btot[i] + (bsum[i].x + bsum[i].y);
#pragma unroll
          for (int x = kHalves ? 2 : 4; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
          if (dj == 0) rows[group * kM + i * kRowsD + dr] = s;
        }
        named_bar_sync(1, kWorkThreads);
        if (threadIdx.x < kM && o0 + (int)threadIdx.x < a.oc) {
          float s = 0.f;
#pragma unroll
          for (int g = 0; g < kGroups; ++g) s += rows[g * kM + threadIdx.x];
          db[o0 + threadIdx.x] = s;
        }
      }
    }
    // a warp's 32 x 32 sums through shared memory, to whole 128-byte lines
    float* mine = stage_f + warp * 32 * 33;
#pragma unroll
    for (int j = 0; j < 32; ++j) mine[lane * 33 + j] = acc[j];
    __syncwarp();
    const int o1 = o0 + (warp & 3) * 32, col = i0 + c0 + lane;
    float* out = a.dw + ((long long)split * a.oc + o1) * a.c + col;
    if (col < a.c)
      for (int r = 0; r < min(32, a.oc - o1); ++r) out[(long long)r * a.c] = mine[r * 33 + lane];
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
// chunks' time for what a CTA does once (start, write its partial tile) and for the second launch.
int choose_splits(long long tiles, long long chunks, int sms) {
  long long best = 1;
  double cost = 1e300;
  const long long most = std::min<long long>({chunks, std::max<long long>(1, 4LL * sms / tiles), 1024});
  for (long long s = 1; s <= most; ++s) {
    const double rounds = (double)((tiles * s + sms - 1) / sms);
    const double t = rounds * ((double)((chunks + s - 1) / s) + 8.0) + (s > 1 ? 6.0 : 0.0);
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
    // rows on 16-byte boundaries, and 16 positions of the codes all in a row or past it
    const bool vec = aligned(dd, (size_t)p * es) && aligned(dc, (size_t)p);
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
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
      a.d_elems = (long long)n * oc * p;
      a.x_elems = (long long)n * c * p;
      a.chunks_img = (p + kChunk - 1) / kChunk;
      a.chunks = (long long)n * a.chunks_img;
      a.splits = choose_splits(tiles, a.chunks, ctx->sms);
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
      CUtensorMap md = {}, mx = {};
      if (vec) {
        // d_out in boxes of 128 rows of 128 bytes, swizzled; the codes in boxes of 128 rows of 64
        ZJAI_TRY(make_planar_map(ctx, &md, dd, (int)es, p, oc, n, 128 / (int)es, kM, true));
        ZJAI_TRY(make_planar_map(ctx, &mx, dc, 1, p, c, n, kChunk, kN, false));
      }
      auto k = vec ? weight_grad_kernel<true, T> : weight_grad_kernel<false, T>;
      const int smem = vec ? smem_bytes<true, T>() : smem_bytes<false, T>();
      ZJAI_TRY(cuda_check(cudaFuncSetAttribute((const void*)k,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                          me));
      k<<<dim3((unsigned)tiles, a.splits), kThreads, smem, ctx->stream>>>(md, mx, a);
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
