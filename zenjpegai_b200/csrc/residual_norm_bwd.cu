// Backward pass of the residual step with its norms, gate and scale
// (zjai_gated_residual_norm_backward): the mathematics and the layout are in residual_norm.cuh.
#include "residual_norm.cuh"

namespace zjai {
namespace {

template <class T>
struct BwdArgs {
  const T *dy, *dz, *f, *gate, *y;
  zjai_residual_tapes tp;  // taped f, gate, y
  int gate_c, c, p, cluster, share;
  long long tiles;
  zjai_residual_params prm;
  T *dx, *df, *dgate;
  float* sums;  // [blocks][5][c]: scale, post_weight, post_bias, pre_weight, pre_bias
};

// A row's four positions of a kept map, codes and exponent of a tape or values, as loaded.
template <bool kTaped, bool kVec, class T>
struct Kept {
  F4 v;
  __device__ __forceinline__ void load(const T* map, const zjai_tape&, long long e0, long long,
                                       int at, int p) {
    v = load4<kVec>(map + e0, at, p);
  }
  __device__ __forceinline__ F4 get() const { return v; }
};
template <bool kVec, class T>
struct Kept<true, kVec, T> {
  uint32_t w;
  int e;
  __device__ __forceinline__ void load(const T*, const zjai_tape& t, long long e0, long long ge,
                                       int at, int p) {
    w = load_codes<kVec>(t.codes + e0, at, p);
    e = __ldg(t.exps + ge);
  }
  __device__ __forceinline__ F4 get() const { return taped4(w, e); }
};

// Rows held, the next tile copied ahead. Per thread a slot has dy, dz, and f, y and the gate as they
// were kept. Two slots where 16 warps' fit the SM's shared memory; with one the next tile is copied
// as soon as the current one has been read.
// The parameter gradients are summed over a block's tiles in registers, written out per block.
template <int kMode, bool kTaped, class T>
struct BwdSlot {
  using Grad = Region<kMode, T>;
  using Kept = Region<kMode, typename std::conditional<kTaped, int8_t, T>::type>;
  // bytes per warp: of a slot's maps and exponents (words), and of b
  static constexpr int kMaps = kStagedRows * (2 * Grad::kBytes + 3 * Kept::kBytes);
  static constexpr int kExps = kTaped ? 3 * 4 * kStagedRows * 4 : 0;
  static constexpr int kB = sizeof(T) == 4 ? 0 : kStagedRows * 32 * (int)sizeof(float4);
  // two slots where 227 KB hold them; one for rows that start anywhere, whose copies want the rest as
  // L1 cache (8 x 128 x 127 x 129 taped, two and one: f32 227 and 200 us, bf16 189 and 181 us)
  static constexpr int kRest = tail_bytes<4>(kBlockC, kMaxWarps) + 9 * 32 * (int)sizeof(float);
  static constexpr int kSlots =
      kMode != kAnywhere && (2 * (kMaps + kExps) + kB) * kMaxWarps + kRest <= 227 * 1024 ? 2 : 1;
  static constexpr int kBytes = kSlots * (kMaps + kExps) + kB;
};
template <int kMode, bool kTaped, class T>
__global__ void __launch_bounds__(kThreadsMost, 1)
    residual_norm_bwd_staged_kernel(const BwdArgs<T> a) {
  using S = BwdSlot<kMode, kTaped, T>;
  constexpr bool kWhole = kMode == kWholeTiles, kVec = kMode != kAnywhere;
  constexpr int kRows = kStagedRows;
  __shared__ __align__(16) float totals[9 * 32];  // f 0, 1, y 2, 3, a 4, 5, b 6, 7, gate 8
  extern __shared__ __align__(16) char slots[];
  const int warps = blockDim.x >> 5, wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cluster cl(a.cluster);
  const int ch0 = cl.rank * a.share, c = min(a.share, a.c - ch0);  // of the block
  const Rows<kRows, kWhole> rows(c, a.share, a.c, warps);
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, per_row = a.gate_c > 1;
  const bool need_f = post || a.gate_c || a.prm.scale;
  // two sums at a time are joined by four warps each where there are eight
  const bool two = warps >= 8;
  auto join_first = [&](auto f) {
    if (!two || wp < 4) f(wp, two ? 4 : warps);
  };
  auto join_second = [&](auto f) {
    if (!two || (wp >= 4 && wp < 8)) f(two ? wp - 4 : wp, two ? 4 : warps);
  };
  const StagedRows<kMode> row(c, a.p, groups);
  // the warp's shared memory: slots of maps, slots of exponents, b
  char* mine = slots + wp * S::kBytes;
  Params<kRows> prm = {nullptr, a.share};
  Exchange<4> ex = {nullptr, totals};
  take_tail(slots + warps * S::kBytes, a.share, &prm.v, &ex);
  auto grad_at = [&](int slot, int k, int j) {
    return mine + slot * S::kMaps + (k * kRows + j) * S::Grad::kBytes;
  };
  auto kept_at = [&](int slot, int k, int j) {
    return mine + slot * S::kMaps + 2 * kRows * S::Grad::kBytes + (k * kRows + j) * S::Kept::kBytes;
  };
  // a row's exponent comes as the aligned word that holds it, copied by one lane per row of the warp
  constexpr int kWarpRows = 4 * kRows;
  auto exp_at = [&](int slot, int k, int r) {
    return mine + S::kSlots * S::kMaps + ((slot * 3 + k) * kWarpRows + r) * 4;
  };
  // how far behind an aligned word a tape's exponents begin (kVec: they begin with one)
  auto exp_sub = [](const zjai_tape& tp) {
    return kVec ? 0u : (uint32_t)reinterpret_cast<uintptr_t>(tp.exps) & 3u;
  };
  // b of a row, until df: where dy was, or (f16, bf16) in a place of its own
  auto b_at = [&](int slot, int j) {
    return reinterpret_cast<float4*>(sizeof(T) == 4 ? grad_at(slot, 0, j)
                                                    : mine + S::kSlots * (S::kMaps + S::kExps) +
                                                          j * 32 * (int)sizeof(float4)) +
           lane;
  };
  // exponents of the whole map (the gate's too: this path takes its own rows only where it has c)
  const long long x_all = a.tiles * a.c, elems = a.tiles / groups * a.c * a.p;
  auto copy = [&](const Tiles& t, int slot) {
    const long long e = ((long long)t.img * a.c + ch0) * a.p + t.g * kTapeGroup;
    const long long x = ((long long)t.img * a.c + ch0) * groups + t.g;
    const int nv = kWhole ? 4 : a.p - (t.g * kTapeGroup + (lane & 7) * 4);
    auto keep_exps = [&](const zjai_tape& tp, int k) {
      const int ch = wp * kWarpRows + lane;
      if (lane >= kWarpRows || (!kWhole && ch >= c)) return;
      // counted from the aligned word that holds the tape's first exponent: of memory before or
      // behind the tape no more than the rest of a word with one of its bytes is touched
      const uint32_t sub = exp_sub(tp);
      const long long first = (x + sub) & ~3LL;
      const uint32_t at = ((uint32_t)((x + sub) & 3) + (uint32_t)ch * (uint32_t)groups) & ~3u;
      const int8_t* src = tp.exps - sub + first + at;
      // whole tiles: a multiple of four exponents in all
      const int bytes = kWhole ? 4 : (int)min(4LL, x_all + sub - first - at);
      stage_copy_some(exp_at(slot, k, lane), src, bytes);
    };
    if (kTaped) {
      if (need_f) keep_exps(a.tp.f, 0);
      if (pre) keep_exps(a.tp.y, 1);
      if (per_row) keep_exps(a.tp.gate, 2);
    }
    auto keep = [&](const T* map, const zjai_tape& tp, int k) {
      if constexpr (kTaped)
        S::Kept::copy(kept_at(slot, k, 0), tp.codes + e, row, nv, tp.codes + elems);
      else
        S::Kept::copy(kept_at(slot, k, 0), map + e, row, nv, map + elems);
    };
    auto grad = [&](const T* map, int k) {
      S::Grad::copy(grad_at(slot, k, 0), map + e, row, nv, map + elems);
    };
    if (need_f) keep(a.f, a.tp.f, 0);
    if (pre) keep(a.y, a.tp.y, 1);
    if (pre) grad(a.dz, 1);
    if (per_row) keep(a.gate, a.tp.gate, 2);
    grad(a.dy, 0);
  };
  float acc[kRows][5];
#pragma unroll
  for (int j = 0; j < kRows; ++j)
#pragma unroll
    for (int i = 0; i < 5; ++i) acc[j][i] = 0.f;
  prm.load(a.prm, ch0, c);
  __syncthreads();
  Tiles tile(a.tiles, groups, cl.size), ahead = tile;
  if (ahead.on()) copy(ahead, 0);
  stage_commit();
  for (int slot = 0; tile.on(); tile.next(), slot ^= S::kSlots - 1) {
    const int at = tile.g * kTapeGroup + (lane & 7) * 4;
    const int nv = kWhole ? 4 : a.p - at;
    const long long e0 = ((long long)tile.img * a.c + ch0) * a.p + tile.g * kTapeGroup;
    const uint32_t x0 = (uint32_t)(((long long)tile.img * a.c + ch0) * groups + tile.g);
    auto kept = [&](const T* map, const zjai_tape& tp, int k, int j) {
      if constexpr (kTaped) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(exp_at(slot, k, j * 4 + (lane >> 3)));
        const int e = (int)(int8_t)(w >> ((x0 + row.x(j) + exp_sub(tp)) & 3) * 8);
        return taped4(S::Kept::words(kept_at(slot, k, j), tp.codes + e0, row, j, nv).x, e);
      } else {
        return S::Kept::get(kept_at(slot, k, j), map + e0, row, j, nv);
      }
    };
    auto grad = [&](const T* map, int k, int j) {
      return S::Grad::get(grad_at(slot, k, j), map + e0, row, j, nv);
    };
    F4 sg1 = all(1.f), slope1 = all(0.f);
    if (a.gate_c == 1) {
      Kept<kTaped, kVec, T> k;
      k.load(a.gate, a.tp.gate, (long long)tile.img * a.p, (long long)tile.img * groups + tile.g, at,
             a.p);
      sigmoid4(k.get(), &sg1, &slope1);
    }
    ahead.next();
    if (S::kSlots == 2) {
      if (ahead.on()) copy(ahead, slot ^ 1);
      stage_commit();
    }
    stage_wait<S::kSlots - 1>();
    if (kTaped || !kVec) __syncwarp();  // what other lanes copied
    F4 f[kRows], y[kRows];  // then LN(f), LN(y)
    if (need_f)
#pragma unroll
      for (int j = 0; j < kRows; ++j) f[j] = kept(a.f, a.tp.f, 0, j);
    if (pre)
#pragma unroll
      for (int j = 0; j < kRows; ++j) y[j] = kept(a.y, a.tp.y, 1, j);
    if (post) stats_part(rows, [&](int j) { return f[j]; }, ex, 0, cl.rank);
    if (pre) stats_part(rows, [&](int j) { return y[j]; }, ex, 2, cl.rank);
    if (post || pre) {
      cl.sync();
      if (post)
        join_first([&](int n, int of) { stats_join(rows, ex, 0, 0, inv_c, warps, cl, n, of); });
      if (pre)
        join_second([&](int n, int of) { stats_join(rows, ex, 2, 2, inv_c, warps, cl, n, of); });
      cl.sync();
    }
    F4 r2 = all(1.f), am = all(0.f), ay = all(0.f);
    if (post) {
      const F4 nm = total4(ex, 0), r1 = total4(ex, 1);
#pragma unroll
      for (int j = 0; j < kRows; ++j) f[j] = (f[j] + nm) * r1;
    }
    if (pre) {
      const F4 nm = total4(ex, 2);
      r2 = total4(ex, 3);
      F4 s0 = all(0.f), s1 = all(0.f);
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        y[j] = (y[j] + nm) * r2;
        const F4 t = grad(a.dz, 1, j) * prm.get(a.prm, kPreW, row.ch(j));
        if (row.on(j)) {
          s0 = s0 + t;
          s1 = fma4(t, y[j], s1);
        }
      }
      rows_to_part(s0, ex.at(0, wp));
      rows_to_part(s1, ex.at(1, wp));
      cl.sync();
      join_first([&](int n, int of) { sum_join(ex, 0, 4, -inv_c, warps, cl, n, of); });
      join_second([&](int n, int of) { sum_join(ex, 1, 5, -inv_c, warps, cl, n, of); });
      cl.sync();
      am = total4(ex, 4);  // negated means
      ay = total4(ex, 5);
    }
    F4 t0 = all(0.f), t1 = all(0.f), t2 = all(0.f);
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int ch = row.ch(j);
      const bool on = row.on(j);
      F4 d = grad(a.dy, 0, j);
      if (pre) {
        const F4 dz = grad(a.dz, 1, j);
        acc[j][3] += dot4(dz, y[j]);
        acc[j][4] += sum4(dz);
        d = fma4(fma4(y[j], ay, dz * prm.get(a.prm, kPreW, ch) + am), r2, d);
      }
      staged_store<kMode>(a.dx + e0, d, row, j, nv, ex.at(0, wp));
      if (!need_f) continue;
      const F4 u = post ? fma4(f[j], prm.get(a.prm, kPostW, ch), prm.get(a.prm, kPostB, ch)) : f[j];
      const F4 ds = d * prm.get(a.prm, kScale, ch);
      F4 sg = sg1, du = ds;
      if (per_row) {
        F4 slope;
        sigmoid4(kept(a.gate, a.tp.gate, 2, j), &sg, &slope);
        staged_store<kMode>(a.dgate + e0, ds * u * slope, row, j, nv, ex.at(0, wp));
      }
      if (a.gate_c) du = ds * sg;
      acc[j][0] += dot4(d * sg, u);
      if (a.gate_c == 1 && on) t2 = fma4(ds, u, t2);
      if (post) {
        acc[j][1] += dot4(du, f[j]);
        acc[j][2] += sum4(du);
        const F4 b = du * prm.get(a.prm, kPostW, ch);
        *b_at(slot, j) = flat(b);
        if (on) {
          t0 = t0 + b;
          t1 = fma4(b, f[j], t1);
        }
      } else {
        staged_store<kMode>(a.df + e0, du, row, j, nv, ex.at(0, wp));
      }
    }
    if (!need_f && a.df)
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        F4 d = grad(a.dy, 0, j);
        if (pre)
          d = fma4(fma4(y[j], ay, grad(a.dz, 1, j) * prm.get(a.prm, kPreW, row.ch(j)) + am), r2, d);
        staged_store<kMode>(a.df + e0, d, row, j, nv, ex.at(0, wp));
      }
    if (kTaped || !kVec) __syncwarp();  // read, before another lane copies over it
    // one slot: read now, but for b where dy was
    auto copy_one = [&]() {
      if (S::kSlots == 1) {
        if (ahead.on()) copy(ahead, 0);
        stage_commit();
      }
    };
    if (sizeof(T) != 4 || !post) copy_one();
    if (!post && a.gate_c != 1) continue;
    if (post) rows_to_part(t0, ex.at(0, wp)), rows_to_part(t1, ex.at(1, wp));
    if (a.gate_c == 1) rows_to_part(t2, ex.at(2, wp));
    cl.sync();
    if (post) {
      join_first([&](int n, int of) { sum_join(ex, 0, 6, -inv_c, warps, cl, n, of); });
      join_second([&](int n, int of) { sum_join(ex, 1, 7, -inv_c, warps, cl, n, of); });
    }
    if (a.gate_c == 1) sum_join(ex, 2, 8, 1.f, warps, cl, wp, warps);
    cl.sync();
    if (a.gate_c == 1 && threadIdx.x < 8 && cl.rank == 0)
      store4<kVec>(a.dgate + (long long)tile.img * a.p, at, a.p, total4(ex, 8) * slope1);
    if (!post) continue;
    const F4 bm = total4(ex, 6), bf = total4(ex, 7), r1 = total4(ex, 1);  // negated means
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      staged_store<kMode>(a.df + e0, fma4(f[j], bf, make4(*b_at(slot, j)) + bm) * r1, row, j, nv,
                          ex.at(0, wp));
    if (sizeof(T) == 4) copy_one();
  }
  stage_wait<0>();
  float* out = a.sums + (long long)(blockIdx.x / (unsigned)cl.size) * 5 * a.c + ch0;
#pragma unroll
  for (int j = 0; j < kRows; ++j)
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      float s = acc[j][i];
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if ((lane & 7) == 0 && row.on(j)) out[i * a.c + row.ch(j)] = s;
    }
}

// Any channel count and alignment: rows are read again for each pass, the parameter sums per channel
// in shared memory.
template <bool kTaped, bool kVec, class T>
__global__ void __launch_bounds__(kThreadsMost, 1) residual_norm_bwd_kernel(const BwdArgs<T> a) {
  constexpr int kRows = 0;
  __shared__ __align__(16) float parts[kMaxWarps * Exchange<4>::kPitch], totals[4 * 32];
  const Params<kRows> prm = {};
  extern __shared__ float acc_c[];  // [5][c of the block]
  const int warps = blockDim.x >> 5, wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cluster cl(a.cluster);
  const int ch0 = cl.rank * a.share, c = min(a.share, a.c - ch0);  // of the block
  const Rows<kRows> rows(c, a.share, a.c, warps);
  const Exchange<4> ex = {parts, totals};
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, per_row = a.gate_c > 1;
  const bool need_f = post || a.gate_c || a.prm.scale;
  for (int i = threadIdx.x; i < 5 * c; i += blockDim.x) acc_c[i] = 0.f;
  __syncthreads();
  for (Tiles tile(a.tiles, groups, cl.size); tile.on(); tile.next()) {
    const long long img = tile.img, base = img * a.c + ch0;
    const int g = tile.g, at = g * kTapeGroup + (lane & 7) * 4;
    using K = Kept<kTaped, kVec, T>;
    auto e0 = [&](int j) { return (base + rows.param(j)) * a.p; };
    auto grad = [&](const T* v, int j) {
      return rows.on(j) ? load4<kVec>(v + e0(j), at, a.p) : all(0.f);
    };
    auto kept = [&](const T* v, const zjai_tape& t, int j) {
      K k;
      k.load(v, t, e0(j), (base + rows.param(j)) * groups + g, at, a.p);
      return k.get();
    };
    F4 sg1 = all(1.f), slope1 = all(0.f);
    if (a.gate_c == 1) {
      K k;
      k.load(a.gate, a.tp.gate, img * a.p, img * groups + g, at, a.p);
      sigmoid4(k.get(), &sg1, &slope1);
    }
    F4 nm1 = all(0.f), r1 = all(1.f), nm2 = all(0.f), r2 = all(1.f), am = all(0.f), ay = all(0.f);
    if (post) stats_part(rows, [&](int j) { return kept(a.f, a.tp.f, j); }, ex, 0, cl.rank);
    if (pre) stats_part(rows, [&](int j) { return kept(a.y, a.tp.y, j); }, ex, 2, cl.rank);
    if (post || pre) {
      cl.sync();
      if (post) stats_join(rows, ex, 0, 0, inv_c, warps, cl, wp, warps);
      if (pre) stats_join(rows, ex, 2, 2, inv_c, warps, cl, wp, warps);
      cl.sync();
      if (post) nm1 = total4(ex, 0), r1 = total4(ex, 1);
      if (pre) nm2 = total4(ex, 2), r2 = total4(ex, 3);
    }
    auto fn_of = [&](int j) {
      const F4 f = kept(a.f, a.tp.f, j);
      return post ? (f + nm1) * r1 : f;
    };
    auto yn_of = [&](int j) { return (kept(a.y, a.tp.y, j) + nm2) * r2; };
    if (pre) {
      F4 s0 = all(0.f), s1 = all(0.f);
      FOR_ROWS(j) if (rows.on(j)) {
        const F4 t = grad(a.dz, j) * prm.get(a.prm, kPreW, ch0 + rows.param(j));
        s0 = s0 + t;
        s1 = fma4(t, yn_of(j), s1);
      }
      rows_to_part(s0, ex.at(0, wp));
      rows_to_part(s1, ex.at(1, wp));
      cl.sync();
      sum_join(ex, 0, 0, -inv_c, warps, cl, wp, warps);
      sum_join(ex, 1, 1, -inv_c, warps, cl, wp, warps);
      cl.sync();
      am = total4(ex, 0);  // negated means
      ay = total4(ex, 1);
    }
    auto d_of = [&](int j) {
      const F4 d = grad(a.dy, j);
      if (!pre) return d;
      const F4 t = grad(a.dz, j) * prm.get(a.prm, kPreW, ch0 + rows.param(j));
      return fma4(fma4(yn_of(j), ay, t + am), r2, d);
    };
    auto gate_of = [&](int j, F4* s, F4* slope) {
      *s = sg1;
      *slope = slope1;
      if (per_row) sigmoid4(kept(a.gate, a.tp.gate, j), s, slope);
    };
    F4 t0 = all(0.f), t1 = all(0.f), t2 = all(0.f);
    FOR_ROWS(j) {
      const int ch = ch0 + rows.param(j);
      const bool on = rows.on(j);
      const F4 d = d_of(j), fn = need_f ? fn_of(j) : all(0.f);
      F4 sg, slope;
      gate_of(j, &sg, &slope);
      const F4 u = fma4(fn, prm.get(a.prm, kPostW, ch), prm.get(a.prm, kPostB, ch));
      const F4 ds = d * prm.get(a.prm, kScale, ch), du = ds * sg, b = du * prm.get(a.prm, kPostW, ch);
      if (on) {
        store4<kVec>(a.dx + e0(j), at, a.p, d);
        if (!post && a.df) store4<kVec>(a.df + e0(j), at, a.p, du);
        if (per_row) store4<kVec>(a.dgate + e0(j), at, a.p, ds * u * slope);
        t0 = t0 + b;
        t1 = fma4(b, fn, t1);
        t2 = fma4(ds, u, t2);
      }
      const F4 dz = pre ? grad(a.dz, j) : all(0.f);
      const float v[5] = {dot4(d * sg, u), dot4(du, fn), sum4(du), pre ? dot4(dz, yn_of(j)) : 0.f,
                          sum4(dz)};
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        float s = v[i];
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((lane & 7) == 0 && on) acc_c[i * c + ch - ch0] += s;
      }
    }
    if (!post && a.gate_c != 1) continue;
    if (post) rows_to_part(t0, ex.at(0, wp)), rows_to_part(t1, ex.at(1, wp));
    if (a.gate_c == 1) rows_to_part(t2, ex.at(2, wp));
    cl.sync();
    if (post) {
      sum_join(ex, 0, 0, -inv_c, warps, cl, wp, warps);
      sum_join(ex, 1, 1, -inv_c, warps, cl, wp, warps);
    }
    if (a.gate_c == 1) sum_join(ex, 2, 2, 1.f, warps, cl, wp, warps);
    cl.sync();
    if (a.gate_c == 1 && threadIdx.x < 8 && cl.rank == 0)
      store4<kVec>(a.dgate + img * a.p, at, a.p, total4(ex, 2) * slope1);
    if (!post) continue;
    const F4 bm = total4(ex, 0), bf = total4(ex, 1);  // negated means
    FOR_ROWS(j) if (rows.on(j)) {
      const int ch = ch0 + rows.param(j);
      F4 sg, slope;
      gate_of(j, &sg, &slope);
      const F4 b = d_of(j) * prm.get(a.prm, kScale, ch) * sg * prm.get(a.prm, kPostW, ch);
      store4<kVec>(a.df + e0(j), at, a.p, fma4(fn_of(j), bf, b + bm) * r1);
    }
  }
  float* out = a.sums + (long long)(blockIdx.x / (unsigned)cl.size) * 5 * a.c + ch0;
  __syncthreads();
  for (int i = threadIdx.x; i < 5 * c; i += blockDim.x) out[(i / c) * a.c + i % c] = acc_c[i];
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

}  // namespace
}  // namespace zjai

using namespace zjai;

extern "C" {

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
    VecCheck vec(p);
    vec.map(ddy, es).map(ddz, es).map(df, es).map(dg, es).map(dyy, es);
    vec.map(gx, es).map(gf, es).map(gg, es);
    vec.map(dt.f.codes, 1).map(dt.gate.codes, 1).map(dt.y.codes, 1);
    vec.map(dt.f.exps, 1).map(dt.gate.exps, 1).map(dt.y.exps, 1);
    const Shape sh = shape_of(c, p, vec.ok);
    int blocks = 0;
    float* sums = nullptr;
    auto run = [&](auto t, auto tp) -> int {
      using T = decltype(t);
      constexpr bool kTaped = decltype(tp)::value;
      BwdArgs<T> a = {(const T*)ddy, (const T*)ddz, (const T*)df, (const T*)dg, (const T*)dyy, dt,
                      gate_channels, c, p, sh.cluster, sh.share, tiles, dp, (T*)gx, (T*)gf, (T*)gg,
                      nullptr};
      void (*k)(BwdArgs<T>) = vec.ok ? residual_norm_bwd_kernel<kTaped, true, T>
                                     : residual_norm_bwd_kernel<kTaped, false, T>;
      int smem = 5 * sh.share * (int)sizeof(float);
      if (sh.mode >= 0)
        smem = by_mode(sh.mode, [&](auto m) {
          using S = BwdSlot<decltype(m)::value, kTaped, T>;
          k = residual_norm_bwd_staged_kernel<decltype(m)::value, kTaped, T>;
          return S::kBytes * sh.warps + tail_bytes<4>(sh.share, sh.warps);
        });
      ZJAI_TRY(cuda_check(blocks_of(sh, k, smem, tiles, ctx->sms, &blocks), me));
      sums = static_cast<float*>(ctx->arena.alloc((size_t)blocks * 5 * c * sizeof(float)));
      if (!sums) return fail(ZJAI_LIMIT_EXCEEDED, "device arena exhausted (parameter sums)");
      a.sums = sums;
      return cuda_check(launch(sh, k, smem, blocks, ctx->stream, a), me);
    };
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      return taped ? run(t, std::true_type()) : run(t, std::false_type());
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
