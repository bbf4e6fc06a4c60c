// The residual step of a block with its norms, gate and scale (zjai_gated_residual_norm): the
// mathematics and the layout are in residual_norm.cuh.
#include "residual_norm.cuh"

namespace zjai {
namespace {

template <class T>
struct FwdArgs {
  const T *x, *f, *gate;
  int gate_c, c, p, cluster, share;
  long long tiles;
  zjai_residual_params prm;
  T *y, *z;
  zjai_residual_tapes tp;
};

// Rows held, the next tile copied ahead into the other of two slots; with one, as soon as the current
// one has been read: rows that start anywhere, whose copies want the rest as L1 cache (8 x 128 x 127 x
// 129, two and one: f32 146 and 114 us, bf16 98 and 94 us).
template <int kMode>
constexpr int fwd_slots() {
  return kMode == kAnywhere ? 1 : 2;
}
template <int kMode, class T>
constexpr int fwd_slot_bytes() {  // per warp: f, x and the gate's logits
  return 3 * kStagedRows * Region<kMode, T>::kBytes;
}
template <int kMode, class T>
__global__ void __launch_bounds__(kThreadsMost, 1)
    residual_norm_staged_kernel(const FwdArgs<T> a) {
  using R = Region<kMode, T>;
  constexpr int kRows = kStagedRows;
  constexpr bool kWhole = kMode == kWholeTiles, kVec = kMode != kAnywhere;
  __shared__ __align__(16) float totals[2 * 32];
  extern __shared__ __align__(16) char slots[];
  const int warps = blockDim.x >> 5, wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cluster cl(a.cluster);
  const int ch0 = cl.rank * a.share, c = min(a.share, a.c - ch0);  // of the block
  const Rows<kRows, kWhole> rows(c, a.share, a.c, warps);
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, per_row = a.gate_c > 1;
  const StagedRows<kMode> row(c, a.p, groups);
  constexpr int kSlots = fwd_slots<kMode>();
  char* mine = slots + wp * kSlots * fwd_slot_bytes<kMode, T>();
  Params<kRows> prm = {nullptr, a.share};
  Exchange<2> ex = {nullptr, totals};
  take_tail(slots + warps * kSlots * fwd_slot_bytes<kMode, T>(), a.share, &prm.v, &ex);
  auto place = [&](int slot, int k, int j) {
    return mine + ((slot * 3 + k) * kRows + j) * R::kBytes;
  };
  const long long elems = a.tiles / groups * a.c * a.p;
  auto copy = [&](const Tiles& t, int slot) {
    const long long e = ((long long)t.img * a.c + ch0) * a.p + t.g * kTapeGroup;
    const int nv = kWhole ? 4 : a.p - (t.g * kTapeGroup + (lane & 7) * 4);
    R::copy(place(slot, 0, 0), a.f + e, row, nv, a.f + elems);
    R::copy(place(slot, 1, 0), a.x + e, row, nv, a.x + elems);
    if (per_row) R::copy(place(slot, 2, 0), a.gate + e, row, nv, a.gate + elems);
  };
  prm.load(a.prm, ch0, c);
  __syncthreads();
  Tiles tile(a.tiles, groups, cl.size), ahead = tile;
  if (ahead.on()) copy(ahead, 0);
  stage_commit();
  for (int slot = 0; tile.on(); tile.next(), slot ^= kSlots - 1) {
    ahead.next();
    if (kSlots == 2) {
      if (ahead.on()) copy(ahead, slot ^ 1);
      stage_commit();
    }
    const int at = tile.g * kTapeGroup + (lane & 7) * 4;
    const int nv = kWhole ? 4 : a.p - at;
    const long long e0 = ((long long)tile.img * a.c + ch0) * a.p + tile.g * kTapeGroup;
    const long long x0 = ((long long)tile.img * a.c + ch0) * groups + tile.g;
    F4 gate1 = all(0.f), sg1 = all(1.f), unused;
    if (a.gate_c == 1) {
      gate1 = load4<kVec>(a.gate + (long long)tile.img * a.p, at, a.p);
      sigmoid4(gate1, &sg1, &unused);
    }
    stage_wait<kSlots - 1>();
    if (!kVec) __syncwarp();  // what other lanes copied
    auto hold = [&](const zjai_tape& t, int j, F4 v) {
      staged_hold<kMode>(t.codes + e0, t.exps + x0, v, row, j, nv, ex.at(0, wp));
    };
    F4 nm = all(0.f), r = all(1.f);  // of f, then of y: the negated mean and 1 / sigma
    auto exchange = [&](auto v) {
      stats_part(rows, v, ex, 0, cl.rank);
      cl.sync();
      stats_join(rows, ex, 0, 0, inv_c, warps, cl, wp, warps);
      cl.sync();
      nm = total4(ex, 0);
      r = total4(ex, 1);
    };
    auto get = [&](const T* map, int k, int j) {
      return R::get(place(slot, k, j), map + e0, row, j, nv);
    };
    if (post) exchange([&](int j) { return get(a.f, 0, j); });
    if (a.gate_c == 1 && a.tp.gate.codes && wp == 0 && cl.rank == 0)
      tape_store4<kVec>(a.tp.gate, (long long)tile.img * a.p, (long long)tile.img * groups + tile.g,
                        at, a.p, gate1, lane < 8);
    F4 y[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const F4 f = get(a.f, 0, j);
      F4 u = f, s = sg1;
      if (post)
        u = fma4((f + nm) * r, prm.get(a.prm, kPostW, row.ch(j)), prm.get(a.prm, kPostB, row.ch(j)));
      if (a.tp.f.codes) hold(a.tp.f, j, f);
      if (per_row) {
        const F4 g = get(a.gate, 2, j);
        sigmoid4(g, &s, &unused);
        if (a.tp.gate.codes) hold(a.tp.gate, j, g);
      }
      y[j] = fma4(s * prm.get(a.prm, kScale, row.ch(j)), u, get(a.x, 1, j));
      staged_store<kMode>(a.y + e0, y[j], row, j, nv, ex.at(0, wp));
      if (a.tp.y.codes) hold(a.tp.y, j, kWhole ? y[j] : clip4<kVec>(y[j], at, a.p));
    }
    if (kSlots == 1) {
      __syncwarp();  // read, before another lane copies over it
      if (ahead.on()) copy(ahead, 0);
      stage_commit();
    }
    if (!pre) continue;
    exchange([&](int j) { return y[j]; });
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const F4 z =
          fma4((y[j] + nm) * r, prm.get(a.prm, kPreW, row.ch(j)), prm.get(a.prm, kPreB, row.ch(j)));
      staged_store<kMode>(a.z + e0, z, row, j, nv, ex.at(0, wp));
      if (a.tp.z.codes) hold(a.tp.z, j, kWhole ? z : clip4<kVec>(z, at, a.p));
    }
  }
  stage_wait<0>();
}

// Any channel count and alignment: rows are read again for each pass.
template <bool kVec, class T>
__global__ void __launch_bounds__(kThreadsMost, 1) residual_norm_kernel(const FwdArgs<T> a) {
  constexpr int kRows = 0;
  __shared__ __align__(16) float parts[kMaxWarps * Exchange<2>::kPitch], totals[2 * 32];
  const Params<kRows> prm = {};
  const int warps = blockDim.x >> 5, wp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Cluster cl(a.cluster);
  const int ch0 = cl.rank * a.share, c = min(a.share, a.c - ch0);  // of the block
  const Rows<kRows> rows(c, a.share, a.c, warps);
  const Exchange<2> ex = {parts, totals};
  const int groups = (int)tape_groups(a.p);
  const float inv_c = 1.f / (float)a.c;
  const bool post = a.prm.post_weight, pre = a.prm.pre_weight, per_row = a.gate_c > 1;
  for (Tiles tile(a.tiles, groups, cl.size); tile.on(); tile.next()) {
    const long long img = tile.img, base = img * a.c + ch0;
    const int g = tile.g, at = g * kTapeGroup + (lane & 7) * 4;
    // a row's first element; its group's place among the exponents
    auto e0 = [&](int j) { return (base + rows.row(j)) * a.p; };
    auto ge = [&](int j) { return (base + rows.row(j)) * groups + g; };
    auto load = [&](const T* v, int j) {
      return rows.on(j) ? load4<kVec>(v + e0(j), at, a.p) : all(0.f);
    };
    F4 gate1 = all(0.f), sg1 = all(1.f), unused;
    if (a.gate_c == 1) {
      gate1 = load4<kVec>(a.gate + img * a.p, at, a.p);
      sigmoid4(gate1, &sg1, &unused);
      if (a.tp.gate.codes && wp == 0 && cl.rank == 0)
        tape_store4<kVec>(a.tp.gate, img * a.p, img * groups + g, at, a.p, gate1, lane < 8);
    }
    F4 nm = all(0.f), r = all(1.f);  // of f, then of y: the negated mean and 1 / sigma
    auto exchange = [&](auto v) {
      stats_part(rows, v, ex, 0, cl.rank);
      cl.sync();
      stats_join(rows, ex, 0, 0, inv_c, warps, cl, wp, warps);
      cl.sync();
      nm = total4(ex, 0);
      r = total4(ex, 1);
    };
    if (post) exchange([&](int j) { return load(a.f, j); });
    const F4 nm1 = nm, r1 = r;
    auto y_of = [&](int j) {
      const int ch = ch0 + rows.param(j);
      F4 u = load(a.f, j), s = sg1;
      if (post)
        u = fma4((u + nm1) * r1, prm.get(a.prm, kPostW, ch), prm.get(a.prm, kPostB, ch));
      if (per_row) sigmoid4(load(a.gate, j), &s, &unused);
      return fma4(s * prm.get(a.prm, kScale, ch), u, load(a.x, j));
    };
    if (pre) exchange(y_of);
    FOR_ROWS(j) {
      const bool on = rows.on(j);
      const F4 y = y_of(j);
      if (on) store4<kVec>(a.y + e0(j), at, a.p, y);
      if (a.tp.f.codes) tape_store4<kVec>(a.tp.f, e0(j), ge(j), at, a.p, load(a.f, j), on);
      if (per_row && a.tp.gate.codes)
        tape_store4<kVec>(a.tp.gate, e0(j), ge(j), at, a.p, load(a.gate, j), on);
      if (a.tp.y.codes)
        tape_store4<kVec>(a.tp.y, e0(j), ge(j), at, a.p, clip4<kVec>(y, at, a.p), on);
      if (!pre) continue;
      const int ch = ch0 + rows.param(j);
      const F4 z = fma4((y + nm) * r, prm.get(a.prm, kPreW, ch), prm.get(a.prm, kPreB, ch));
      if (on) store4<kVec>(a.z + e0(j), at, a.p, z);
      if (a.tp.z.codes)
        tape_store4<kVec>(a.tp.z, e0(j), ge(j), at, a.p, clip4<kVec>(z, at, a.p), on);
    }
  }
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
    VecCheck vec(p);
    vec.map(dx, es).map(df, es).map(dg, es).map(dyo, es).map(dzo, es);
    for (zjai_tape* t : tt) vec.map(t->codes, 1);
    const long long tiles = (long long)n * (long long)groups;
    const Shape sh = shape_of(c, p, vec.ok);
    ZJAI_TRY(by_dtype(dtype, [&](auto t) -> int {
      using T = decltype(t);
      FwdArgs<T> a = {(const T*)dx, (const T*)df, (const T*)dg, gate_channels, c, p, sh.cluster,
                      sh.share, tiles, dp, (T*)dyo, (T*)dzo, dt};
      void (*k)(FwdArgs<T>) = vec.ok ? residual_norm_kernel<true, T> : residual_norm_kernel<false, T>;
      int smem = 0;
      if (sh.mode >= 0)
        smem = by_mode(sh.mode, [&](auto m) {
          constexpr int kMode = decltype(m)::value;
          k = residual_norm_staged_kernel<kMode, T>;
          return fwd_slots<kMode>() * fwd_slot_bytes<kMode, T>() * sh.warps +
                 tail_bytes<2>(sh.share, sh.warps);
        });
      int count = 0;
      ZJAI_TRY(cuda_check(blocks_of(sh, k, smem, tiles, ctx->sms, &count), me));
      return cuda_check(launch(sh, k, smem, count, ctx->stream, a), me);
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

}  // extern "C"
