// Packed causal attention, backward.  With P from the saved row statistics (log2 units, P = 2^(s c - lse)):
//   delta_i = sum_d o_id dO_id,  dP = dO V^T,  dS = P (dP - delta),  dQ = sm_scale dS K,  dK = sm_scale dS^T Q,
//   dV = P^T dO, dK and dV summed over the query heads that share the key / value head.
//
// Two kernels, as the flash-entropy backward has them (no atomics, so a gradient's bits do not depend on timing):
//  * packed_bwd_dq: 128 queries of one head, 32 a wave, one a lane; S^T = K Q^T and dP^T = V dO^T over 64-key stages up to
//    the diagonal, then dQ^T += K^T dS^T.  Its prologue forms delta.
//  * packed_bwd_dkdv: 128 keys of one key / value head, 32 a wave, one a lane; over 32-query stages from the diagonal on,
//    for one query head of the group after the other, S = Q K^T and dP = dO V^T, then dV^T += dO^T P, dK^T += Q^T dS.
// Where some workgroups have far more to do than others, heavy tiles are split (packed.h; dk / dv: over the group's heads
// first), into fp32 sums that packed_bwd_join (or packed_bwd_sum) adds in order.
// Both are bound by the matrix pipes at the chip's power (prompts of 12000 and 4384 tokens, 8 heads over 2 of 128: dq 451 us,
// 1.11 PFLOP/s of its three products; dk / dv 619 us, 1.08 of its four; 1.7-1.8 GHz, 62-67% of the busy CUs' MFMA cycles).
// Stages that a wave does not see at all are skipped, those on the diagonal (or at a sequence's end) masked.
// P and dS are rounded to the 16-bit type as operands, the gradients once at the end.  delta takes o as it was before its
// rounding, from the forward's o and the rounding's error beside it: with the rounded o alone, delta's error was a third of
// what the roundings of dS and of the gradients give (fp16, dq and dk: 1.52 times the error of one rounding, 1.43 so).
#include "packed.h"

namespace vmo {

constexpr int kDqKeys = 64;      // keys of a dq stage
constexpr int kKvQueries = 32;   // queries of a dk / dv stage

template <int D> constexpr int packed_dq_lds() {
  constexpr int ring = 2 * kDqKeys * D * 2 * 2;
  constexpr int least = kPackedWaves * kEpiPatchBytes;
  return ring > least ? ring : least;
}
// V's 128 rows in LDS at D = 128 (in registers they would spill)
template <int D> constexpr bool packed_v_in_lds() { return D >= 128; }
template <int D> constexpr int packed_kv_stage() { return kKvQueries * D * 2 * 2 + 512; }
template <int D> constexpr int packed_kv_lds() {
  constexpr int ring = 2 * packed_kv_stage<D>() + (packed_v_in_lds<D>() ? kPackedTile * D * 2 : 0);
  constexpr int least = kPackedWaves * kEpiPatchBytes;
  return ring > least ? ring : least;
}

template <class V8, int RB>
__device__ __forceinline__ V8 packed_tr(const VMO_LDS char* block16, int trow, int tchunk, int tbyte, int a) {
  const int c0 = trow * RB + (((4 * a + tchunk) ^ swz_rows<RB>(trow)) * 16 + tbyte);
  return lds_read_tr8<V8>(block16 + c0, block16 + 8 * RB + (c0 ^ 32));
}

template <bool F16, int D>
__global__ __launch_bounds__(64 * kPackedWaves, 2) void packed_bwd_dq_kernel(PackedParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  using V8 = typename E::V8;
  constexpr int RB = D * 2, K_BYTES = kDqKeys * RB, STAGE = 2 * K_BYTES, NA = D / 32, NDS = D / 16;
  constexpr int PF = D <= 64 ? 0 : 2;   // operand reads in flight ahead of their product
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  VMO_LDS char* smem = (VMO_LDS char*)smem_raw;
  const uint32_t smem_u32 = (uint32_t)(uintptr_t)smem;
  auto uni = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };

  const PackedPlace place = packed_place(p, blockIdx.x);
  const int head = uni(packed_head(place.pos, p.heads));
  const PackedTile w = packed_tile<false>(p, place.idx);
  const int slot_no = w.number * p.per + place.pos;
  packed_record<false>(p, w, slot_no);
  if (w.tile < 0) {
    packed_zero_rest<T, D>((T*)p.dq + head * p.dq_sh, p.dq_sn, p.q_off, p.n, p.tq, w.which, w.spare);
    return;
  }
  const int nq = uni(w.s.nq), nk = uni(w.s.nk), qb = uni(w.s.qb), kb = uni(w.s.kb);
  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int q0 = uni(w.tile) * kPackedTile + wave * 32;
  const bool live = q0 < nq;
  const int past = nk - nq;
  auto keys_of = [&](int row) __attribute__((always_inline)) { return p.causal ? min(max(past + row + 1, 0), nk) : nk; };
  const int row = min(q0 + l32, nq - 1);
  const int lim = keys_of(row);
  const int lo = uni(keys_of(min(q0, nq - 1))), hi = uni(keys_of(min(q0 + 31, nq - 1)));
  const int stages = uni((keys_of(min(uni(w.tile) * kPackedTile + kPackedTile - 1, nq - 1)) + kDqKeys - 1) / kDqKeys);
  const int parts = uni(w.parts), t0 = uni((int)((int64_t)w.part * stages / parts)), t1 = uni((int)((int64_t)(w.part + 1) * stages / parts));

  // Q^T and dO^T as B operands (one query a lane); delta in fp32
  V8 qf[NDS], dof[NDS];
  float delta = 0.f;
  const int64_t tok = qb + row;
  {
    const T* qp = (const T*)p.q + (int64_t)head * p.q_sh + tok * p.q_sn + hl * 8;
    const T* dp = (const T*)p.dO + (int64_t)head * p.do_sh + tok * p.do_sn + hl * 8;
    const T* op = (const T*)p.o + (int64_t)head * p.o_sh + tok * p.o_sn + hl * 8;
    const T* lp = p.o_low ? (const T*)p.o_low + (int64_t)head * p.o_sh + tok * p.o_sn + hl * 8 : nullptr;
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      qf[ds] = *(const V8*)(qp + ds * 16);
      asm volatile("" : "+v"(qf[ds]));
    }
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      dof[ds] = *(const V8*)(dp + ds * 16);
      asm volatile("" : "+v"(dof[ds]));
      const V8 y = *(const V8*)(op + ds * 16), z = lp ? *(const V8*)(lp + ds * 16) : V8{};
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)dof[ds][e], (float)y[e] + (float)z[e], delta);
    }
  }
  float alpha = -wave_sum32(delta);
  float lse = p.lse[(int64_t)head * p.st_sh + tok];
  asm volatile("" : "+v"(alpha), "+v"(lse));   // waited for here: a wait in the loop would also wait for the copies
  if (live && w.part == 0 && hl == 0 && q0 + l32 < nq) p.neg_delta[(int64_t)head * p.tq + tok] = alpha;

  const T* kbase = (const T*)p.k + (int64_t)(head / p.group) * p.k_sh + (int64_t)kb * p.k_sn;
  const T* vbase = (const T*)p.v + (int64_t)(head / p.group) * p.v_sh + (int64_t)kb * p.v_sn;
  const TileCopy<T, D, kPackedWaves> kcopy(kbase, p.k_sn, wave, lane), vcopy(vbase, p.v_sn, wave, lane);
  auto issue = [&](int t) __attribute__((always_inline)) {
    const uint32_t st = smem_u32 + (uint32_t)((t & 1) * STAGE);
    kcopy.issue(t * kDqKeys, nk, st);
    vcopy.issue(t * kDqKeys, nk, st + K_BYTES);
  };
  f32x16 acc[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) acc[a] = f32x16{};
  const float c = p.c;
  const int sw = swz_rows<RB>(l32);
  const int trow = 4 * hl + ((lane & 15) >> 2), tchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), tbyte = (lane & 1) * 8;

  auto stage = [&](int t, auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const VMO_LDS char* Ks = smem + (t & 1) * STAGE;
    const VMO_LDS char* Vs = Ks + K_BYTES;
    f32x16 s[2] = {f32x16{}, f32x16{}}, dp[2] = {f32x16{}, f32x16{}};
    prefetched_chain<4 * NDS, PF>(
        [&](int i) __attribute__((always_inline)) {
          const int kb2 = i / (2 * NDS), j = i % (2 * NDS);
          return lds_read8<V8>((j < NDS ? Ks : Vs) + (32 * kb2 + l32) * RB + ((2 * (j % NDS) + hl) ^ sw) * 16);
        },
        [&](int i, const V8& x) __attribute__((always_inline)) {
          const int kb2 = i / (2 * NDS), j = i % (2 * NDS);
          if (j < NDS) s[kb2] = E::mfma(x, qf[j], s[kb2]);
          else dp[kb2] = E::mfma(x, dof[j - NDS], dp[kb2]);
        });
    if constexpr (PF > 0) {
      struct Chain {
        static constexpr int reads(int) { return 1; }
        static constexpr int mfmas(int) { return 1; }
        static constexpr int ahead(int) { return 2; }
        static constexpr int lead() { return 0; }
      };
      pin_chain<Chain, 4 * NDS>();
    }
    V8 G[2][2];
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float g = fast_exp2(fmaf(s[kb2][r], c, -lse)) * (dp[kb2][r] + alpha);
        if (MASKED) g = t * kDqKeys + 32 * kb2 + 8 * (r >> 2) + 4 * hl + (r & 3) < lim ? g : 0.f;
        G[kb2][r >> 3][r & 7] = to_elem<T>(g);
      }
    if constexpr (MASKED) {
#pragma unroll
      for (int kb2 = 0; kb2 < 2; ++kb2) {
        const int nvis = lim - t * kDqKeys - 32 * kb2;
        masked_product<F16, RB, 1>(acc, Ks + 32 * kb2 * RB, G[kb2], lane, [&](int key) { return key < nvis; });
      }
    } else {
      prefetched_chain<4 * NA, PF>(
          [&](int i) __attribute__((always_inline)) {
            return packed_tr<V8, RB>(Ks + 16 * (i % 4) * RB, trow, tchunk, tbyte, i / 4);
          },
          [&](int i, const V8& x) __attribute__((always_inline)) {
            acc[i / 4] = E::mfma(x, G[(i % 4) >> 1][i & 1], acc[i / 4]);
          });
    }
  };
  if (t1 > t0) {
    issue(t0);
    const int n_full = live ? uni(min(max(lo / kDqKeys, t0), t1)) : t0;
    auto top = [&](int t) __attribute__((always_inline)) {
      tile_sync<0>();   // stage t has landed for every wave, and stage t - 1's slot is free
      if (t + 1 < t1) issue(t + 1);
    };
    int t = t0;
    for (; t < n_full; ++t) {
      top(t);
      stage(t, std::false_type{});
    }
    for (; t < t1; ++t) {
      top(t);
      if (live && t * kDqKeys < hi) stage(t, std::true_type{});
    }
  }
  __syncthreads();
  if (!live) return;
  VMO_LDS float* patch = (VMO_LDS float*)(smem + wave * kEpiPatchBytes);
  if (parts > 1) {
    float* out = p.part + ((int64_t)slot_no * kPackedTile + wave * 32) * D;
    store_acc_rows<F16>(patch, acc, NA, p.sm_scale, kGradStoreF32, (char*)out, D * 4, min(32, nq - q0), lane);
    return;
  }
  T* out = (T*)p.dq + (int64_t)head * p.dq_sh + (int64_t)(qb + q0) * p.dq_sn;
  store_acc_rows<F16>(patch, acc, NA, p.sm_scale, kGradStore, (char*)out, p.dq_sn * 2, min(32, nq - q0), lane);
}

template <bool F16, int D>
__global__ __launch_bounds__(64 * kPackedWaves, 2) void packed_bwd_dkdv_kernel(PackedParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  using V8 = typename E::V8;
  constexpr int RB = D * 2, Q_BYTES = kKvQueries * RB, STAGE = packed_kv_stage<D>(), NA = D / 32, NDS = D / 16;
  constexpr bool V_LDS = packed_v_in_lds<D>();
  constexpr int PF = 2;
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  VMO_LDS char* smem = (VMO_LDS char*)smem_raw;
  const uint32_t smem_u32 = (uint32_t)(uintptr_t)smem;
  auto uni = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };

  // kv_heads x splits workgroups of one key tile (a share stays on its XCDs, so its heads' rows do)
  const PackedPlace place = packed_place(p, blockIdx.x);
  const int hs = uni(packed_head(place.pos, p.per));
  const int kvh = hs / p.splits, split = hs % p.splits;
  const PackedTile w = packed_tile<true>(p, place.idx);
  const int slot_no = w.number * p.per + place.pos;
  packed_record<true>(p, w, slot_no);
  if (w.tile < 0) {
    if (p.splits == 1) {
      packed_zero_rest<T, D>((T*)p.dk + kvh * p.dk_sh, p.dk_sn, p.k_off, p.n, p.tk, w.which, w.spare);
      packed_zero_rest<T, D>((T*)p.dv + kvh * p.dv_sh, p.dv_sn, p.k_off, p.n, p.tk, w.which, w.spare);
    }
    return;
  }
  const int nq = uni(w.s.nq), nk = uni(w.s.nk), qb = uni(w.s.qb), kb = uni(w.s.kb);
  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int tile0 = uni(w.tile) * kPackedTile, k0 = tile0 + wave * 32;
  const bool live = k0 < nk;
  const int key = min(k0 + l32, nk - 1);
  // the first row that sees a key, counted from the wave's and the workgroup's first keys
  const int past = nk - nq;
  auto first_row = [&](int j) __attribute__((always_inline)) { return p.causal ? max(j - past, 0) : 0; };
  const int from = first_row(key);
  const int w_from = uni(first_row(min(k0, nk - 1))), w_whole = uni(first_row(min(k0 + 31, nk - 1)));
  const int t0 = uni(first_row(tile0) / kKvQueries), t1 = uni((nq + kKvQueries - 1) / kKvQueries);
  // the share's heads; the part's steps of all (head, stage) pairs: from stage b0 of head g0 up to stage b1 of head g1
  const int per = p.group / p.splits;
  const int steps = t1 > t0 ? t1 - t0 : 0, parts = uni(w.parts);
  const int64_t all = (int64_t)steps * per;
  const int i0 = uni((int)(w.part * all / parts)), i1 = uni((int)((w.part + 1) * all / parts)), n_it = i1 - i0;
  const int g0 = steps ? uni(i0 / steps) : 0, g1 = steps ? uni((i1 - 1) / steps) : -1, h0 = kvh * p.group + split * per + g0;
  const int b0 = t0 + i0 - g0 * steps, b1 = t0 + i1 - g1 * steps;

  const T* kp0 = (const T*)p.k + (int64_t)kvh * p.k_sh + (int64_t)kb * p.k_sn;
  const T* vp0 = (const T*)p.v + (int64_t)kvh * p.v_sh + (int64_t)kb * p.v_sn;
  V8 kf[NDS], vf[V_LDS ? 1 : NDS];
#pragma unroll
  for (int ds = 0; ds < NDS; ++ds) {
    kf[ds] = *(const V8*)(kp0 + (int64_t)key * p.k_sn + hl * 8 + ds * 16);
    asm volatile("" : "+v"(kf[ds]));
  }
  const VMO_LDS char* vt_row = smem + 2 * STAGE + (wave * 32 + l32) * RB;
  if constexpr (V_LDS) {   // the workgroup's 128 V rows, once (landed by the first tile_sync)
    const TileCopy<T, D, kPackedWaves, D, kPackedTile> vrows(vp0, p.v_sn, wave, lane);
    vrows.issue(tile0, nk, smem_u32 + 2 * STAGE);
  } else {
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      vf[ds] = *(const V8*)(vp0 + (int64_t)key * p.v_sn + hl * 8 + ds * 16);
      asm volatile("" : "+v"(vf[ds]));
    }
  }

  TileCopy<T, D, kPackedWaves, D, kKvQueries> qcopy((const T*)p.q + (int64_t)h0 * p.q_sh + (int64_t)qb * p.q_sn, p.q_sn, wave, lane);
  TileCopy<T, D, kPackedWaves, D, kKvQueries> docopy((const T*)p.dO + (int64_t)h0 * p.do_sh + (int64_t)qb * p.do_sn, p.do_sn, wave,
                                                     lane);
  const float* lse_h = p.lse + (int64_t)h0 * p.st_sh + qb;
  const float* nd_h = p.neg_delta + (int64_t)h0 * p.tq + qb;
  int t_next = b0;   // the stage that the next issue copies; past the last one comes the next head's first
  auto issue = [&](int slot) __attribute__((always_inline)) {
    const uint32_t st = smem_u32 + (uint32_t)(slot * STAGE);
    const int row0 = t_next * kKvQueries;
    qcopy.issue(row0, nq, st);
    docopy.issue(row0, nq, st + Q_BYTES);
    if (wave == 0) {   // the rows' lse and -delta (64 places each, 32 used), from scalar bases: as 64-bit lane addresses they
      // were kept in scratch, whose reload waits for every copy in flight
      const uint32_t at = (uint32_t)min(row0 + lane, nq - 1) * 4;
      dma4_async_s((uint64_t)(uintptr_t)lse_h, at, st + 2 * Q_BYTES);
      dma4_async_s((uint64_t)(uintptr_t)nd_h, at, st + 2 * Q_BYTES + 256);
    }
    if (++t_next == t1) {
      t_next = t0;
      qcopy.ubase = uniform64(qcopy.ubase + (uint64_t)p.q_sh * 2);
      docopy.ubase = uniform64(docopy.ubase + (uint64_t)p.do_sh * 2);
      lse_h += p.st_sh;
      nd_h += p.tq;
    }
  };

  f32x16 dk[NA], dv[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) dk[a] = dv[a] = f32x16{};
  const float c = p.c;
  const int sw = swz_rows<RB>(l32);
  const int trow = 4 * hl + ((lane & 15) >> 2), tchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), tbyte = (lane & 1) * 8;

  auto stage = [&](int slot, int row0, auto masked_tag) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked_tag)::value;
    const VMO_LDS char* Qs = smem + slot * STAGE;
    const VMO_LDS char* dOs = Qs + Q_BYTES;
    const VMO_LDS float* sts = (const VMO_LDS float*)(dOs + Q_BYTES);
    f32x16 s = f32x16{}, dp;
#pragma unroll
    for (int g = 0; g < 4; ++g) {   // dP starts from -delta
      const f32x4 av = *(const VMO_LDS f32x4*)(sts + 64 + 8 * g + 4 * hl);
#pragma unroll
      for (int e = 0; e < 4; ++e) dp[4 * g + e] = av[e];
    }
    struct Ops { V8 a, b; };
    prefetched_chain<2 * NDS, PF>(
        [&](int i) __attribute__((always_inline)) {
          Ops o;
          const int off = ((2 * (i % NDS) + hl) ^ sw) * 16;
          o.a = lds_read8<V8>((i < NDS ? Qs : dOs) + l32 * RB + off);
          o.b = i < NDS ? kf[i] : V_LDS ? lds_read8<V8>(vt_row + off) : vf[V_LDS ? 0 : i - NDS];
          return o;
        },
        [&](int i, const Ops& o) __attribute__((always_inline)) {
          if (i < NDS) s = E::mfma(o.a, o.b, s);
          else dp = E::mfma(o.a, o.b, dp);
        });
    struct Chain {
      static constexpr int reads(int i) { return i < NDS ? 1 : 1 + (V_LDS ? 1 : 0); }
      static constexpr int mfmas(int) { return 1; }
      static constexpr int ahead(int) { return 2; }
      static constexpr int lead() { return 4; }
    };
    pin_chain<Chain, 2 * NDS>();
    auto sees = [&](int r) __attribute__((always_inline)) { return row0 + r >= from && row0 + r < nq; };
    V8 P[2], G[2];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 lv = *(const VMO_LDS f32x4*)(sts + 8 * g + 4 * hl);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * g + e;
        float pv = fast_exp2(fmaf(s[r], c, -lv[e]));
        float gv = pv * dp[r];
        if (MASKED) {
          const bool ok = sees(8 * g + 4 * hl + e);
          pv = ok ? pv : 0.f;
          gv = ok ? gv : 0.f;
        }
        P[r >> 3][r & 7] = to_elem<T>(pv);
        G[r >> 3][r & 7] = to_elem<T>(gv);
      }
    }
    if constexpr (MASKED) {
      masked_product<F16, RB, 1>(dv, dOs, P, lane, sees);
      masked_product<F16, RB, 1>(dk, Qs, G, lane, sees);
    } else {
      prefetched_chain<4 * NA, PF>(
          [&](int i) __attribute__((always_inline)) {
            return packed_tr<V8, RB>((i < 2 * NA ? dOs : Qs) + 16 * (i % 2) * RB, trow, tchunk, tbyte, (i / 2) % NA);
          },
          [&](int i, const V8& x) __attribute__((always_inline)) {
            if (i < 2 * NA) dv[i / 2] = E::mfma(x, P[i % 2], dv[i / 2]);
            else dk[i / 2 - NA] = E::mfma(x, G[i % 2], dk[i / 2 - NA]);
          });
    }
  };
  if (n_it > 0) {
    issue(0);
    // a head's stages: those before the wave's keys are seen whole, those that its 32 keys see whole, the partial last one
    // (three loops: with both kinds in one body the compiler spills the accumulators)
    const int a0 = min(max((w_whole + kKvQueries - 1) / kKvQueries, t0), t1), a1 = live ? max(nq / kKvQueries, a0) : a0;
    int it = 0;
    auto top = [&]() __attribute__((always_inline)) {
      tile_sync<0>();   // this stage has landed for every wave, and the other slot is free
      if (it + 1 < n_it) issue((it + 1) & 1);
    };
    auto masked = [&](int t) __attribute__((always_inline)) {
      top();
      if (live && (t + 1) * kKvQueries > w_from) stage(it & 1, t * kKvQueries, std::true_type{});
      ++it;
    };
    for (int g = g0; g <= g1; ++g) {
      int t = g == g0 ? b0 : t0;
      const int end = g == g1 ? b1 : t1;
      for (const int upto = live ? min(a0, end) : end; t < upto; ++t) masked(t);
      for (const int upto = min(a1, end); t < upto; ++t) {
        top();
        stage(it & 1, t * kKvQueries, std::false_type{});
        ++it;
      }
      for (; t < end; ++t) masked(t);
    }
  } else {
    tile_sync<0>();   // V's copies have landed before the patches take their place
  }
  __syncthreads();
  if (!live) return;
  VMO_LDS float* patch = (VMO_LDS float*)(smem + wave * kEpiPatchBytes);
  const int nrows = min(32, nk - k0);
  if (parts > 1 || p.splits > 1) {
    const bool slot = parts > 1;
    const int64_t r = (slot ? (int64_t)slot_no * kPackedTile + wave * 32 : (int64_t)(split * p.kv_heads + kvh) * p.tk + kb + k0) * D;
    store_acc_rows<F16>(patch, dk, NA, p.sm_scale, kGradStoreF32, (char*)((slot ? p.part : p.sum) + r), D * 4, nrows, lane);
    store_acc_rows<F16>(patch, dv, NA, 1.0f, kGradStoreF32, (char*)((slot ? p.part2 : p.sum2) + r), D * 4, nrows, lane);
  } else {
    store_acc_rows<F16>(patch, dk, NA, p.sm_scale, kGradStore,
                        (char*)((T*)p.dk + (int64_t)kvh * p.dk_sh + (int64_t)(kb + k0) * p.dk_sn), p.dk_sn * 2, nrows, lane);
    store_acc_rows<F16>(patch, dv, NA, 1.0f, kGradStore,
                        (char*)((T*)p.dv + (int64_t)kvh * p.dv_sh + (int64_t)(kb + k0) * p.dv_sn), p.dv_sn * 2, nrows, lane);
  }
}

// dq, or dk and dv, of split tiles from their parts, in the parts' order: the workgroup of part k takes its share of the
// tile's rows, D / 4 lanes a row, kJoinRows of them at a time.
template <bool F16, int D, bool KEYS>
__device__ __forceinline__ void packed_bwd_join(const PackedParams& p) {
  using T = typename Elem<F16>::T;
  using V4 = typename Elem<F16>::V4;
  constexpr int TPR = D / 4, STEP = 256 / TPR;
  if (p.split_least == 0) return;
  const i32x4 rec = p.records[blockIdx.x];   // first row, rows, part, parts
  if (rec[3] <= 1) return;
  const int shares = p.per, hs = packed_head(packed_place(p, blockIdx.x).pos, shares), parts = rec[3];
  const int head = KEYS ? hs / p.splits : hs, d4 = (threadIdx.x % TPR) * 4;
  const int64_t slot0 = (int)blockIdx.x - rec[2] * shares;
  const int end = (rec[2] + 1) * rec[1] / parts;
  for (int r0 = rec[2] * rec[1] / parts + threadIdx.x / TPR; r0 < end; r0 += kJoinRows * STEP) {
    f32x4 a[kJoinRows], b[kJoinRows];
#pragma unroll
    for (int j = 0; j < kJoinRows; ++j) a[j] = b[j] = f32x4{};
#pragma unroll 2
    for (int i = 0; i < parts; ++i)
#pragma unroll
      for (int j = 0; j < kJoinRows; ++j) {
        const int64_t at = ((slot0 + i * shares) * kPackedTile + min(r0 + j * STEP, end - 1)) * D + d4;
        a[j] += *(const f32x4*)(p.part + at);
        if constexpr (KEYS) b[j] += *(const f32x4*)(p.part2 + at);
      }
#pragma unroll
    for (int j = 0; j < kJoinRows; ++j) {
      if (r0 + j * STEP >= end) break;
      const int64_t tok = rec[0] + r0 + j * STEP;
      if (KEYS && p.splits > 1) {   // a share's sums: packed_bwd_sum adds the shares
        const int64_t at = ((int64_t)(hs % p.splits * p.kv_heads + head) * p.tk + tok) * D + d4;
        *(f32x4*)(p.sum + at) = a[j];
        *(f32x4*)(p.sum2 + at) = b[j];
        continue;
      }
      V4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = to_elem<T>(a[j][e]);
        y[e] = to_elem<T>(b[j][e]);
      }
      if constexpr (KEYS) {
        *(V4*)((T*)p.dk + (int64_t)head * p.dk_sh + tok * p.dk_sn + d4) = x;
        *(V4*)((T*)p.dv + (int64_t)head * p.dv_sh + tok * p.dv_sn + d4) = y;
      } else {
        *(V4*)((T*)p.dq + (int64_t)head * p.dq_sh + tok * p.dq_sn + d4) = x;
      }
    }
  }
}

// All of them in one launch: a launch that finds little to add takes 4 to 5 us.
template <bool F16, int D>
__global__ __launch_bounds__(256) void packed_bwd_join_kernel(PackedParams of_k, PackedParams of_q) {
  if (blockIdx.y == 0) packed_bwd_join<F16, D, true>(of_k);
  else packed_bwd_join<F16, D, false>(of_q);
}

// dk and dv from the sums of workgroups that had some of the group's heads each, in their order; rows outside every sequence
// (they have no sums) are zeros.
template <bool F16, int D>
__global__ __launch_bounds__(256) void packed_bwd_sum_kernel(PackedParams p) {
  using T = typename Elem<F16>::T;
  using V4 = typename Elem<F16>::V4;
  constexpr int TPR = D / 4;
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)p.kv_heads * p.tk;
  const int tok = (int)(gid / TPR), c4 = (int)(gid % TPR) * 4;
  if (tok >= p.tk) return;
  const int first = p.k_off[0], last = p.k_off[p.n];
  const bool held = tok >= min(max(first, 0), p.tk) && tok < min(max(last, 0), p.tk);
  for (int kvh = blockIdx.y; kvh < p.kv_heads; kvh += (int)gridDim.y) {
    const int64_t r = (int64_t)kvh * p.tk + tok;
    f32x4 a = f32x4{}, b = f32x4{};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {   // (of a row of no sequence: whatever lies there, not used)
      const int64_t at = (s * rows + r) * D + c4;
      a += *(const f32x4*)(p.sum + at);
      b += *(const f32x4*)(p.sum2 + at);
    }
    V4 x, y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = to_elem<T>(held ? a[e] : 0.f);
      y[e] = to_elem<T>(held ? b[e] : 0.f);
    }
    *(V4*)((T*)p.dk + (int64_t)kvh * p.dk_sh + (int64_t)tok * p.dk_sn + c4) = x;
    *(V4*)((T*)p.dv + (int64_t)kvh * p.dv_sh + (int64_t)tok * p.dv_sn + c4) = y;
  }
}

// Workgroups that share a key tile, each with some of the group's heads: as many as divide the group and bring the launch to
// two rounds of the chip's slots.  Where heads are shared this comes before parts of a tile, whose queries every XCD's L2 would
// have to hold (8 heads over 2, prompts of 12000 and 4384 tokens: 651 us so, 790 in parts alone).
int packed_bwd_splits(int64_t tk, int kv_heads, int group) {
  const int64_t tiles = ((tk + kPackedTile - 1) / kPackedTile) * kv_heads;
  int splits = 1;
  while (splits < group && tiles * splits < 2 * kPackedSlots) {
    int next = splits + 1;
    while (group % next) ++next;
    splits = next;
  }
  return splits;
}

template <bool F16, int D>
static int launch_packed_bwd(PackedParams p, hipStream_t s) {
  constexpr int LDS_Q = packed_dq_lds<D>(), LDS_KV = packed_kv_lds<D>();
  static_assert(LDS_Q <= 65536 && LDS_KV <= 80 * 1024, "two workgroups a CU");
  PackedParams q = p;   // dq's launch
  q.records = p.records + kPackedParts;
  q.part = p.part_q;
  int rc = VMO_OK;
  if (p.tq > 0) {
    q.split_least = packed_splits(p.tk) ? kPackedSplit : 0;
    rc = packed_begin<false>(&q, p.tq, p.heads, s);
    if (rc != VMO_OK) return rc;
    hipLaunchKernelGGL((packed_bwd_dq_kernel<F16, D>), dim3((unsigned)(q.blocks * q.per)), dim3(64 * kPackedWaves), LDS_Q, s, q);
    rc = launch_status("packed_bwd_dq");
    if (rc != VMO_OK) return rc;
  }
  if (p.tk == 0) return VMO_OK;   // (no tile of dq's is split)
  auto kern = packed_bwd_dkdv_kernel<F16, D>;
  if (LDS_KV > 65536 &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS_KV) != hipSuccess)
    return set_error(VMO_ERR_LAUNCH, "packed_bwd: cannot raise the LDS limit to %d bytes", LDS_KV);
  p.split_least = packed_splits(p.tq) ? kPackedSplit : 0;
  rc = packed_begin<true>(&p, p.tk, p.kv_heads * p.splits, s);
  if (rc != VMO_OK) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)(p.blocks * p.per)), dim3(64 * kPackedWaves), LDS_KV, s, p);
  rc = launch_status("packed_bwd_dkdv");
  if (rc != VMO_OK) return rc;
  if (p.split_least > 0 || q.split_least > 0) {
    hipLaunchKernelGGL((packed_bwd_join_kernel<F16, D>), dim3(kPackedParts, 2), dim3(256), 0, s, p, q);
    rc = launch_status("packed_bwd_join");
  }
  if (rc != VMO_OK || p.splits == 1) return rc;
  const int64_t threads = (int64_t)p.tk * (D / 4);
  hipLaunchKernelGGL((packed_bwd_sum_kernel<F16, D>), dim3((unsigned)((threads + 255) / 256), (unsigned)min(p.kv_heads, 65535)),
                     dim3(256), 0, s, p);
  return launch_status("packed_bwd_sum");
}

int packed_bwd_launch(const PackedParams& p, bool f16, int d, hipStream_t s) {
  if (d == 64) return f16 ? launch_packed_bwd<true, 64>(p, s) : launch_packed_bwd<false, 64>(p, s);
  return f16 ? launch_packed_bwd<true, 128>(p, s) : launch_packed_bwd<false, 128>(p, s);
}

}  // namespace vmo
