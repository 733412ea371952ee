// Packed causal attention, forward: o_i = sum_j P_ij v_j, P = softmax over the keys j of row i's sequence that it sees
// (j <= i + past), grouped heads (a key / value head serves `group` query heads).
//
// The mapping is that of the flash-entropy forward: a workgroup of 4 waves takes 128 queries of one head (32 a wave),
// S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16, so that a lane owns one query; K and V tiles of 64 keys go by
// global_load_lds through a ring of LDS slots; the two 32-key blocks of a stage are software-pipelined.  What differs:
//  * a wave's keys fall into three ranges: stages that all its rows see whole (no mask), those on the diagonal (masked),
//    and those that none sees (skipped; the wave still meets the barriers and copies its share).  Half of the square is
//    never touched; the diagonal costs a 128-query tile about one stage and a half of its own.
//  * the reference point m of p = 2^(s c - m) moves only when a lane's block sum passes a limit that keeps p within the
//    16-bit type: then m becomes the row's maximum and the sums so far are scaled.  The first block sets m (it starts at
//    -3e38).  Even the test for it is left out of the steady loop: its branch behind every block kept the next block's
//    products waiting (16384 tokens, 12 heads of 128, not causal: 1054 TFLOP/s with it, 1217 without; a running maximum
//    costs 16 vector operations a block more).  The loop notes that a limit was passed, and then the workgroup runs its
//    keys again with the test; rows that pass no limit have the same bits both ways.
//  * workgroups take the heaviest tile first (packed_locate).
//  * tiles whose keys would take longer than the rest of the launch are cut into parts, whose sums packed_fwd_join adds.
// The row sums add the fp32 p; p is rounded to the 16-bit type as the operand of P V, o once at the end.
// Long prompts are bound by the matrix pipes at the chip's power (16384 tokens, 12 heads over 4 of 128: 735 us, 1.12 PFLOP/s at
// 1.55 GHz, 67% of the busy CUs' MFMA cycles), short ones by a workgroup's latency (up to 200 tokens: 8.3 us).
#include "packed.h"

namespace vmo {

// a lane's 16 weights of a block may sum to this before m moves: P stays finite in 16 bits (and in bf16 the sums in 32)
template <bool F16> constexpr float kSumMost = F16 ? 32768.f : 1099511627776.f;
constexpr float kNoMax = -3.0e38f;    // m of a row that has seen no key

template <int D> constexpr int packed_stage_bytes() { return kFwdBN * D * 2 * 2; }
template <int D> constexpr int packed_fwd_lds() {
  constexpr int ring = fwd_slots(packed_stage_bytes<D>()) * packed_stage_bytes<D>();
  constexpr int least = kPackedWaves * kEpiPatchBytes;
  return ring > least ? ring : least;
}

template <bool F16, int D>
__global__ __launch_bounds__(64 * kPackedWaves, 2) void packed_fwd_kernel(PackedParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  using V8 = typename E::V8;
  using V2 = typename E::V2;
  constexpr int RB = D * 2, K_BYTES = kFwdBN * RB, STAGE = packed_stage_bytes<D>(), NSLOT = fwd_slots(STAGE);
  constexpr int NA = D / 32, NDS = D / 16;
  constexpr int DMA_PER_TILE = STAGE / 1024 / kPackedWaves;
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  VMO_LDS char* smem = (VMO_LDS char*)smem_raw;
  auto uni = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };

  const PackedPlace place = packed_place(p, blockIdx.x);
  const int head = uni(packed_head(place.pos, p.heads));
  const PackedTile w = packed_tile<false>(p, place.idx);
  const int slot_no = w.number * p.per + place.pos;
  packed_record<false>(p, w, slot_no);
  if (w.tile < 0) {
    if (p.zero_rest)
      packed_zero_rest<T, D>((T*)p.out + head * p.o_sh, p.o_sn, p.q_off, p.n, p.tq, w.which, w.spare);
    return;
  }
  const int nq = uni(w.s.nq), nk = uni(w.s.nk), qb = uni(w.s.qb), kb = uni(w.s.kb);
  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int q0 = uni(w.tile) * kPackedTile + wave * 32;   // the wave's first row of the sequence
  const bool live = q0 < nq;
  // keys that row i sees: the first sees(i) of the sequence
  const int past = nk - nq;
  auto keys_of = [&](int row) __attribute__((always_inline)) { return p.causal ? min(max(past + row + 1, 0), nk) : nk; };
  const int row = min(q0 + l32, nq - 1);
  const int lim = keys_of(row);
  const int lo = uni(keys_of(min(q0, nq - 1))), hi = uni(keys_of(min(q0 + 31, nq - 1)));   // least and most of the wave
  // the part's stages: n_tiles from `begin` on
  const int stages = uni((keys_of(min(uni(w.tile) * kPackedTile + kPackedTile - 1, nq - 1)) + kFwdBN - 1) / kFwdBN);
  const int parts = uni(w.parts), begin = uni((int)((int64_t)w.part * stages / parts));
  const int n_tiles = uni((int)((int64_t)(w.part + 1) * stages / parts)) - begin;

  const T* kbase = (const T*)p.k + (int64_t)(head / p.group) * p.k_sh + (int64_t)kb * p.k_sn;
  const T* vbase = (const T*)p.v + (int64_t)(head / p.group) * p.v_sh + (int64_t)kb * p.v_sn;
  const TileCopy<T, D, kPackedWaves> kcopy(kbase, p.k_sn, wave, lane), vcopy(vbase, p.v_sn, wave, lane);
  auto issue = [&](int t) __attribute__((always_inline)) {
    uint32_t sb = (uint32_t)(uintptr_t)smem;
    asm volatile("" : "+s"(sb));
    const uint32_t st = sb + (uint32_t)((t % NSLOT) * STAGE);
    kcopy.issue((begin + t) * kFwdBN, nk, st);   // (a tile that runs past the sequence repeats its last key: masked)
    vcopy.issue((begin + t) * kFwdBN, nk, st + K_BYTES);
  };

  auto prime = [&]() __attribute__((always_inline)) {
    issue(0);
    if (NSLOT == 3 && n_tiles > 1) issue(1);
  };
  if (n_tiles > 0) prime();   // the first copies are under way while the queries come
  V8 qf[NDS];   // Q^T as the B operand: lane (query l32, half hl) holds features 16 ds + 8 hl + 0..7
  {
    const T* qp = (const T*)p.q + (int64_t)head * p.q_sh + (int64_t)(qb + row) * p.q_sn + hl * 8;
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      qf[ds] = *(const V8*)(qp + ds * 16);
      asm volatile("" : "+v"(qf[ds]));
    }
  }

  const float c = p.c;
  float m_run = kNoMax, l_run = 0.f;
  bool passed = false;   // some untested block's sum was over the limit
  f32x16 acc[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) acc[a] = f32x16{};
  const int srow_sw = swz_rows<RB>(l32);
  const int trow = 4 * hl + ((lane & 15) >> 2);
  const int tchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int tbyte = (lane & 1) * 8;

  // S^T of 32 keys; with `pin` the operand reads run two ahead of the MFMAs
  auto qk_block = [&](const VMO_LDS char* Ks, int kb2, f32x16& x, auto pin) __attribute__((always_inline)) {
    const VMO_LDS char* arow = Ks + (32 * kb2 + l32) * RB;
    V8 a[NDS];
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) a[ds] = lds_read8<V8>(arow + ((2 * ds + hl) ^ srow_sw) * 16);
    x = f32x16{};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) x = E::mfma(a[ds], qf[ds], x);
    if constexpr (decltype(pin)::value) {
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
      for (int ds = 0; ds < NDS - 2; ++ds) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    }
  };
  // p = 2^(s c - m) of one block, packed as two B operands, added to the row sum.  nvis: the block's keys below it are
  // seen (MASKED); m moves in tested blocks only.
  auto softmax_block = [&](const f32x16& s, V8 (&P)[2], int nvis, auto masked, auto tested) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked)::value;
    auto seen = [&](int r) __attribute__((always_inline)) { return 8 * (r >> 2) + 4 * hl + (r & 3) < nvis; };
    auto weights = [&]() __attribute__((always_inline)) {
      float ls0 = 0.f, ls1 = 0.f;
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      uint32_t w8[8];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float x0 = fmaf(s[r], c, -m_run), x1 = fmaf(s[r + 1], c, -m_run);
        if constexpr (MASKED) {
          x0 = seen(r) ? x0 : kMaskLogit;
          x1 = seen(r + 1) ? x1 : kMaskLogit;
        }
        const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
        w8[r / 2] = __builtin_bit_cast(uint32_t, E::pack2(p0, p1));
        if (r == 0) ls0 = p0 + p1;
        else if (r == 2) ls1 = p0 + p1;
        else if (r & 2) ls1 += p0 + p1;
        else ls0 += p0 + p1;
      }
      P[0] = __builtin_bit_cast(V8, u32x4{w8[0], w8[1], w8[2], w8[3]});
      P[1] = __builtin_bit_cast(V8, u32x4{w8[4], w8[5], w8[6], w8[7]});
      return ls0 + ls1;
    };
    float ls = weights();
    const bool over = !(ls <= kSumMost<F16>);
    if constexpr (!decltype(tested)::value) {
      passed |= over;
    } else if (__builtin_amdgcn_ballot_w64(over) != 0) {
      // m moves to the row's maximum so far, in the rows that need it (either half of a row's lanes): a row's bits do not
      // depend on its neighbours
      const auto either = __builtin_amdgcn_permlane32_swap(over, over, false, false);
      float mx = kNoMax;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, !MASKED || seen(r) ? s[r] * c : kNoMax);
      const float m_new = either[0] | either[1] ? fmaxf(m_run, wave_max32(mx)) : m_run;
      const float f = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= f;
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[a][r] *= f;
      ls = weights();
    }
    l_run += ls;
  };
  // O^T += V^T P^T of one block
  auto pv_block = [&](const VMO_LDS char* Vs, int kb2, const V8 (&P)[2], auto pin) __attribute__((always_inline)) {
    V8 wt[2 * NA];
    const int tsw = swz_rows<RB>(trow);
#pragma unroll
    for (int a = 0; a < NA; ++a) {
      const int c0 = trow * RB + (((4 * a + tchunk) ^ tsw) * 16 + tbyte);
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const VMO_LDS char* rp = Vs + (32 * kb2 + 16 * h2) * RB;
        wt[2 * a + h2] = lds_read_tr8<V8>(rp + c0, rp + 8 * RB + (c0 ^ 32));
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * NA; ++i) acc[i / 2] = E::mfma(wt[i], P[i % 2], acc[i / 2]);
    if constexpr (decltype(pin)::value) {
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < 2 * NA - 2; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
    }
  };
  // a stage that every row of the wave sees whole: S of block 1 beside the softmax of block 0, P V of block 0 beside the
  // softmax of block 1
  auto full_stage = [&](const VMO_LDS char* Ks, auto tested) __attribute__((always_inline)) {
    f32x16 s0, s1;
    V8 P0[2], P1[2];
    qk_block(Ks, 0, s0, std::true_type{});
    __builtin_amdgcn_sched_barrier(0);
    qk_block(Ks, 1, s1, std::false_type{});
    softmax_block(s0, P0, 0, std::false_type{}, tested);
    __builtin_amdgcn_sched_barrier(0);
    pv_block(Ks + K_BYTES, 0, P0, std::false_type{});
    softmax_block(s1, P1, 0, std::false_type{}, tested);
    __builtin_amdgcn_sched_barrier(0);
    pv_block(Ks + K_BYTES, 1, P1, std::true_type{});
  };
  // a stage on the diagonal, or at the end: both blocks' S first
  auto masked_stage = [&](const VMO_LDS char* Ks, int key0) __attribute__((always_inline)) {
    f32x16 s[2];
    const bool two = key0 + 32 < hi;
    qk_block(Ks, 0, s[0], std::false_type{});
    if (two) qk_block(Ks, 1, s[1], std::false_type{});
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2) {
      if (kb2 == 1 && !two) break;
      V8 P[2];
      const int nvis = lim - key0 - 32 * kb2;
      softmax_block(s[kb2], P, nvis, std::true_type{}, std::true_type{});
      masked_product<F16, RB, NA>(acc, Ks + K_BYTES + 32 * kb2 * RB, P, lane, [&](int key) { return key < nvis; });
    }
  };

  // Tile t sits in ring slot t % NSLOT; at its top this wave's copies of it have landed (only those of tile t + 1 may be
  // under way), after the barrier every wave's have, and the slot of tile t - 1 is free for tile t + NSLOT - 1.
  constexpr int kSteadyPending = NSLOT == 3 ? DMA_PER_TILE : 0;
  const int n_full = live ? uni(min(max(lo / kFwdBN - begin, 0), n_tiles)) : 0;
  auto top = [&](int t) __attribute__((always_inline)) {
    if (NSLOT == 3 && t + 1 < n_tiles) tile_sync<kSteadyPending>();
    else tile_sync<0>();
    if (t + NSLOT - 1 < n_tiles) issue(t + NSLOT - 1);
  };
  auto slot = [&](int t) __attribute__((always_inline)) { return (const VMO_LDS char*)smem + (t % NSLOT) * STAGE; };
  // stages that some wave of the workgroup runs untested (the last wave's rows see most)
  const int untested = uni(max(keys_of(min(uni(w.tile) * kPackedTile + kPackedTile - 32, nq - 1)) / kFwdBN - begin - 1, 0));
  for (bool again = false; n_tiles > 0; again = true) {
    if (again) prime();
    int t = 0;
    const int tested = again ? n_full : min(1, n_full);   // the first stage sets m
    for (; t < tested; ++t) {
      top(t);
      full_stage(slot(t), std::true_type{});
    }
    for (; t + NSLOT <= n_full; t += NSLOT)   // (t = 1, 1 + NSLOT, ..: slots at compile-time offsets)
      static_for<0, NSLOT>([&](auto i) __attribute__((always_inline)) {
        top(t + decltype(i)::value);
        full_stage((const VMO_LDS char*)smem + ((1 + decltype(i)::value) % NSLOT) * STAGE, std::false_type{});
      });
    for (; t < n_full; ++t) {
      top(t);
      full_stage(slot(t), std::false_type{});
    }
    for (; t < n_tiles; ++t) {
      top(t);
      const int key0 = (begin + t) * kFwdBN;
      if (live && key0 < hi) masked_stage(slot(t), key0);
    }
    __syncthreads();   // the ring is free
    if (again || untested == 0) break;
    // whether any row of the workgroup passed the limit untested: a word a wave in the ring
    VMO_LDS int* words = (VMO_LDS int*)smem;
    const bool mine = __builtin_amdgcn_ballot_w64(passed) != 0;
    if (lane == 0) words[wave] = mine;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int i = 0; i < kPackedWaves; ++i) any |= words[i];
    __syncthreads();
    if (!any) break;
    m_run = kNoMax;
    l_run = 0.f;
#pragma unroll
    for (int a = 0; a < NA; ++a) acc[a] = f32x16{};
  }
  if (!live) return;
  const float l_tot = wave_sum32(l_run);
  const int nrows = min(32, nq - q0);
  VMO_LDS float* patch = (VMO_LDS float*)(smem + wave * kEpiPatchBytes);
  if (parts > 1) {
    const int64_t at = (int64_t)slot_no * kPackedTile + wave * 32;
    store_acc_rows<F16>(patch, acc, NA, 1.f, kGradStoreF32, (char*)(p.part + at * D), D * 4, nrows, lane);
    if (hl == 0 && l32 < nrows) {
      p.part2[2 * (at + l32)] = m_run;
      p.part2[2 * (at + l32) + 1] = l_tot;
    }
    return;
  }
  const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;   // (a row that sees no key)
  T* out = (T*)p.out + (int64_t)head * p.o_sh + (int64_t)(qb + q0) * p.o_sn;
  store_acc_rows<F16>(patch, acc, NA, inv, kGradStore, (char*)out, p.o_sn * 2, nrows, lane);
  if (p.o_low) {
#pragma unroll
    for (int a = 0; a < NA; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = acc[a][r] * inv;
        acc[a][r] = x - (float)to_elem<T>(x);
      }
    T* low = (T*)p.o_low + (int64_t)head * p.o_sh + (int64_t)(qb + q0) * p.o_sn;
    store_acc_rows<F16>(patch, acc, NA, 1.f, kGradStore, (char*)low, p.o_sn * 2, nrows, lane);
  }
  if (p.lse && hl == 0 && l32 < nrows)
    p.lse[(int64_t)head * p.st_sh + qb + q0 + l32] = l_tot == 0.f ? 0.f : m_run + fast_log2(l_tot);
}

// o (and lse) of split tiles from their parts: the workgroup of part k takes its share of the tile's rows, D / 4 lanes a row,
// kJoinRows of them at a time, whose loads are under way together.
template <bool F16, int D>
__global__ __launch_bounds__(256) void packed_fwd_join_kernel(PackedParams p) {
  using T = typename Elem<F16>::T;
  constexpr int TPR = D / 4, STEP = 256 / TPR;
  const i32x4 rec = p.records[blockIdx.x];   // first row, rows, part, parts
  if (rec[3] <= 1) return;
  const int head = packed_head(packed_place(p, blockIdx.x).pos, p.heads), d4 = (threadIdx.x % TPR) * 4, parts = rec[3];
  const int slot0 = (int)blockIdx.x - rec[2] * p.heads;
  const int end = (rec[2] + 1) * rec[1] / parts;
  for (int r0 = rec[2] * rec[1] / parts + threadIdx.x / TPR; r0 < end; r0 += kJoinRows * STEP) {
    float m[kJoinRows], l[kJoinRows];
    f32x4 acc[kJoinRows];
#pragma unroll
    for (int j = 0; j < kJoinRows; ++j) {
      m[j] = kNoMax;
      l[j] = 0.f;
      acc[j] = f32x4{};
    }
#pragma unroll 2
    for (int i = 0; i < parts; ++i)
#pragma unroll
      for (int j = 0; j < kJoinRows; ++j) {
        const int64_t at = (int64_t)(slot0 + i * p.heads) * kPackedTile + min(r0 + j * STEP, end - 1);
        const float pm = p.part2[2 * at], pl = p.part2[2 * at + 1];
        const f32x4 y = *(const f32x4*)(p.part + at * D + d4);
        const float m_new = fmaxf(m[j], pm), f = fast_exp2(m[j] - m_new), pf = fast_exp2(pm - m_new);
        m[j] = m_new;
        l[j] = fmaf(l[j], f, pl * pf);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(acc[j][e], f, y[e] * pf);
      }
#pragma unroll
    for (int j = 0; j < kJoinRows; ++j) {
      const int r = r0 + j * STEP;
      if (r >= end) break;
      const float inv = l[j] == 0.f ? 0.f : 1.0f / l[j];
      typename Elem<F16>::V4 y, low;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = acc[j][e] * inv;
        y[e] = to_elem<T>(x);
        low[e] = to_elem<T>(x - (float)y[e]);
      }
      const int64_t tok = rec[0] + r, at = (int64_t)head * p.o_sh + tok * p.o_sn + d4;
      *(typename Elem<F16>::V4*)((T*)p.out + at) = y;
      if (p.o_low) *(typename Elem<F16>::V4*)((T*)p.o_low + at) = low;
      if (p.lse && d4 == 0) p.lse[(int64_t)head * p.st_sh + tok] = l[j] == 0.f ? 0.f : m[j] + fast_log2(l[j]);
    }
  }
}

template <bool F16, int D>
static int launch_packed_fwd(PackedParams p, hipStream_t s) {
  constexpr int LDS = packed_fwd_lds<D>();
  static_assert(LDS <= 65536, "LDS within the default limit");
  int rc = packed_begin<false>(&p, p.tq, p.heads, s);
  if (rc != VMO_OK) return rc;
  hipLaunchKernelGGL((packed_fwd_kernel<F16, D>), dim3((unsigned)(p.blocks * p.per)), dim3(64 * kPackedWaves), LDS, s, p);
  rc = launch_status("packed_fwd");
  if (rc != VMO_OK || p.split_least == 0) return rc;
  hipLaunchKernelGGL((packed_fwd_join_kernel<F16, D>), dim3(kPackedParts), dim3(256), 0, s, p);
  return launch_status("packed_fwd_join");
}

int packed_fwd_launch(const PackedParams& p, bool f16, int d, hipStream_t s) {
  if (d == 64) return f16 ? launch_packed_fwd<true, 64>(p, s) : launch_packed_fwd<false, 64>(p, s);
  return f16 ? launch_packed_fwd<true, 128>(p, s) : launch_packed_fwd<false, 128>(p, s);
}

}  // namespace vmo
