// Packed causal attention: launch parameters, the order of its workgroups and what a masked block's products take, shared
// by the forward (packed_fwd.hip) and the backward (packed_bwd.hip).
//
// Sequence s holds query rows [q_off[s], q_off[s + 1]) and keys [k_off[s], k_off[s + 1]) of the packed tensors.  With
// past = nk - nq, its row i sees the keys j <= i + past (causal), or all of them.  The offsets are read on the GPU, so a
// captured graph replays with others; they are cut to the tensors, so none reaches outside.
#pragma once

#include "fea_fwd.h"

namespace vmo {

constexpr int kPackedMaxSeqs = 2048;   // a call's sequences: they wait in LDS while a workgroup finds its tile
constexpr int kPackedTile = 128;       // queries of a forward / dq workgroup, keys of a dk / dv one
constexpr int kPackedWaves = 4;

struct PackedParams {
  const void *q, *k, *v, *o, *dO;
  void *out, *dq, *dk, *dv;
  void* o_low;                             // o's rounding error in 16 bits, laid out as o (or null): delta is of the unrounded o
  int64_t q_sh, q_sn, k_sh, k_sn, v_sh, v_sn, o_sh, o_sn, do_sh, do_sn;
  int64_t dq_sh, dq_sn, dk_sh, dk_sn, dv_sh, dv_sn;
  const int32_t *q_off, *k_off;
  int n, tq, tk, heads, kv_heads, group;   // group = heads / kv_heads
  int causal, zero_rest;                   // zero_rest: rows outside every sequence are written as zeros
  float* lse;                              // (heads, tq), log2 units, rows of st_sh
  int64_t st_sh;
  float* neg_delta;                        // (heads, tq): -rowsum(o dO), from the dq kernel to the dk / dv one
  float *part, *part2;                     // parts of split tiles: (slots, 128, D) fp32 sums; the forward's m and l (.., 2), or dv's
  float *sum, *sum2;                       // splits > 1: dk's and dv's (splits, kv_heads, tk, D) fp32
  i32x4* records;                          // of the first kPackedParts workgroups: first row, rows, part and parts of its tile
  i32x4* plan;                             // two of each `idx` (packed_plan): its tile; null: the workgroups find theirs
  int blocks, per;                         // a launch's workgroups: `blocks` times the `per` of one tile
  uint32_t per_rcp;                        // (2^32 - 1) / per
  int splits;                              // dk / dv: workgroups that share a key tile, each with group / splits of the heads
  int split_least;                         // tiles of up to so many units are never split (0: no tile is)
  float c, sm_scale;                       // c = sm_scale log2 e
  int half;                                // kPackedSlots / 2 / per
  float* part_q;                           // the backward's launch: dq's parts (part, part2: dk's and dv's)
};

// ---- integer sums over a wave (DPP: row shifts, then the rows' last lanes broadcast) --------------------------------
__device__ __forceinline__ int wave_scan_i32(int v) {   // inclusive prefix sum over the lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}
__device__ __forceinline__ int wave_max_i32(int v) {   // of values >= 0
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_sum_i32(int v) { return __builtin_amdgcn_readlane(wave_scan_i32(v), 63); }

// ---- which tile a workgroup takes ------------------------------------------------------------------------------------
struct PackedSeq { int qb, nq, kb, nk; };

__device__ __forceinline__ PackedSeq packed_seq(const PackedParams& p, int s) {
  PackedSeq r;
  r.qb = min(max(p.q_off[s], 0), p.tq);
  r.nq = min(max(p.q_off[s + 1], r.qb), p.tq) - r.qb;
  r.kb = min(max(p.k_off[s], 0), p.tk);
  r.nk = min(max(p.k_off[s + 1], r.kb), p.tk) - r.kb;
  return r;
}

// Tiles of a sequence in the order u = 0, 1, .. of falling work: u's work, in tiles of the other side, is
// max(0, min(cap, top - u)).  Query tiles: a causal row's keys grow with it, so u counts from the last tile; key tiles: a
// key's queries fall with it.
struct PackedTiles { int tiles, top, cap; };
template <bool KEYS>
__device__ __forceinline__ PackedTiles packed_tiles(const PackedParams& p, const PackedSeq& s) {
  constexpr int T = kPackedTile, kMany = 1 << 28;
  const int qt = (s.nq + T - 1) / T, kt = (s.nk + T - 1) / T;
  if constexpr (KEYS) return PackedTiles{kt, p.causal ? kt : kMany, qt};
  return PackedTiles{qt, p.causal ? kt : kMany, kt};
}
// how many of a sequence's tiles have at least the work `level`
__device__ __forceinline__ int packed_count(const PackedTiles& t, int level) {
  if (level <= 0) return t.tiles;
  return level <= t.cap ? min(max(t.top - level + 1, 0), t.tiles) : 0;
}

// Heavy tiles are split: one long prompt's last tile sees all its keys, and alone can take longer than the whole launch's mean
// work.  S is 1.75 times the mean of the chip's kPackedSlots workgroups -- one that has its CU alone runs about that much
// faster than two that share it, so up to S a tile is no later than the rest --, or 6 above 1.25 times the mean where that is
// less (long prompts, beside whose stages a part's own cost is small), and `split_least` at least; where the heaviest tile has
// 1.25 S, those of L > S units are cut into ceil(L / S) parts of equal length.  One prompt of 16384 tokens, 2 heads of 128
// over one: 248 -> 153 us; of 8192, 4 heads: 129 -> 87; 4 prompts of 20 to 5000, 4 heads: 85 -> 51.  Training steps of the
// first two: 658 -> 632 and 374 -> 370 us against 1.75 times the mean everywhere; 1.25 times everywhere cost short batches (12
// prompts of 40 to 3900 keys, 12 heads: 75 -> 84 us).  Eight waves of two key groups instead, which halve every tile's time,
// did less (176 and 99 -> 218 and 116).  Parts and whole tiles stand in one order, by their work, so the launch's last round
// is made of light ones; as no part has less than half of S, all parts are among the first 2 kPackedSlots / 1.25 workgroups.
// A part's fp32 sums go to slot = its number in that order times per + pos; a second kernel adds them.
constexpr int kPackedSlots = 512;
constexpr int kPackedParts = 2 * kPackedSlots + 128;
constexpr int kJoinRows = 4;   // rows that a lane of an adding kernel has under way
struct PackedSplit {
  int S, most;   // units a part has at most; parts a tile has at most
  __device__ __forceinline__ int parts(int L) const { return L > S ? (L + S - 1) / S : 1; }
  // a sequence's tiles of P parts with more than x units each
  __device__ __forceinline__ int above(const PackedTiles& t, int P, int x) const {
    return x < S ? packed_count(t, max((P - 1) * S, P * x) + 1) - packed_count(t, P * S + 1) : 0;
  }
  // parts of a sequence's tiles that have at least the work `level`
  __device__ __forceinline__ int count(const PackedTiles& t, int level) const {
    if (most == 1) return packed_count(t, level);
    int c = 0;
    for (int P = 1; P <= most; ++P) c += P * above(t, P, max(level, 1) - 1);
    if (level <= 0) c += t.tiles - packed_count(t, 1);   // tiles without work
    return c;
  }
};
// the work of a sequence's tiles
__device__ __forceinline__ float packed_work(const PackedTiles& t) {
  const int n_cap = min(max(t.top - t.cap + 1, 0), t.tiles);
  const int most = min(t.cap - 1, t.top), least = max(t.top - t.tiles + 1, 1);
  const float m = (float)most, l = (float)least;
  return (float)n_cap * (float)t.cap + (most >= least ? 0.5f * (m + l) * (m - l + 1.f) : 0.f);
}

struct PackedTile {
  PackedSeq s;
  int tile;           // of the sequence; below 0: none
  int part, parts;
  int number;         // of the part, heaviest first
  int which, spare;   // of no tile: the spare workgroup's number, and how many there are
};
constexpr int kPackedSeqBytes = 16;   // LDS of a sequence while a wave finds its tile
constexpr int kPackedFew = 64;        // up to so many sequences a workgroup finds its own tile: one a lane

// Workgroup x is the pos-th of the `per` of part idx.
struct PackedPlace { int idx, pos; };
__device__ __forceinline__ PackedPlace packed_place(const PackedParams& p, uint32_t x) {
  uint32_t q = __umulhi(x, p.per_rcp), r = x - q * (uint32_t)p.per;   // (q or one less than it)
  if (r >= (uint32_t)p.per) {
    ++q;
    r -= p.per;
  }
  return PackedPlace{(int)q, (int)r};
}

// The part that the idx-th workgroups take.  The first `half` go to CUs of their own, the next ones beside them, in the same
// order: so of the first 2 half, where all CUs have two, the second half is taken from its end, the lightest beside the
// heaviest; where there are fewer parts than that, the CUs with two have the lightest.  (Training steps of one prompt of 16384
// tokens, 2 heads of 128: 662 -> 632 us; of 8192, 4 heads: 385 -> 370; 12 prompts of 40 to 2900, 12 heads, in three rounds:
// 68.5 -> 69.1.)
__device__ __forceinline__ int packed_turn(int idx, int busy, int half) {
  const int n = min(busy, 2 * half), two = n - half;
  if (two <= 0 || idx >= n) return idx;
  if (idx >= half) return n - 1 - (idx - half);
  return idx < two ? idx + half - two : idx - two;
}

// The part in turn idx over all sequences' tiles, heaviest tiles first (a tile's time is its keys, or queries: with the heavy ones
// first the chip's last round is made of light ones); p.per workgroups take each.  The largest level whose parts and those
// above are more than idx is found by bisection over per-sequence counts, from rows and keys that lie in LDS (free again
// after the call) if MANY, in the lanes else; a level holds the sequences in order.  Every wave of a workgroup calls it.
template <bool KEYS, bool MANY>
__device__ __forceinline__ PackedTile packed_locate(const PackedParams& p, int idx, VMO_LDS int* lds) {
  const int lane = threadIdx.x & 63;
  if constexpr (MANY) {
    for (int s = threadIdx.x; s < p.n; s += (int)blockDim.x) {
      const PackedSeq q = packed_seq(p, s);
      *(VMO_LDS i32x4*)(lds + 4 * s) = i32x4{q.qb, q.nq, q.kb, q.nk};
    }
    __syncthreads();
  }
  auto seq = [&](int s) __attribute__((always_inline)) {
    const i32x4 x = *(const VMO_LDS i32x4*)(lds + 4 * s);
    return PackedSeq{x[0], x[1], x[2], x[3]};
  };
  PackedSeq mine{0, 0, 0, 0};
  if (lane < p.n) mine = MANY ? seq(lane) : packed_seq(p, lane);
  const PackedTiles first = packed_tiles<KEYS>(p, mine);
  int best = first.tiles > 0 ? min(first.top, first.cap) : 0;
  float work = packed_work(first);
  if constexpr (MANY)
    for (int s = lane + 64; s < p.n; s += 64) {
      const PackedTiles t = packed_tiles<KEYS>(p, seq(s));
      best = max(best, t.tiles > 0 ? min(t.top, t.cap) : 0);
      work += packed_work(t);
    }
  best = wave_max_i32(best);
  PackedSplit split{max(best, 1), 1};
  if (p.split_least > 0 && 4 * best >= 5 * p.split_least) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) work += __shfl_xor(work, m);
    const float mean = work * (float)p.per * (1.001f / kPackedSlots);
    const int S = max(__builtin_amdgcn_readfirstlane((int)ceilf(fminf(fminf(1.75f * mean, 1.25f * mean + 6.f), 1.0e9f))), p.split_least);
    if (4 * best >= 5 * S) split = PackedSplit{S, (best + S - 1) / S};
  }
  auto total = [&](int level) __attribute__((always_inline)) {
    int c = split.count(first, level);
    if constexpr (MANY)
      for (int s = lane + 64; s < p.n; s += 64) c += split.count(packed_tiles<KEYS>(p, seq(s)), level);
    return wave_sum_i32(c);
  };
  PackedTile r;
  r.s = PackedSeq{0, 0, 0, 0};
  r.tile = -1;
  r.part = 0;
  r.parts = 1;
  r.number = idx;
  r.which = 0;
  r.spare = 1;
  int lo = 1, above = 0;   // the level, and the parts above it
  const int busy = total(1);
  r.number = idx = packed_turn(idx, busy, p.half);
  bool found = idx < busy;
  if (found) {
    int hi = min(split.S, best) + 1;   // total(lo) > idx >= total(hi) = above
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, t = total(mid);
      if (t > idx) lo = mid;
      else hi = mid, above = t;
    }
  } else {   // tiles without work, then none
    const int all = total(0);
    lo = 0;
    above = busy;
    found = idx < all;
    r.which = idx - all;
    r.spare = p.blocks - all;
  }
  if (found) {
    int left = idx - above;
    for (int s0 = 0; s0 < (MANY ? p.n : 1); s0 += 64) {
      const PackedSeq q = !MANY || s0 == 0 ? mine : s0 + lane < p.n ? seq(s0 + lane) : PackedSeq{0, 0, 0, 0};
      const PackedTiles t = packed_tiles<KEYS>(p, q);
      const int here = split.count(t, lo) - split.count(t, lo + 1);
      const int upto = wave_scan_i32(here), sum = __builtin_amdgcn_readlane(upto, 63);
      if (left < sum) {
        const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > left));
        left -= __builtin_amdgcn_readlane(upto, who) - __builtin_amdgcn_readlane(here, who);
        r.s = PackedSeq{__builtin_amdgcn_readlane(q.qb, who), __builtin_amdgcn_readlane(q.nq, who),
                        __builtin_amdgcn_readlane(q.kb, who), __builtin_amdgcn_readlane(q.nk, who)};
        const PackedTiles it = packed_tiles<KEYS>(p, r.s);
        int u = packed_count(it, lo + 1) + left;   // of one part
        if (split.most > 1 && lo > 0) {
          int P = 1;
          for (; P < split.most; ++P) {
            const int of_p = P * (split.above(it, P, lo - 1) - split.above(it, P, lo));
            if (left < of_p) break;
            left -= of_p;
          }
          u = packed_count(it, min(P * split.S, P * lo) + 1) + left / P;
          r.parts = P;
          r.part = left % P;
        }
        r.tile = KEYS || !p.causal ? u : it.tiles - 1 - u;
        break;
      }
      left -= sum;
    }
  }
  if constexpr (MANY) __syncthreads();   // every wave has read the sequences
  return r;
}

// More than kPackedFew sequences: a launch of its own first, a wave an idx, which leaves each one's tile in the workspace.
// (Each workgroup looking through all of them for itself: 65 sequences of 100 tokens, 64 heads of 64, 97 us against 64 so; 2048
// of them, 4 heads: 722 against 135.  With few sequences the search, 1.1 us, is shorter than a launch.)
template <bool KEYS>
__global__ __launch_bounds__(64 * kPackedWaves) void packed_plan_kernel(PackedParams p) {
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  const int idx = __builtin_amdgcn_readfirstlane((int)blockIdx.x * kPackedWaves + (int)(threadIdx.x >> 6));
  const PackedTile w = packed_locate<KEYS, true>(p, idx, (VMO_LDS int*)(VMO_LDS char*)smem_raw);
  if (idx < p.blocks && (threadIdx.x & 63) == 0) {
    p.plan[2 * idx] = i32x4{w.s.qb, w.s.nq, w.s.kb, w.s.nk};
    p.plan[2 * idx + 1] = w.tile < 0 ? i32x4{-1, w.which, w.spare, w.number} : i32x4{w.tile, w.part, w.parts, w.number};
  }
}
// this workgroup's tile
template <bool KEYS>
__device__ __forceinline__ PackedTile packed_tile(const PackedParams& p, int idx) {
  if (!p.plan) return packed_locate<KEYS, false>(p, idx, nullptr);
  typedef const __attribute__((address_space(4))) i32x4* scalar_rows;
  const scalar_rows plan = (scalar_rows)(uintptr_t)p.plan;
  const i32x4 s = plan[2 * idx], t = plan[2 * idx + 1];
  PackedTile r;
  r.s = PackedSeq{s[0], s[1], s[2], s[3]};
  r.tile = t[0];
  r.part = t[0] < 0 ? 0 : t[1];
  r.parts = t[0] < 0 ? 1 : t[2];
  r.number = t[3];
  r.which = t[1];
  r.spare = t[2];
  return r;
}

// What the adding kernel has to know of this workgroup's tile (rows of the side that the tile is of).
template <bool KEYS>
__device__ __forceinline__ void packed_record(const PackedParams& p, const PackedTile& w, int slot) {
  if (p.split_least > 0 && slot < kPackedParts && threadIdx.x == 0) {
    const int first = w.tile * kPackedTile, rows = min(kPackedTile, (KEYS ? w.s.nk : w.s.nq) - first);
    p.records[slot] = i32x4{(KEYS ? w.s.kb : w.s.qb) + first, rows, w.part, w.tile < 0 ? 1 : w.parts};
  }
}

// Zeros for the rows outside every sequence, 128-row pieces dealt to the spare workgroups (there is one at least
// whenever there is such a row: packed_grid).
template <class T, int D>
__device__ __forceinline__ void packed_zero_rest(T* rows, int64_t sn, const int32_t* off, int n, int total, int which,
                                                 int spare) {
  static_assert(sizeof(T) == 2, "16-bit rows");
  constexpr int CH = D / 8;
  const int first = min(max(off[0], 0), total), last = min(max(off[n], 0), total);
  for (int r0 = max(which, 0) * kPackedTile; r0 < total; r0 += max(spare, 1) * kPackedTile)
    for (int i = threadIdx.x; i < kPackedTile * CH; i += (int)blockDim.x) {
      const int r = r0 + i / CH;
      if (r < total && (r < first || r >= last)) *(uint4*)((char*)(rows + r * sn) + (i % CH) * 16) = uint4{0, 0, 0, 0};
    }
}

// ---- products over a block with masked rows ---------------------------------------------------------------------------
template <bool F16> constexpr uint32_t kInfBits = F16 ? 0x7c00u : 0x7f80u;   // from here on: an infinity or a NaN

// acc[a] += W^T P for 32 rows W of an LDS tile (RB-byte rows, swizzled) and the packed weights P of the accumulator layout
// (element e of P[h]: row 16 h + 8 (e / 4) + 4 hl + e % 4 of the lane's column).  Rows that the lane's column does not see
// have weight 0, but 0 times an infinity or NaN is a NaN: where a wave's operands hold such values they are taken as 0,
// and a second pass adds them to the columns that do see their row.  STEP accumulator blocks are tested at a time: all of
// them where the registers hold their operands (one branch), else one.
template <bool F16, int RB, int STEP, int NA, class Sees>
__device__ __forceinline__ void masked_product(f32x16 (&acc)[NA], const VMO_LDS char* W, const typename Elem<F16>::V8 (&P)[2],
                                               int lane, Sees sees) {
  using E = Elem<F16>;
  using T = typename E::T;
  using V8 = typename E::V8;
  using V4 = typename E::V4;
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
  const int hl = lane >> 5;
  const int trow = 4 * hl + ((lane & 15) >> 2), tchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), tbyte = (lane & 1) * 8;
  bool odd = false;
#pragma unroll
  for (int a0 = 0; a0 < NA; a0 += STEP) {
    V8 w[2 * STEP];
    u16x2 big = {0, 0};
#pragma unroll
    for (int i = 0; i < 2 * STEP; ++i) {
      const int c0 = trow * RB + (((4 * (a0 + i / 2) + tchunk) ^ swz_rows<RB>(trow)) * 16 + tbyte);
      const VMO_LDS char* rp = W + 16 * (i % 2) * RB;
      w[i] = lds_read_tr8<V8>(rp + c0, rp + 8 * RB + (c0 ^ 32));
    }
#pragma unroll
    for (int i = 0; i < 2 * STEP; ++i) {
      const u32x4 bits = __builtin_bit_cast(u32x4, w[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, bits[j] & 0x7fff7fffu));
    }
    if (__builtin_amdgcn_ballot_w64(max((uint32_t)big[0], (uint32_t)big[1]) >= kInfBits<F16>) != 0) {
      odd = true;
#pragma unroll
      for (int i = 0; i < 2 * STEP; ++i) {
        u16x8 b = __builtin_bit_cast(u16x8, w[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = (b[e] & 0x7fff) >= kInfBits<F16> ? 0 : b[e];
        w[i] = __builtin_bit_cast(V8, b);
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * STEP; ++i) acc[a0 + i / 2] = E::mfma(w[i], P[i % 2], acc[a0 + i / 2]);
  }
  if (odd) {
#pragma unroll 1
    for (int row = 0; row < 32; ++row) {
      // the weight of `row`: register 4 (row / 8) + row % 4 of the half (row / 4) % 2
      float x = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) x = r == 4 * (row >> 3) + (row & 3) ? (float)P[r >> 3][r & 7] : x;
      const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      x = __uint_as_float((row >> 2) & 1 ? both[1] : both[0]);
      const bool seen = sees(row);
      const VMO_LDS char* wr = W + row * RB + 8 * hl;
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int g = 0; g < 4; ++g) {   // features 32 a + 8 g + 4 hl .. + 3
          const u16x4 b = *(const VMO_LDS u16x4*)(wr + ((4 * a + g) ^ swz_rows<RB>(row)) * 16);
          const V4 f = __builtin_bit_cast(V4, b);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = fmaf(x, (float)f[e], acc[a][4 * g + e]);
            acc[a][4 * g + e] = seen && (b[e] & 0x7fff) >= kInfBits<F16> ? y : acc[a][4 * g + e];
          }
        }
    }
  }
}

// Head of position `pos` among the workgroups of one tile: block b runs on XCD b % 8, so with g = gcd(8, heads) the
// positions of one residue mod g stay on 8 / g XCDs; they take neighbouring heads, whose keys and values are shared.
__device__ __forceinline__ int packed_head(int pos, int heads) {
  const int log = __builtin_ctz(heads | 8), g = 1 << log;
  return (pos & (g - 1)) * (heads >> log) + (pos >> log);
}

// The parts that a launch has workgroups for, `per` each: every tile (a partial one a sequence), the parts of split ones, and
// one spare at least wherever a row is of no sequence.
inline int64_t packed_blocks(int rows, int n, int per, bool split) {
  return (int64_t)(rows + kPackedTile - 1) / kPackedTile + n + (split ? (kPackedParts + per - 1) / per : 0);
}
// Whether tiles may be split (`others`: rows of the other side, in all: offsets are on the GPU): the second kernel's launch,
// 3 us where it finds nothing to add, is spared short batches.
constexpr int kPackedSplit = 5;
inline bool packed_splits(int64_t others) { return others > 1536; }

// The shape of a launch, and with many sequences the launch that finds their tiles first.
template <bool KEYS>
inline int packed_begin(PackedParams* p, int rows, int per, hipStream_t s) {
  p->per = per;
  p->per_rcp = 0xffffffffu / (uint32_t)per;
  p->blocks = (int)packed_blocks(rows, p->n, per, p->split_least > 0);
  p->half = kPackedSlots / 2 / per > 0 ? kPackedSlots / 2 / per : 1;
  if (!p->plan) return VMO_OK;
  hipLaunchKernelGGL((packed_plan_kernel<KEYS>), dim3((unsigned)((p->blocks + kPackedWaves - 1) / kPackedWaves)),
                     dim3(64 * kPackedWaves), (size_t)p->n * kPackedSeqBytes, s, *p);
  return launch_status("packed_plan");
}

int packed_fwd_launch(const PackedParams& p, bool f16, int d, hipStream_t s);
int packed_bwd_launch(const PackedParams& p, bool f16, int d, hipStream_t s);
int packed_bwd_splits(int64_t tk, int kv_heads, int group);

}  // namespace vmo
