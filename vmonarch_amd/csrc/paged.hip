// A paged key / value cache: attention of one new token a sequence over it, new rows into it, pages copied within it.
//
// Pages are (pages, heads, page tokens, D); token t of sequence b lies at place t % page of page table[b][t / page].  Table
// and lengths are read on the GPU, so a captured graph replays with others.  A page number outside the cache, or a length
// beyond the table, is not followed: attention gives NaN for that sequence, appending leaves the row out.
#include "packed.h"

#include <stdlib.h>

namespace vmo {

constexpr int kPagedTile = 32;   // keys of a tile, one step of a wave
constexpr float kPagedSumMost = 32768.f, kPagedNoMax = -3.0e38f;   // as in the forward of whole prompts

struct PagedParams {
  const void *q, *k, *v;
  void* o;
  int64_t q_sb, q_sh, o_sb, o_sh, k_sp, k_sh, k_sn, v_sp, v_sh, v_sn;
  const int32_t *table, *lengths;
  int64_t t_sb;
  int batch, heads, kv_heads, group, pages, page_log, width;   // width: page numbers a sequence has in the table
  int blocks, per;           // a sequence's rows: kv_heads x blocks of `per` (at most 32) query heads
  int waves, q_rows;         // waves launched; query rows that an LDS slot holds (per, in whole copies)
  float *part_o, *part_ml;   // (waves + batch kv_heads blocks) parts of (per, D), and of (per, 2): sums, then m and l
  int* starts;
  float c;
};

// A sequence's tiles.  One without tokens, or whose length is beyond the table (bad), has one that sees nothing: somebody
// writes its rows.
struct PagedSeq { int len, tiles; bool bad; };
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int len) {
  PagedSeq s;
  s.bad = len > ((int64_t)p.width << p.page_log);
  s.len = s.bad ? 0 : max(len, 0);
  s.tiles = max((s.len + kPagedTile - 1) / kPagedTile, 1);
  return s;
}
// Tiles of all rows stand in one order (sequence, row of it, tile) and are dealt to the waves in equal shares of their
// cost: a tile counts 1, a row's begin and end c_row more (1 where a wave has two tiles at least: 64 sequences of 16 to 8192
// tokens, 8 heads of 128: 83.6 -> 73.3 us, as the short rows otherwise end up with a few waves).  A row that several waves
// hold has a part from each, in place (wave + row): along the order one of the two grows with every part, so places are its
// own.  starts[w]: the row that wave w begins inside of, or -1.

// ------------------------------------------------------------------------------------------------
// A wave is a workgroup of its own and walks its share of the tiles, over the ends of sequences: 32 keys of one key / value
// head against the query heads of its group, the columns of the 32-wide products (S^T = K Q^T, O^T += V^T P^T, a lane one
// query head, as in the forward of whole prompts).  Two LDS slots take a tile's K and V; once tile i has landed it goes to
// registers whole and tile i + 2 is fetched into its place before anything is computed, so that the copies of two tiles
// are under way all the time (with K and V held in LDS through their products 24 KB a wave are, 32 KB so: 64 sequences of
// 84k tokens in all, 8 heads of 128, 87.2 -> 83.6 us), and no barrier is met.  Page numbers and lengths come through the scalar unit, whose waits
// leave the copies alone; a copy instruction lies within one page (pages hold 8 tokens at least), so its address is scalar.
// Bound by the bytes of the cache, 2 D 2 a key and head, and by how many of them are in flight: those 64 sequences' 356 MB in 68
// us, 5.2 TB/s.
template <bool F16, int D>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagedParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  using V8 = typename E::V8;
  typedef const __attribute__((address_space(4))) int32_t* scalar_ints;
  constexpr int RB = D * 2, UNIT = kPagedTile * RB, NA = D / 32, NDS = D / 16;
  constexpr int CH = D / 8, RPI = 64 / CH, NI = kPagedTile / RPI;   // copies of a K (or V) tile
  constexpr int NV = 16 / RPI;                                      // lane offsets: the swizzle's period is 16 rows
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  VMO_LDS char* smem = (VMO_LDS char*)smem_raw;
  const uint32_t lds = (uint32_t)(uintptr_t)smem;
  auto uni = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };
  const int lane = threadIdx.x, hl = lane >> 5, l32 = lane & 31;
  const scalar_ints lengths = (scalar_ints)(uintptr_t)p.lengths, table = (scalar_ints)(uintptr_t)p.table;
  const int X = p.kv_heads * p.blocks;   // rows of a sequence

  // this wave's tiles: sums of 64 sequences each wait in LDS, then the sequence that holds a position of the order
  // (the first 64, often all, stay in registers)
  auto tiles_of = [&](int at, int len) __attribute__((always_inline)) { return at < p.batch ? paged_seq(p, len).tiles : 0; };
  auto length_at = [&](int at) __attribute__((always_inline)) { return p.lengths[min(at, p.batch - 1)]; };
  VMO_LDS int* sums = (VMO_LDS int*)smem;
  const int n_sums = (p.batch + 63) / 64;
  const int len0 = length_at(lane), tiles0 = tiles_of(lane, len0), upto0 = wave_scan_i32(tiles0);
  int64_t all = __builtin_amdgcn_readlane(upto0, 63);
  if (n_sums > 1) {
    if (lane == 0) sums[0] = (int)all;
#pragma unroll 4
    for (int i = 1; i < n_sums; ++i) {
      const int t = wave_sum_i32(tiles_of(i * 64 + lane, length_at(i * 64 + lane)));
      if (lane == 0) sums[i] = t;
      all += t;
    }
  }
  // 64-bit division is long: 32 bits where both fit
  auto quotient = [](int64_t a, int64_t b) __attribute__((always_inline)) {
    return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
  };
  const int c_row = all * X >= 2 * (int64_t)p.waves ? 1 : 0;
  const int64_t total = (all + (int64_t)c_row * p.batch) * X, W = p.waves < total ? p.waves : total, w = blockIdx.x;
  if (w >= W) {
    if (lane == 0) p.starts[w] = -1;
    return;
  }
  struct Place { int b, x, tile, len; int64_t tiles; };   // tiles: of all rows before it
  auto place_of = [&](int64_t pos) __attribute__((always_inline)) {
    Place r;
    int64_t before = 0;   // tiles of the sequences before, of one row
    int i = 0;
    while (i + 1 < n_sums && (before + sums[i] + (int64_t)c_row * 64 * (i + 1)) * X <= pos) before += sums[i++];
    int len = len0, tiles = tiles0, upto = upto0;
    if (i > 0) {
      len = length_at(i * 64 + lane);
      tiles = tiles_of(i * 64 + lane, len);
      upto = wave_scan_i32(tiles);
    }
    const uint64_t over = __builtin_amdgcn_ballot_w64((before + upto + (int64_t)c_row * (i * 64 + lane + 1)) * X > pos);
    const int who = over ? __builtin_ctzll(over) : min(63, p.batch - 1 - i * 64);   // (none: the end of the last sequence)
    const int mine = __builtin_amdgcn_readlane(tiles, who);
    r.b = __builtin_amdgcn_readfirstlane(i * 64 + who);
    r.len = __builtin_amdgcn_readlane(len, who);
    before += __builtin_amdgcn_readlane(upto, who) - mine;
    const int64_t rest = pos - (before + (int64_t)c_row * r.b) * X;
    r.x = (int)quotient(rest, mine + c_row);
    r.tile = max((int)(rest - (int64_t)r.x * (mine + c_row)) - c_row, 0);
    r.tiles = before * X + (int64_t)r.x * mine + r.tile;
    return r;
  };
  const Place from = place_of(quotient(w * total, W)), to = place_of(quotient((w + 1) * total, W));
  const int n = (int)(to.tiles - from.tiles);
  if (lane == 0) p.starts[w] = from.tile > 0 ? from.b * X + from.x : -1;
  if (n <= 0) return;
  __syncthreads();   // (one wave: its LDS reads are done before the copies come)
  struct Cursor { int b, x, tile; PagedSeq s; };   // row x of sequence b, its tile
  Cursor at;
  at.b = uni(from.b);
  at.x = uni(from.x);
  at.tile = uni(from.tile);
  at.s = paged_seq(p, uni(from.len));
  auto advance = [&](Cursor& c) __attribute__((always_inline)) {
    if (++c.tile < c.s.tiles) return;
    c.tile = 0;
    if (++c.x < X) return;
    c.x = 0;
    c.b = min(c.b + 1, p.batch - 1);
    c.s = paged_seq(p, lengths[c.b]);
  };

  // lane offsets of the copies (rows r0 + lane / CH of a tile, chunks swizzled by the row)
  uint32_t koff[NV], voff[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int r = j * RPI + lane / CH;
    const uint32_t chunk = ((lane % CH) ^ swz_rows<RB>(r)) * 16;
    koff[j] = (uint32_t)((lane / CH) * p.k_sn * 2) + chunk;
    voff[j] = (uint32_t)((lane / CH) * p.v_sn * 2) + chunk;
  }
  // The tile under `next`.  Its page numbers (raw[j]: rows 8 j .. 8 j + 7) are asked for when the tile before is issued.  A
  // number outside the cache is not followed: page 0 instead, and the row is marked (bit i % 4 of `wrong`).  Offsets within
  // a page have 32 bits, and so have page strides in bytes.
  Cursor next = at;
  int raw[4];
  uint32_t wrong = 0;
  const int place_mask = (1 << p.page_log) - 1;
  const uint32_t k_row = (uint32_t)p.k_sn * 2, v_row = (uint32_t)p.v_sn * 2, k_page = (uint32_t)(p.k_sp * 2), v_page = (uint32_t)(p.v_sp * 2);
  auto ask_pages = [&]() __attribute__((always_inline)) {
    // (a sequence without tokens reads its first place, which the table has)
    const int first_page = (next.tile * kPagedTile) >> p.page_log, last = max((next.s.len - 1) >> p.page_log, 0);
    const scalar_ints row = table + next.b * p.t_sb;
#pragma unroll
    for (int j = 0; j < 4; ++j) raw[j] = row[min(first_page + ((8 * j) >> p.page_log), last)];
  };
  const uint32_t q_slots = lds + 4 * UNIT;
  const int slot_bytes = p.q_rows * RB;
  auto issue = [&](int i) __attribute__((always_inline)) {
    const int kvh = next.x / p.blocks;
    if (next.tile == 0 || i == 0) {   // the row's queries too
      const int h0 = kvh * p.group + (next.x % p.blocks) * p.per, most = min(p.per, p.group - (next.x % p.blocks) * p.per) - 1;
      for (int r = 0; r < p.q_rows; r += RPI)
        dma16_async((const T*)p.q + next.b * p.q_sb + (h0 + min(r + lane / CH, most)) * p.q_sh + (lane % CH) * 8,
                    q_slots + (i & 3) * slot_bytes + r * RB);
    }
    bool bad = next.s.bad;
    uint32_t id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool out = (uint32_t)raw[j] >= (uint32_t)p.pages;
      bad |= out && next.s.len > 0;
      id[j] = out ? 0 : raw[j];
    }
    wrong = (wrong & ~(1u << (i & 3))) | (bad ? 1u << (i & 3) : 0u);
    const uint32_t key0 = next.tile * kPagedTile, dst = lds + (i & 1) * 2 * UNIT;
    auto copy_tile = [&](const void* base, int64_t sh, uint32_t page, uint32_t row, const uint32_t (&off)[NV], uint32_t to)
        __attribute__((always_inline)) {
      const uint64_t head = (uint64_t)(uintptr_t)base + (uint64_t)(kvh * sh * 2) + (uint64_t)((key0 & place_mask) * row);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint64_t at8 = head + (uint64_t)id[j] * page + (uint64_t)(((8 * j) & place_mask) * row);
#pragma unroll
        for (int h = 0; h < 8 / RPI; ++h)
          dma16_async_s(at8 + (uint64_t)(h * RPI) * row, off[(j * (8 / RPI) + h) % NV], to + (j * (8 / RPI) + h) * 1024);
      }
    };
    copy_tile(p.k, p.k_sh, k_page, k_row, koff, dst);
    copy_tile(p.v, p.v_sh, v_page, v_row, voff, dst + UNIT);
    if (i + 1 < n) {
      advance(next);
      ask_pages();
    }
  };
  auto reads_done = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); };

  const float c = p.c;
  V8 qf[NDS];
  float m_run = kPagedNoMax, l_run = 0.f;
  f32x16 acc[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) acc[a] = f32x16{};
  const int sw = swz_rows<RB>(l32);
  const int trow = 4 * hl + ((lane & 15) >> 2), tchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), tbyte = (lane & 1) * 8;
  bool begun = at.tile == 0, row_wrong = false;   // whether the wave has the row from its first tile

  ask_pages();
  issue(0);
  if (n > 1) issue(1);
  for (int i = 0; i < n; ++i) {
    VMO_LDS char* Ks = smem + (i & 1) * 2 * UNIT;
    if (i + 1 < n) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * NI) : "memory");   // all but tile i + 1 has landed
    else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    const int nh = min(p.per, p.group - (at.x % p.blocks) * p.per);
    if (at.tile == 0 || i == 0) {
      const VMO_LDS char* qs = smem + 4 * UNIT + (i & 3) * slot_bytes + min(l32, nh - 1) * RB + hl * 16;
#pragma unroll
      for (int ds = 0; ds < NDS; ++ds) qf[ds] = lds_read8<V8>(qs + ds * 32);
    }
    row_wrong |= (wrong >> (i & 3)) & 1;
    const int nvis = at.s.len - at.tile * kPagedTile;   // keys of the tile that there are
    if (nvis < kPagedTile) {   // places without a token hold anything: 0 times that need not be 0
      const int gone = max(nvis, 0);
      for (int j = lane; j < (kPagedTile - gone) * CH; j += 64) *(VMO_LDS f32x4*)(Ks + UNIT + gone * RB + j * 16) = f32x4{};
      reads_done();
    }
    // the whole tile into registers, so that its slots can be filled again before anything is computed
    V8 kf[NDS], vf[2 * NA];
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) kf[ds] = lds_read8<V8>(Ks + l32 * RB + ((2 * ds + hl) ^ sw) * 16);
#pragma unroll
    for (int j = 0; j < 2 * NA; ++j) {
      const int c0 = trow * RB + (((4 * (j / 2) + tchunk) ^ swz_rows<RB>(trow)) * 16 + tbyte);
      const VMO_LDS char* rp = Ks + UNIT + 16 * (j % 2) * RB;
      vf[j] = lds_read_tr8<V8>(rp + c0, rp + 8 * RB + (c0 ^ 32));
    }
    reads_done();
    if (i + 2 < n) issue(i + 2);

    f32x16 s = f32x16{};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) s = E::mfma(kf[ds], qf[ds], s);
    V8 P[2];
    auto weights = [&]() __attribute__((always_inline)) {
      float ls = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = fmaf(s[r], c, -m_run);
        x = 8 * (r >> 2) + 4 * hl + (r & 3) < nvis ? x : kMaskLogit;
        const float y = fast_exp2(x);
        ls += y;
        P[r >> 3][r & 7] = to_elem<T>(y);
      }
      return ls;
    };
    float ls = weights();
    const bool over = !(ls <= kPagedSumMost);
    if (__builtin_amdgcn_ballot_w64(over) != 0) {   // m moves to the row's maximum so far (see the forward of whole prompts)
      const auto either = __builtin_amdgcn_permlane32_swap(over, over, false, false);
      float mx = kPagedNoMax;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, 8 * (r >> 2) + 4 * hl + (r & 3) < nvis ? s[r] * c : kPagedNoMax);
      const float m_new = either[0] | either[1] ? fmaxf(m_run, wave_max32(mx)) : m_run, f = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= f;
#pragma unroll
      for (int a = 0; a < NA; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[a][r] *= f;
      ls = weights();
    }
    l_run += ls;

#pragma unroll
    for (int j = 0; j < 2 * NA; ++j) acc[j / 2] = E::mfma(vf[j], P[j % 2], acc[j / 2]);

    const bool ends = at.tile + 1 == at.s.tiles;
    if (ends || i + 1 == n) {   // the row is done here: whole, or this wave's part of it
      float l = wave_sum32(l_run);
      if (row_wrong) l = __uint_as_float(0x7fc00000u);   // NaN
      const bool mine = l32 < nh;
      if (ends && begun) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* out = (T*)p.o + at.b * p.o_sb + ((int64_t)(at.x / p.blocks) * p.group + (at.x % p.blocks) * p.per + l32) * p.o_sh;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            typename E::V4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = to_elem<T>(acc[a][4 * g + e] * inv);
            if (mine) *(typename E::V4*)(out + 32 * a + 8 * g + 4 * hl) = y;
          }
      } else {
        const int64_t part = (w + (int64_t)at.b * X + at.x) * p.per + l32;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (mine) *(f32x4*)(p.part_o + part * D + 32 * a + 8 * g + 4 * hl) =
                f32x4{acc[a][4 * g], acc[a][4 * g + 1], acc[a][4 * g + 2], acc[a][4 * g + 3]};
        if (mine && hl == 0) {
          p.part_ml[2 * part] = m_run;
          p.part_ml[2 * part + 1] = l;
        }
      }
      m_run = kPagedNoMax;
      l_run = 0.f;
      row_wrong = false;
      begun = true;
#pragma unroll
      for (int a = 0; a < NA; ++a) acc[a] = f32x16{};
    }
    if (i + 1 < n) advance(at);
  }
}

// o of a row that several waves hold, one query head a workgroup: the workgroup of the first wave that begins inside it.
// D / 4 lanes a part, 256 / (D / 4) parts side by side, each group with a running maximum over its own, then the groups in
// LDS in their order.  Bound by the latency of two reads in a row (starts, parts).
template <bool F16, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
  using T = typename Elem<F16>::T;
  constexpr int TPR = D / 4, NG = 256 / TPR;
  __shared__ float sums[NG][D], ml[NG][2];
  const int w = blockIdx.x, in = blockIdx.y, tid = threadIdx.x;
  const int row = p.starts[w], last = w > 0 ? p.starts[w - 1] : -1, near = p.starts[min(w + tid, p.waves - 1)];
  if (row < 0 || row == last) return;
  const int X = p.kv_heads * p.blocks, b = row / X, x = row % X, block = x % p.blocks;
  if (in >= min(p.per, p.group - block * p.per)) return;
  const int h = (x / p.blocks) * p.group + block * p.per + in;
  // waves w .. w + more - 1 begin inside the row; wave w - 1 has its first tiles
  __shared__ int firsts[4];
  int more = 0;
  for (bool on = true; on; ) {
    const int v = w + more + tid;
    const uint64_t out = __builtin_amdgcn_ballot_w64(v >= p.waves || (more == 0 ? near : p.starts[min(v, p.waves - 1)]) != row);
    if ((tid & 63) == 0) firsts[tid >> 6] = out ? __builtin_ctzll(out) : 64;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (on) more += firsts[i];
      on = on && firsts[i] == 64;
    }
    __syncthreads();
  }
  const int g = tid / TPR, d4 = (tid % TPR) * 4;
  float m = kPagedNoMax, l = 0.f;
  f32x4 acc = f32x4{};
#pragma unroll 4
  for (int v = g; v <= more; v += NG) {
    const int64_t part = (w - 1 + v + (int64_t)row) * p.per + in;
    const float pm = p.part_ml[2 * part], pl = p.part_ml[2 * part + 1];
    const f32x4 y = *(const f32x4*)(p.part_o + part * D + d4);
    const float m_new = fmaxf(m, pm), f = fast_exp2(m - m_new), pf = fast_exp2(pm - m_new);
    m = m_new;
    l = fmaf(l, f, pl * pf);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(acc[e], f, y[e] * pf);
  }
  *(f32x4*)&sums[g][d4] = acc;
  if (d4 == 0) {
    ml[g][0] = m;
    ml[g][1] = l;
  }
  __syncthreads();
  if (g > 0) return;
  m = kPagedNoMax;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < NG; ++i) m = fmaxf(m, ml[i][0]);
  acc = f32x4{};
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float f = fast_exp2(ml[i][0] - m);
    l = fmaf(ml[i][1], f, l);
    const f32x4 y = *(const f32x4*)&sums[i][d4];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(y[e], f, acc[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  typename Elem<F16>::V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = to_elem<T>(acc[e] * inv);
  *(typename Elem<F16>::V4*)((T*)p.o + (int64_t)b * p.o_sb + (int64_t)h * p.o_sh + d4) = y;
}

// ------------------------------------------------------------------------------------------------
struct AppendParams {
  const void *k, *v;
  void *kp, *vp;
  int64_t k_sh, k_sn, v_sh, v_sn, k_sp, kp_sh, kp_sn, v_sp, vp_sh, vp_sn;
  const int32_t *table, *lengths, *offsets;   // offsets null: row b belongs to sequence b
  int64_t t_sb;
  int n, tokens, kv_heads, pages, page_log, width, chunks;   // chunks: 16-byte pieces of a row
};

// New rows into their pages: one thread a 16-byte piece of a K row and of the V row beside it.  Row i of sequence b's n_b
// new ones goes to place lengths[b] - n_b + i, the last to the sequence's end.  Bound by memory (12 prompts of 40 to 9000 tokens, 8
// heads of 128, 189 MB: 31 us with the rows in the last-level cache, 41 without), for few rows by the launch (64: 3.7 us).
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per_row = p.kv_heads * p.chunks;
  const int64_t row64 = gid / per_row;
  if (row64 >= p.tokens) return;
  const int row = (int)row64, piece = (int)(gid % per_row), h = piece / p.chunks, ch = piece % p.chunks;
  int b = row, last = row + 1;
  if (p.offsets) {
    int lo = 0, hi = p.n;   // the last sequence that begins at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.offsets[mid] <= row) lo = mid;
      else hi = mid;
    }
    b = lo;
    last = p.offsets[b + 1];
    if (p.offsets[b] > row || last <= row) return;   // no sequence has this row
  }
  const int64_t at = (int64_t)p.lengths[b] - (last - row);
  if (at < 0 || at >= ((int64_t)p.width << p.page_log)) return;
  const int id = p.table[(int64_t)b * p.t_sb + (at >> p.page_log)];
  if (id < 0 || id >= p.pages) return;
  const int64_t place = at & ((1 << p.page_log) - 1);
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 x = *(const u32x4*)((const char*)p.k + (h * p.k_sh + row * p.k_sn) * 2 + ch * 16);
  const u32x4 y = *(const u32x4*)((const char*)p.v + (h * p.v_sh + row * p.v_sn) * 2 + ch * 16);
  *(u32x4*)((char*)p.kp + (id * p.k_sp + h * p.kp_sh + place * p.kp_sn) * 2 + ch * 16) = x;
  *(u32x4*)((char*)p.vp + (id * p.v_sp + h * p.vp_sh + place * p.vp_sn) * 2 + ch * 16) = y;
}

// ------------------------------------------------------------------------------------------------
// Page pairs of a launch travel as its argument, at most 3.5 of its 4 KB; up to 48 pairs a small one (0.2 us less of the 3.8 that
// a call with one pair takes the host).
constexpr int kCopyPairs = 448, kCopyFew = 48;
template <int PAIRS>
struct CopyParams {
  char *k, *v;
  int64_t page_bytes, layer_bytes;
  int pieces;
  int32_t src[PAIRS], dst[PAIRS];
};
constexpr int kCopyPiece = 256 * 16;   // bytes a workgroup moves

// Pages src[i] to dst[i] of every layer, K and V.  Bound by memory (12 layers x 256 pages of 16 KB: 29.7 us, 6.8 TB/s, some of
// it from the last-level cache), the small copies by the launch (32 pages: 4.1 us).  One 16-byte piece a lane: with four the
// two were 9% and 29% slower (fewer workgroups start slower); stored past the caches: 15% on the small one.
template <int PAIRS>
__global__ __launch_bounds__(256) void paged_copy_kernel(CopyParams<PAIRS> p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));   // (HIP's own uint4 went through registers one at a time)
  const int piece = (int)blockIdx.x % p.pieces, pair = (int)blockIdx.x / p.pieces, layer = (int)blockIdx.y;
  char* base = (blockIdx.z ? p.v : p.k) + layer * p.layer_bytes;
  const int64_t at = (int64_t)piece * kCopyPiece + threadIdx.x * 16;
  if (at < p.page_bytes)
    __builtin_nontemporal_store(*(const u32x4*)(base + p.src[pair] * p.page_bytes + at), (u32x4*)(base + p.dst[pair] * p.page_bytes + at));
}

// ---- launches ---------------------------------------------------------------------------------------------------------
template <int PAIRS>
static int launch_copy(const vmo_copy_args* a, int first, int pairs, int pieces, hipStream_t s) {
  CopyParams<PAIRS> p;
  p.k = (char*)a->k; p.v = (char*)a->v; p.page_bytes = a->page_bytes; p.layer_bytes = a->layer_bytes;
  p.pieces = pieces;
  for (int i = 0; i < PAIRS; ++i) {
    p.src[i] = i < pairs ? a->src[first + i] : 0;
    p.dst[i] = i < pairs ? a->dst[first + i] : 0;
  }
  hipLaunchKernelGGL((paged_copy_kernel<PAIRS>), dim3((unsigned)(pieces * pairs), (unsigned)a->layers, 2), dim3(256), 0, s, p);
  return launch_status("copy_pages");
}

// Waves of a launch: as many as the chip holds at once (256 CUs of 160 KB LDS), one round.  LDS of a wave: two K and two V
// tiles, four slots of its group's queries.
struct PagedShape { int blocks, per, q_rows, lds, waves; };
static PagedShape paged_shape(const vmo_paged_args* a) {
  PagedShape s;
  const int group = a->heads / a->kv_heads, rpi = 512 / a->d;
  s.blocks = (group + 31) / 32;
  s.per = (group + s.blocks - 1) / s.blocks;
  s.q_rows = (s.per + rpi - 1) / rpi * rpi;
  s.lds = 4 * kPagedTile * a->d * 2 + 4 * s.q_rows * a->d * 2;
  const int fit = 160 * 1024 / s.lds;
  s.waves = 256 * (fit < 8 ? fit : 8);
  // no more than the tiles that the table has room for
  const int64_t most = (int64_t)a->batch * a->kv_heads * s.blocks * (((int64_t)a->table_width * a->page_size + kPagedTile - 1) / kPagedTile);
  if (most < s.waves) s.waves = most < 1 ? 1 : (int)most;
  return s;
}

template <bool F16, int D>
static int launch_paged(const PagedParams& p, int lds, hipStream_t s) {
  hipLaunchKernelGGL((paged_attention_kernel<F16, D>), dim3((unsigned)p.waves), dim3(64), lds, s, p);
  const int rc = launch_status("paged_attention");
  if (rc != VMO_OK) return rc;
  hipLaunchKernelGGL((paged_join_kernel<F16, D>), dim3((unsigned)p.waves, (unsigned)p.per), dim3(256), 0, s, p);
  return launch_status("paged_join");
}

static int log2_of(int x) {
  int l = 0;
  while ((1 << l) < x) ++l;
  return l;
}
static bool page_size_ok(int n) { return n >= 8 && n <= 1024 && (n & (n - 1)) == 0; }

}  // namespace vmo

extern "C" size_t vmo_paged_attention_workspace_size(const vmo_paged_args* a) {
  if (!a || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || (a->d != 64 && a->d != 128) ||
      a->table_width <= 0 || a->page_size <= 0)
    return 0;
  const vmo::PagedShape s = vmo::paged_shape(a);
  return (size_t)((s.waves + (int64_t)a->batch * a->kv_heads * s.blocks) * s.per * (a->d + 2) * 4 + s.waves * 4);
}

extern "C" int vmo_paged_attention(const vmo_paged_args* a, void* stream) {
  using namespace vmo;
  clear_error();
  if (!a) return set_error(VMO_ERR_INVALID, "paged_attention: null args");
  if (a->dtype != VMO_DTYPE_BF16 && a->dtype != VMO_DTYPE_F16) return set_error(VMO_ERR_INVALID, "paged_attention: dtype %d", a->dtype);
  if (a->batch < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
    return set_error(VMO_ERR_INVALID, "paged_attention: %d query heads over %d key / value heads", a->heads, a->kv_heads);
  if (a->d != 64 && a->d != 128) return set_error(VMO_ERR_UNSUPPORTED, "paged_attention: head dim %d (64 and 128 are built)", a->d);
  if (!page_size_ok(a->page_size))
    return set_error(VMO_ERR_UNSUPPORTED, "paged_attention: pages of %d tokens (powers of two from 8 to 1024)", a->page_size);
  if (a->batch == 0) return VMO_OK;
  if (a->pages < 1 || a->table_width < 1 || (int64_t)a->table_width * a->page_size > (1ll << 28) ||
      (int64_t)a->batch * a->heads > (1ll << 30) || a->batch > (1 << 18))   // (sums of 64 sequences wait in 16 KB of LDS)
    return set_error(VMO_ERR_INVALID, "paged_attention: %d pages, %d page numbers a sequence", a->pages, a->table_width);
  if (!a->table || !a->lengths) return set_error(VMO_ERR_INVALID, "paged_attention: no page table or lengths");
  if (!view_ok(a->k) || !view_ok(a->v) || !a->q.data || !a->o.data || !aligned16(a->q.data) || !aligned16(a->o.data) ||
      a->q.stride_b % 8 || a->q.stride_h % 8 || a->o.stride_b % 8 || a->o.stride_h % 8)
    return set_error(VMO_ERR_INVALID, "paged_attention: tensors need 16-byte aligned rows (strides multiple of 8 elements)");
  if (a->k.stride_n >= (1ll << 27) || a->v.stride_n >= (1ll << 27))   // (32-bit lane offsets over up to 7 rows)
    return set_error(VMO_ERR_UNSUPPORTED, "paged_attention: token stride must be below 2^27 elements");
  for (const vmo_view* x : {&a->k, &a->v})   // offsets within a page, and page strides, in 32 bits of bytes
    if (x->stride_b < 0 || x->stride_b >= (1ll << 31) || x->stride_n * a->page_size >= (1ll << 30))
      return set_error(VMO_ERR_UNSUPPORTED, "paged_attention: pages must be below 2^31 elements apart, a head of one below 2^30 long");
  if (!(a->sm_scale >= 0.f) || a->sm_scale > 3.0e38f)
    return set_error(VMO_ERR_INVALID, "paged_attention: sm_scale must be finite and >= 0");
  PagedParams p{};
  p.q = a->q.data; p.k = a->k.data; p.v = a->v.data; p.o = a->o.data;
  p.q_sb = a->q.stride_b; p.q_sh = a->q.stride_h; p.o_sb = a->o.stride_b; p.o_sh = a->o.stride_h;
  p.k_sp = a->k.stride_b; p.k_sh = a->k.stride_h; p.k_sn = a->k.stride_n;
  p.v_sp = a->v.stride_b; p.v_sh = a->v.stride_h; p.v_sn = a->v.stride_n;
  p.table = a->table; p.lengths = a->lengths; p.t_sb = a->table_stride;
  p.batch = a->batch; p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads;
  p.pages = a->pages; p.page_log = log2_of(a->page_size); p.width = a->table_width;
  const PagedShape shape = paged_shape(a);
  p.blocks = shape.blocks; p.per = shape.per; p.q_rows = shape.q_rows; p.waves = shape.waves;
  const size_t need = vmo_paged_attention_workspace_size(a);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)))
    return set_error(VMO_ERR_WORKSPACE, "paged_attention: needs %llu workspace bytes, has %llu", (unsigned long long)need,
                     (unsigned long long)(a->workspace ? a->workspace_bytes : 0));
  p.part_o = (float*)a->workspace;
  p.part_ml = p.part_o + (p.waves + (int64_t)a->batch * a->kv_heads * p.blocks) * p.per * a->d;
  p.starts = (int*)(p.part_ml + (p.waves + (int64_t)a->batch * a->kv_heads * p.blocks) * p.per * 2);
  p.c = a->sm_scale * kLog2e;
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = a->dtype == VMO_DTYPE_F16;
  if (a->d == 64) return f16 ? launch_paged<true, 64>(p, shape.lds, s) : launch_paged<false, 64>(p, shape.lds, s);
  return f16 ? launch_paged<true, 128>(p, shape.lds, s) : launch_paged<false, 128>(p, shape.lds, s);
}

extern "C" int vmo_append_pages(const vmo_append_args* a, void* stream) {
  using namespace vmo;
  clear_error();
  if (!a) return set_error(VMO_ERR_INVALID, "append_pages: null args");
  if (a->tokens < 0 || a->sequences < 0 || a->kv_heads < 1 || a->d < 8 || a->d % 8 || a->d > 1024)
    return set_error(VMO_ERR_INVALID, "append_pages: %d rows of %d sequences, %d heads of %d", a->tokens, a->sequences, a->kv_heads,
                     a->d);
  if (!page_size_ok(a->page_size))
    return set_error(VMO_ERR_UNSUPPORTED, "append_pages: pages of %d tokens (powers of two from 8 to 1024)", a->page_size);
  if (a->tokens == 0 || a->sequences == 0) return VMO_OK;
  if (!a->offsets && a->tokens != a->sequences)
    return set_error(VMO_ERR_INVALID, "append_pages: without offsets one row a sequence, got %d for %d", a->tokens, a->sequences);
  if (a->pages < 1 || a->table_width < 1 || (int64_t)a->table_width * a->page_size > (1ll << 30))
    return set_error(VMO_ERR_INVALID, "append_pages: %d pages, %d page numbers a sequence", a->pages, a->table_width);
  if (!a->table || !a->lengths) return set_error(VMO_ERR_INVALID, "append_pages: no page table or lengths");
  if (!view_ok(a->k) || !view_ok(a->v) || !view_ok(a->k_pages) || !view_ok(a->v_pages))
    return set_error(VMO_ERR_INVALID, "append_pages: tensors need 16-byte aligned rows (strides multiple of 8 elements)");
  AppendParams p{};
  p.k = a->k.data; p.v = a->v.data; p.kp = a->k_pages.data; p.vp = a->v_pages.data;
  p.k_sh = a->k.stride_h; p.k_sn = a->k.stride_n; p.v_sh = a->v.stride_h; p.v_sn = a->v.stride_n;
  p.k_sp = a->k_pages.stride_b; p.kp_sh = a->k_pages.stride_h; p.kp_sn = a->k_pages.stride_n;
  p.v_sp = a->v_pages.stride_b; p.vp_sh = a->v_pages.stride_h; p.vp_sn = a->v_pages.stride_n;
  p.table = a->table; p.lengths = a->lengths; p.offsets = a->offsets; p.t_sb = a->table_stride;
  p.n = a->sequences; p.tokens = a->tokens; p.kv_heads = a->kv_heads; p.pages = a->pages;
  p.page_log = log2_of(a->page_size); p.width = a->table_width; p.chunks = a->d / 8;
  const int64_t threads = (int64_t)a->tokens * a->kv_heads * p.chunks, blocks = (threads + 255) / 256;
  if (blocks > (1ll << 30)) return set_error(VMO_ERR_UNSUPPORTED, "append_pages: too many rows");
  hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, p);
  return launch_status("append_pages");
}

extern "C" int vmo_copy_pages(const vmo_copy_args* a, void* stream) {
  using namespace vmo;
  clear_error();
  if (!a) return set_error(VMO_ERR_INVALID, "copy_pages: null args");
  if (a->pairs < 0 || a->layers < 0 || a->pages < 0 || a->page_bytes < 0 || a->page_bytes % 16 || a->layer_bytes % 16)
    return set_error(VMO_ERR_INVALID, "copy_pages: %d pairs, %d layers, pages of %lld bytes", a->pairs, a->layers,
                     (long long)a->page_bytes);
  if (a->pairs == 0 || a->layers == 0 || a->page_bytes == 0) return VMO_OK;
  if (!a->k || !a->v || !aligned16(a->k) || !aligned16(a->v) || !a->src || !a->dst)
    return set_error(VMO_ERR_INVALID, "copy_pages: pages need 16-byte alignment, and lists of page numbers");
  const int64_t pieces = (a->page_bytes + kCopyPiece - 1) / kCopyPiece;
  if (a->layers > 65535 || pieces * kCopyPairs > (1ll << 30)) return set_error(VMO_ERR_UNSUPPORTED, "copy_pages: too large");
  // Copies run beside each other: a page written twice, or written and read, would hold whatever came last.
  char* role = (char*)calloc((size_t)a->pages + 1, 1);   // 1: read, 2: written
  if (!role) return set_error(VMO_ERR_WORKSPACE, "copy_pages: no host memory to check %d pages", a->pages);
  int at = -1;
  for (int i = 0; i < a->pairs && at < 0; ++i) {
    if (a->src[i] < 0 || a->src[i] >= a->pages || a->dst[i] < 0 || a->dst[i] >= a->pages || role[a->dst[i]]) at = i;
    else {
      role[a->dst[i]] = 2;
      if (role[a->src[i]] == 2) at = i;
      else role[a->src[i]] = 1;
    }
  }
  free(role);
  if (at >= 0)
    return set_error(VMO_ERR_INVALID, "copy_pages: page %d to %d of %d (each below that, none written twice or written and read)",
                     a->src[at], a->dst[at], a->pages);
  for (int done = 0; done < a->pairs; done += kCopyPairs) {
    const int pairs = a->pairs - done < kCopyPairs ? a->pairs - done : kCopyPairs;
    const int rc = pairs <= kCopyFew ? launch_copy<kCopyFew>(a, done, pairs, (int)pieces, (hipStream_t)stream)
                                     : launch_copy<kCopyPairs>(a, done, pairs, (int)pieces, (hipStream_t)stream);
    if (rc != VMO_OK) return rc;
  }
  return VMO_OK;
}
