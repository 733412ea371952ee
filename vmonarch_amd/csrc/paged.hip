// A paged key / value cache: attention of one new token a sequence over it, new rows into it, pages copied within it.
//
// Pages are (pages, heads, page tokens, D); token t of sequence b lies at place t % page of page table[b][t / page].  Table
// and lengths are read on the GPU, so a captured graph replays with others.  A page number outside the cache, or a length
// beyond the table, is not followed: attention gives NaN for that sequence, appending leaves the row out.
#include <stdlib.h>

#include "fea_fwd.h"

namespace vmo {

constexpr int kPagedWaves = 4;
constexpr int kPagedTile = 32;        // keys of a wave's tile
constexpr int kPagedMaxChunk = 2048;  // keys of a workgroup (their page numbers wait in LDS)
constexpr float kPagedNoMax = -3.0e38f;

struct PagedParams {
  const void *q, *k, *v;
  void* o;
  int64_t q_sb, q_sh, o_sb, o_sh, k_sp, k_sh, k_sn, v_sp, v_sh, v_sn;
  const int32_t *table, *lengths;
  int64_t t_sb;
  int batch, heads, kv_heads, group, pages, page_log, width;   // width: page numbers a sequence has in the table
  int chunk, chunks;                                           // keys a workgroup takes; workgroups a (sequence, head)
  float *part_o, *part_ml;                                     // (batch, heads, chunks, D), (.., 2): sums, then m and l
  float c;
};

// A sequence's length as the kernels take it: none below 0; `bad` beyond the table.
__device__ __forceinline__ int paged_length(const PagedParams& p, int b, bool& bad) {
  const int len = max(p.lengths[b], 0);
  bad = len > ((int64_t)p.width << p.page_log);
  return len;
}

// ------------------------------------------------------------------------------------------------
// One workgroup: `chunk` keys of one (sequence, key / value head), all query heads of its group as the columns of the
// 32-wide products (S^T = K Q^T, O^T += V^T P^T as the forward of whole prompts has them).  A wave takes every fourth tile
// of 32 keys through its own two LDS slots (its copies need no barrier: nobody else reads them), with its own running
// maximum and sum; the four waves are joined in LDS, the workgroups of a sequence by paged_join.
// Bound by the bytes of the cache: 2 D 2 bytes a key and head.
template <bool F16, int D>
__global__ __launch_bounds__(64 * kPagedWaves) void paged_attention_kernel(PagedParams p) {
  using E = Elem<F16>;
  using T = typename E::T;
  using V8 = typename E::V8;
  constexpr int RB = D * 2, K_BYTES = kPagedTile * RB, SLOT = 2 * K_BYTES, NA = D / 32, NDS = D / 16;
  constexpr int CH = D / 8, RPI = 64 / CH, NI = kPagedTile / RPI;   // copies of a K (or V) tile by one wave
  extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
  VMO_LDS char* smem = (VMO_LDS char*)smem_raw;
  VMO_LDS int* ids = (VMO_LDS int*)(smem + kPagedWaves * 2 * SLOT);   // the chunk's page numbers, then a flag
  auto uni = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };

  const int chunk = (int)blockIdx.x % p.chunks, bh = (int)blockIdx.x / p.chunks;
  const int kvh = bh % p.kv_heads, b = bh / p.kv_heads;
  const int h0 = kvh * p.group + (int)blockIdx.y * 32, nh = min(32, p.group - (int)blockIdx.y * 32);
  const int tid = threadIdx.x, wave = uni(tid >> 6), lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  bool bad;
  const int len = uni(paged_length(p, b, bad));
  const int beg = chunk * p.chunk;
  if (beg >= len && !(chunk == 0)) return;
  const int end = min(len, beg + p.chunk);
  int n_keys = bad ? 0 : max(end - beg, 0);

  // page numbers of the chunk, checked
  const int page0 = beg >> p.page_log, n_pages = n_keys > 0 ? ((beg + n_keys - 1) >> p.page_log) - page0 + 1 : 0;
  bool wrong = bad;
  for (int i = tid; i < n_pages; i += 64 * kPagedWaves) {
    const int id = p.table[(int64_t)b * p.t_sb + page0 + i];
    wrong |= id < 0 || id >= p.pages;
    ids[i] = min(max(id, 0), p.pages - 1);
  }
  const int any_wrong = __syncthreads_or(wrong);

  V8 qf[NDS];
  {
    const T* qp = (const T*)p.q + (int64_t)b * p.q_sb + (int64_t)(h0 + min(l32, nh - 1)) * p.q_sh + hl * 8;
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      qf[ds] = *(const V8*)(qp + ds * 16);
      asm volatile("" : "+v"(qf[ds]));
    }
  }
  const int n_tiles = (n_keys + kPagedTile - 1) / kPagedTile;
  const int mine = n_tiles > wave ? (n_tiles - wave + kPagedWaves - 1) / kPagedWaves : 0;
  const uint32_t ring = (uint32_t)(uintptr_t)smem + wave * 2 * SLOT;
  const char* kp = (const char*)p.k + (int64_t)kvh * p.k_sh * 2;
  const char* vp = (const char*)p.v + (int64_t)kvh * p.v_sh * 2;
  auto issue = [&](int i) __attribute__((always_inline)) {
    const uint32_t st = ring + (i & 1) * SLOT;
    const int key0 = beg + (wave + i * kPagedWaves) * kPagedTile;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = j * RPI + lane / CH;
      const int tok = min(key0 + r, end - 1);   // (keys past the end repeat the last one: masked)
      const int64_t id = ids[(tok >> p.page_log) - page0], at = tok & ((1 << p.page_log) - 1);
      const int byte = ((lane % CH) ^ swz_rows<RB>(r)) * 16;
      dma16_async(kp + (id * p.k_sp + at * p.k_sn) * 2 + byte, st + j * 1024);
      dma16_async(vp + (id * p.v_sp + at * p.v_sn) * 2 + byte, st + K_BYTES + j * 1024);
    }
  };
  const float c = p.c;
  float m_run = kPagedNoMax, l_run = 0.f;
  f32x16 acc[NA];
#pragma unroll
  for (int a = 0; a < NA; ++a) acc[a] = f32x16{};
  const int sw = swz_rows<RB>(l32);
  const int trow = 4 * hl + ((lane & 15) >> 2), tchunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), tbyte = (lane & 1) * 8;

  if (mine > 0) issue(0);
  for (int i = 0; i < mine; ++i) {
    if (i + 1 < mine) {
      issue(i + 1);
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * NI) : "memory");   // tile i has landed, i + 1 is under way
    } else {
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    }
    const VMO_LDS char* Ks = smem + wave * 2 * SLOT + (i & 1) * SLOT;
    f32x16 s = f32x16{};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds)
      s = E::mfma(lds_read8<V8>(Ks + l32 * RB + ((2 * ds + hl) ^ sw) * 16), qf[ds], s);
    const int nvis = n_keys - (wave + i * kPagedWaves) * kPagedTile;
    float mx = kPagedNoMax;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = 8 * (r >> 2) + 4 * hl + (r & 3) < nvis ? s[r] * c : -INFINITY;
      mx = fmaxf(mx, s[r]);
    }
    const float m_new = fmaxf(m_run, wave_max32(mx)), f = fast_exp2(m_run - m_new);
    m_run = m_new;
    V8 P[2];
    float ls = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = fast_exp2(s[r] - m_run);
      ls += x;
      P[r >> 3][r & 7] = to_elem<T>(x);
    }
    l_run = fmaf(l_run, f, ls);
#pragma unroll
    for (int a = 0; a < NA; ++a) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][r] *= f;
      const int c0 = trow * RB + (((4 * a + tchunk) ^ swz_rows<RB>(trow)) * 16 + tbyte);
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const VMO_LDS char* rp = Ks + K_BYTES + 16 * h2 * RB;
        acc[a] = E::mfma(lds_read_tr8<V8>(rp + c0, rp + 8 * RB + (c0 ^ 32)), P[h2], acc[a]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");   // the slot's reads are done before it is filled again
  }
  // join the four waves: m and l of each (column, wave), then the sums scaled to the common m, added in the waves' order
  __syncthreads();
  VMO_LDS float* ml = (VMO_LDS float*)smem;                  // [wave][32][2]
  VMO_LDS float* sums = (VMO_LDS float*)(smem + 1024);       // [wave][32][D + 4]
  constexpr int SR = D + 4;
  l_run = wave_sum32(l_run);
  if (hl == 0) {
    ml[(wave * 32 + l32) * 2] = m_run;
    ml[(wave * 32 + l32) * 2 + 1] = l_run;
  }
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[a][4 * g + e];
      if (l32 < nh) *(VMO_LDS f32x4*)(sums + (wave * 32 + l32) * SR + 32 * a + 8 * g + 4 * hl) = x;
    }
  __syncthreads();
  const bool whole = p.chunks == 1;
  for (int i = tid; i < nh * (D / 4); i += 64 * kPagedWaves) {
    const int h = i / (D / 4), d4 = (i % (D / 4)) * 4;
    float m = kPagedNoMax, l = 0.f;
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) m = fmaxf(m, ml[(w * 32 + h) * 2]);
    f32x4 x = f32x4{};
#pragma unroll
    for (int w = 0; w < kPagedWaves; ++w) {
      const float f = fast_exp2(ml[(w * 32 + h) * 2] - m);
      l = fmaf(ml[(w * 32 + h) * 2 + 1], f, l);
      const f32x4 y = *(const VMO_LDS f32x4*)(sums + (w * 32 + h) * SR + d4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], f, x[e]);
    }
    if (any_wrong) l = __uint_as_float(0x7fc00000u);   // NaN: a page number or length that leads outside
    if (whole) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      typename E::V4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = to_elem<T>(x[e] * inv);
      *(typename E::V4*)((T*)p.o + (int64_t)b * p.o_sb + (int64_t)(h0 + h) * p.o_sh + d4) = y;
    } else {
      const int64_t at = ((int64_t)b * p.heads + h0 + h) * p.chunks + chunk;
      *(f32x4*)(p.part_o + at * D + d4) = x;
      if (d4 == 0) {
        p.part_ml[2 * at] = m;
        p.part_ml[2 * at + 1] = l;
      }
    }
  }
}

// o of one (sequence, head) from its workgroups' parts: D / 4 lanes a row, the parts in their order.
template <bool F16, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
  using T = typename Elem<F16>::T;
  constexpr int TPR = D / 4;
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x, row = gid / TPR;
  const int d4 = (int)(gid % TPR) * 4;
  if (row >= (int64_t)p.batch * p.heads) return;
  const int b = (int)(row / p.heads), h = (int)(row % p.heads);
  bool bad;
  const int len = paged_length(p, b, bad);
  const int n = bad ? 1 : max(1, (len + p.chunk - 1) / p.chunk);
  float m = kPagedNoMax, l = 0.f;
  for (int s = 0; s < n; ++s) m = fmaxf(m, p.part_ml[2 * (row * p.chunks + s)]);
  f32x4 x = f32x4{};
  for (int s = 0; s < n; ++s) {
    const int64_t at = row * p.chunks + s;
    const float f = fast_exp2(p.part_ml[2 * at] - m);
    l = fmaf(p.part_ml[2 * at + 1], f, l);
    const f32x4 y = *(const f32x4*)(p.part_o + at * D + d4);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = fmaf(y[e], f, x[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  typename Elem<F16>::V4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = to_elem<T>(x[e] * inv);
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
// new ones goes to place lengths[b] - n_b + i, the last to the sequence's end.
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
constexpr int kCopyPairs = 448;   // page pairs of a launch: they travel as its argument (3.5 KB of 4 KB)
struct CopyParams {
  char *k, *v;
  int64_t page_bytes, layer_bytes;
  int pairs, pieces;
  int32_t src[kCopyPairs], dst[kCopyPairs];
};
constexpr int kCopyPiece = 256 * 16;   // bytes a workgroup moves

// Pages src[i] to dst[i] of every layer, K and V.  Bound by memory, the small copies by the launch: one 16-byte piece a
// lane (12 layers x 256 pages of 16 KB: 24.0 us against 26.1 with four a lane, whose fewer workgroups also start slower: 32
// pages 3.4 against 4.4 us), stored past the caches (3.4 against 3.9 us).
__global__ __launch_bounds__(256) void paged_copy_kernel(CopyParams p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));   // (HIP's own uint4 went through registers one at a time)
  const int piece = (int)blockIdx.x % p.pieces, pair = (int)blockIdx.x / p.pieces, layer = (int)blockIdx.y;
  char* base = (blockIdx.z ? p.v : p.k) + layer * p.layer_bytes;
  const int64_t at = (int64_t)piece * kCopyPiece + threadIdx.x * 16;
  if (at < p.page_bytes)
    __builtin_nontemporal_store(*(const u32x4*)(base + p.src[pair] * p.page_bytes + at), (u32x4*)(base + p.dst[pair] * p.page_bytes + at));
}

// ---- launches ---------------------------------------------------------------------------------------------------------
// Keys a workgroup takes: long chunks keep its start and its join small beside the keys, but at the table's width there
// should be workgroups for four rounds of the chip's 256 CUs.
static int paged_chunk(const vmo_paged_args* a) {
  const int64_t most = (int64_t)a->table_width * a->page_size;
  const int64_t rows = (int64_t)a->batch * a->kv_heads;
  int64_t chunk = (most * rows + 1023) / 1024;
  chunk = (chunk + 127) / 128 * 128;
  return (int)(chunk < 128 ? 128 : chunk > kPagedMaxChunk ? kPagedMaxChunk : chunk);
}

template <bool F16, int D>
static int launch_paged(const PagedParams& p, hipStream_t s) {
  constexpr int RING = kPagedWaves * 2 * 2 * kPagedTile * D * 2, LDS = RING + kPagedMaxChunk * 4 / 8;
  static_assert(1024 + kPagedWaves * 32 * (D + 4) * 4 <= RING + 2048, "the join fits the ring");
  auto kern = paged_attention_kernel<F16, D>;
  if (LDS > 65536 && hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess)
    return set_error(VMO_ERR_LAUNCH, "paged_attention: cannot raise the LDS limit to %d bytes", LDS);
  const dim3 grid((unsigned)((int64_t)p.batch * p.kv_heads * p.chunks), (unsigned)((p.group + 31) / 32));
  hipLaunchKernelGGL(kern, grid, dim3(64 * kPagedWaves), LDS, s, p);
  const int rc = launch_status("paged_attention");
  if (rc != VMO_OK || p.chunks == 1) return rc;
  const int64_t threads = (int64_t)p.batch * p.heads * (D / 4);
  hipLaunchKernelGGL((paged_join_kernel<F16, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, p);
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
  if (!a || a->batch <= 0 || a->heads <= 0 || a->kv_heads <= 0 || a->table_width <= 0 || a->page_size <= 0 || a->d <= 0) return 0;
  const int chunk = vmo::paged_chunk(a);
  const int64_t chunks = ((int64_t)a->table_width * a->page_size + chunk - 1) / chunk;
  return chunks <= 1 ? 0 : (size_t)((int64_t)a->batch * a->heads * chunks * (a->d + 2) * 4);
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
  if (a->pages < 1 || a->table_width < 1 || (int64_t)a->table_width * a->page_size > (1ll << 30) ||
      (int64_t)a->batch * a->heads > (1ll << 30))
    return set_error(VMO_ERR_INVALID, "paged_attention: %d pages, %d page numbers a sequence", a->pages, a->table_width);
  if (!a->table || !a->lengths) return set_error(VMO_ERR_INVALID, "paged_attention: no page table or lengths");
  if (!view_ok(a->k) || !view_ok(a->v) || !a->q.data || !a->o.data || !aligned16(a->q.data) || !aligned16(a->o.data) ||
      a->q.stride_b % 8 || a->q.stride_h % 8 || a->o.stride_b % 8 || a->o.stride_h % 8)
    return set_error(VMO_ERR_INVALID, "paged_attention: tensors need 16-byte aligned rows (strides multiple of 8 elements)");
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
  p.chunk = paged_chunk(a);
  const int64_t chunks = ((int64_t)a->table_width * a->page_size + p.chunk - 1) / p.chunk;
  if ((int64_t)a->batch * a->kv_heads * chunks > (1ll << 30)) return set_error(VMO_ERR_UNSUPPORTED, "paged_attention: batch too large");
  p.chunks = (int)chunks;
  const size_t need = vmo_paged_attention_workspace_size(a);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)))
    return set_error(VMO_ERR_WORKSPACE, "paged_attention: needs %llu workspace bytes, has %llu", (unsigned long long)need,
                     (unsigned long long)(a->workspace ? a->workspace_bytes : 0));
  p.part_o = (float*)a->workspace;
  p.part_ml = p.part_o + (int64_t)a->batch * a->heads * chunks * a->d;
  p.c = a->sm_scale * kLog2e;
  const hipStream_t s = (hipStream_t)stream;
  const bool f16 = a->dtype == VMO_DTYPE_F16;
  if (a->d == 64) return f16 ? launch_paged<true, 64>(p, s) : launch_paged<false, 64>(p, s);
  return f16 ? launch_paged<true, 128>(p, s) : launch_paged<false, 128>(p, s);
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
    CopyParams p{};
    p.k = (char*)a->k; p.v = (char*)a->v; p.page_bytes = a->page_bytes; p.layer_bytes = a->layer_bytes;
    p.pairs = a->pairs - done < kCopyPairs ? a->pairs - done : kCopyPairs;
    p.pieces = (int)pieces;
    for (int i = 0; i < p.pairs; ++i) {
      p.src[i] = a->src[done + i];
      p.dst[i] = a->dst[done + i];
    }
    hipLaunchKernelGGL(paged_copy_kernel, dim3((unsigned)(p.pieces * p.pairs), (unsigned)a->layers, 2), dim3(256), 0,
                       (hipStream_t)stream, p);
    const int rc = launch_status("copy_pages");
    if (rc != VMO_OK) return rc;
  }
  return VMO_OK;
}
