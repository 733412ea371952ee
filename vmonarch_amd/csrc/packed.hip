// Packed causal attention: the C entries (argument checks, launch parameters).
#include "packed.h"

namespace vmo {

static int packed_prepare(const vmo_packed_args* a, bool bwd, const char* what, PackedParams* out) {
  if (!a) return set_error(VMO_ERR_INVALID, "%s: null args", what);
  if (a->dtype != VMO_DTYPE_BF16 && a->dtype != VMO_DTYPE_F16) return set_error(VMO_ERR_INVALID, "%s: dtype %d", what, a->dtype);
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
    return set_error(VMO_ERR_INVALID, "%s: %d query heads over %d key / value heads", what, a->heads, a->kv_heads);
  if (a->n < 0 || a->tq < 0 || a->tk < 0) return set_error(VMO_ERR_INVALID, "%s: negative size", what);
  if (a->n > VMO_PACKED_MAX_SEQUENCES)
    return set_error(VMO_ERR_UNSUPPORTED, "%s: %d sequences (at most %d in one call)", what, a->n, VMO_PACKED_MAX_SEQUENCES);
  if (a->d != 64 && a->d != 128) return set_error(VMO_ERR_UNSUPPORTED, "%s: head dim %d (64 and 128 are built)", what, a->d);
  if (!(a->sm_scale >= 0.f) || a->sm_scale > 3.0e38f)
    return set_error(VMO_ERR_INVALID, "%s: sm_scale must be finite and >= 0", what);
  if (!a->q_offsets || !a->k_offsets) return set_error(VMO_ERR_INVALID, "%s: no offsets", what);
  const vmo_view *rows_q[] = {&a->q, &a->o, &a->grad_o, &a->grad_q}, *rows_k[] = {&a->k, &a->v, &a->grad_k, &a->grad_v};
  // tile copies address up to 8 rows from a lane with a 32-bit byte offset
  const int64_t kMaxRowStride = 1ll << 27;
  for (int i = 0; i < (bwd ? 4 : 2); ++i)
    for (const vmo_view* x : {rows_q[i], rows_k[i]}) {
      if ((x == rows_q[i] ? a->tq : a->tk) == 0) continue;   // (an empty tensor has no address)
      if (!x->data || !aligned16(x->data) || x->stride_h % 8 || x->stride_n % 8 || x->stride_n <= 0)
        return set_error(VMO_ERR_INVALID, "%s: tensors need 16-byte aligned rows (strides multiple of 8 elements)", what);
      if (x->stride_n >= kMaxRowStride) return set_error(VMO_ERR_UNSUPPORTED, "%s: row stride must be below 2^27 elements", what);
    }
  if (a->o_low && !aligned16(a->o_low)) return set_error(VMO_ERR_INVALID, "%s: o_low needs 16-byte alignment", what);
  if (bwd && a->tq > 0 && !a->lse) return set_error(VMO_ERR_INVALID, "%s: needs the forward's lse", what);
  const int64_t tiles = ((int64_t)(a->tq > a->tk ? a->tq : a->tk) + kPackedTile - 1) / kPackedTile + a->n;
  if (a->tq > (1 << 26) || a->tk > (1 << 26) || tiles * a->heads > (1ll << 30))   // (counts of tiles stay within 32 bits)
    return set_error(VMO_ERR_UNSUPPORTED, "%s: too many rows", what);
  PackedParams p{};
  p.q = a->q.data; p.k = a->k.data; p.v = a->v.data; p.o = p.out = a->o.data; p.dO = a->grad_o.data;
  p.dq = a->grad_q.data; p.dk = a->grad_k.data; p.dv = a->grad_v.data;
  p.q_sh = a->q.stride_h; p.q_sn = a->q.stride_n; p.k_sh = a->k.stride_h; p.k_sn = a->k.stride_n;
  p.v_sh = a->v.stride_h; p.v_sn = a->v.stride_n; p.o_sh = a->o.stride_h; p.o_sn = a->o.stride_n;
  p.do_sh = a->grad_o.stride_h; p.do_sn = a->grad_o.stride_n;
  p.dq_sh = a->grad_q.stride_h; p.dq_sn = a->grad_q.stride_n;
  p.dk_sh = a->grad_k.stride_h; p.dk_sn = a->grad_k.stride_n;
  p.dv_sh = a->grad_v.stride_h; p.dv_sn = a->grad_v.stride_n;
  p.o_low = a->o_low;
  p.q_off = a->q_offsets; p.k_off = a->k_offsets;
  p.n = a->n; p.tq = a->tq; p.tk = a->tk; p.heads = a->heads; p.kv_heads = a->kv_heads; p.group = a->heads / a->kv_heads;
  p.causal = a->causal != 0; p.zero_rest = a->zero_rest != 0;
  p.lse = a->lse; p.st_sh = a->stat_stride;
  p.sm_scale = a->sm_scale; p.c = a->sm_scale * kLog2e;
  *out = p;
  return VMO_OK;
}

// Workspaces: the plan of many sequences; the records of split tiles and their parts (the forward's with their m and l, the
// backward's of dk, dv and dq); the backward's -delta and the sums of its shares.
static int64_t part_floats(int d) { return (int64_t)kPackedParts * kPackedTile * d; }
constexpr int64_t kRecordFloats = (int64_t)kPackedParts * 4;
// the tiles of many sequences, as a launch before finds them
static int64_t plan_floats(const vmo_packed_args* a, int rows, int per, int others) {
  return a->n > kPackedFew ? packed_blocks(rows, a->n, per, packed_splits(others)) * 8 : 0;
}
struct FwdLayout { int64_t plan, bytes; };
static FwdLayout fwd_layout(const vmo_packed_args* a) {
  FwdLayout l;
  l.plan = plan_floats(a, a->tq, a->heads, a->tk);
  l.bytes = (l.plan + (packed_splits(a->tk) ? kRecordFloats + part_floats(a->d) + part_floats(2) : 0)) * 4;
  return l;
}
struct BwdLayout { int64_t plan, delta, part_q, part, sum, bytes; int splits; };   // floats of -delta, dq's and dk's parts, dk's shares' sums
static BwdLayout bwd_layout(const vmo_packed_args* a) {
  BwdLayout l;
  l.delta = ((int64_t)a->heads * a->tq + 63) / 64 * 64;
  l.splits = packed_bwd_splits(a->tk, a->kv_heads, a->heads / a->kv_heads);
  l.part_q = packed_splits(a->tk) ? part_floats(a->d) : 0;
  l.part = packed_splits(a->tq) ? part_floats(a->d) : 0;
  l.sum = l.splits > 1 ? (int64_t)l.splits * a->kv_heads * a->tk * a->d : 0;
  const int64_t of_q = plan_floats(a, a->tq, a->heads, a->tk), of_k = plan_floats(a, a->tk, a->kv_heads * l.splits, a->tq);
  l.plan = of_q > of_k ? of_q : of_k;   // (dq's is read before dk's is written)
  l.bytes = (l.plan + 2 * kRecordFloats + l.delta + l.part_q + 2 * l.part + 2 * l.sum) * 4;
  return l;
}
static bool sizes_ok(const vmo_packed_args* a) {
  return a && a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->n >= 0 && a->tq >= 0 && a->tk >= 0 && (a->d == 64 || a->d == 128);
}
static int workspace_check(const vmo_packed_args* a, int64_t need, const char* what) {
  if (need > 0 && (!a->workspace || a->workspace_bytes < (size_t)need || !aligned16(a->workspace)))
    return set_error(VMO_ERR_WORKSPACE, "%s: needs %lld workspace bytes, has %llu", what, (long long)need,
                     (unsigned long long)(a->workspace ? a->workspace_bytes : 0));
  return VMO_OK;
}

}  // namespace vmo

extern "C" size_t vmo_packed_fwd_workspace_size(const vmo_packed_args* a) { return vmo::sizes_ok(a) ? (size_t)vmo::fwd_layout(a).bytes : 0; }

extern "C" int vmo_packed_fwd(const vmo_packed_args* a, void* stream) {
  using namespace vmo;
  clear_error();
  PackedParams p;
  int rc = packed_prepare(a, false, "packed_fwd", &p);
  if (rc != VMO_OK || a->tq == 0) return rc;
  const FwdLayout l = fwd_layout(a);
  rc = workspace_check(a, l.bytes, "packed_fwd");
  if (rc != VMO_OK) return rc;
  if (l.plan > 0) p.plan = (i32x4*)a->workspace;
  if (packed_splits(a->tk)) {
    p.split_least = kPackedSplit;
    p.records = (i32x4*)((float*)a->workspace + l.plan);
    p.part = (float*)p.records + kRecordFloats;
    p.part2 = p.part + part_floats(a->d);
  }
  return packed_fwd_launch(p, a->dtype == VMO_DTYPE_F16, a->d, (hipStream_t)stream);
}

extern "C" size_t vmo_packed_bwd_workspace_size(const vmo_packed_args* a) {
  return vmo::sizes_ok(a) ? (size_t)vmo::bwd_layout(a).bytes : 0;
}

extern "C" int vmo_packed_bwd(const vmo_packed_args* a, void* stream) {
  using namespace vmo;
  clear_error();
  PackedParams p;
  int rc = packed_prepare(a, true, "packed_bwd", &p);
  if (rc != VMO_OK || (a->tq == 0 && a->tk == 0)) return rc;
  const BwdLayout l = bwd_layout(a);
  rc = workspace_check(a, l.bytes, "packed_bwd");
  if (rc != VMO_OK) return rc;
  p.splits = l.splits;
  if (l.plan > 0) p.plan = (i32x4*)a->workspace;
  p.records = (i32x4*)((float*)a->workspace + l.plan);
  p.neg_delta = (float*)p.records + 2 * kRecordFloats;   // (dk's and dv's records, then dq's)
  p.part_q = p.neg_delta + l.delta;
  p.part = p.part_q + l.part_q;
  p.part2 = p.part + l.part;
  p.sum = p.part2 + l.part;
  p.sum2 = p.sum + l.sum;
  return packed_bwd_launch(p, a->dtype == VMO_DTYPE_F16, a->d, (hipStream_t)stream);
}
