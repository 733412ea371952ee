"""Causal attention over packed prompts: sequences of different lengths one behind the other, grouped heads, forward and
backward in HIP (csrc/packed_fwd.hip, csrc/packed_bwd.hip).  No counterpart in the reference, whose attention is neither
causal nor packed."""
import torch

from . import _lib
from .kernel import _recorded


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, k_offsets, sm_scale, causal):
        o, low, lse = _lib.host().packed_fwd(q, k, v, offsets, k_offsets, sm_scale, causal, None, True)
        ctx.save_for_backward(q, k, v, o, low, lse, offsets, k_offsets)
        ctx.sm_scale, ctx.causal = sm_scale, causal
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, low, lse, offsets, k_offsets = ctx.saved_tensors
        return (*_lib.host().packed_bwd(q, k, v, o, low, lse, do.to(q.dtype), offsets, k_offsets, ctx.sm_scale, ctx.causal),
                None, None, None, None)


def packed_attention(q, k, v, offsets, k_offsets=None, sm_scale=None, causal=True, out=None):
    """
    Attention within each of several sequences that lie one behind the other.

    Args:
        q: (H, Tq, D), bf16 or fp16, D 64 or 128; any strides with contiguous features, for example a projection's
            (Tq, H, D) buffer viewed so
        k, v: (Hkv, Tk, D); H is a multiple of Hkv, and key / value head h // (H // Hkv) serves query head h
        offsets: (n + 1,) int32 on the GPU: sequence s has the rows offsets[s] .. offsets[s + 1] - 1 of q
        k_offsets: the same for k and v (default: offsets)
        sm_scale: softmax scale, defaults to 1 / sqrt(D)
        causal: row i of a sequence with nq queries and nk keys sees the keys j <= i + nk - nq (its queries are the last
            tokens); False: all of the sequence's keys
        out: written instead of a new tensor (not with gradients); it may be q's memory, not k's or v's
    Returns:
        o: (H, Tq, D) in q's dtype and memory order; 0 in rows that see no key.  Rows outside every sequence are 0 (with
        `out`: left as they were), and so are gradients there.

    The offsets are read on the GPU when the kernels run: a captured graph replays with what they then hold, and what
    reaches outside the tensors is cut.  They must not fall from one sequence to the next; at most 2048 sequences a call.
    What a row does not see -- later tokens, other sequences, rows behind the last one -- has no part in its result,
    infinities and NaN included.  To capture the backward in a graph, take the gradients with torch.autograd.grad, of leaves
    that no eager graph of another stream still holds (where q, k or v is such a leaf the capture is refused).
    """
    if k_offsets is None:
        k_offsets = offsets
    if sm_scale is None:
        sm_scale = q.shape[-1] ** -0.5
    if _recorded(q, k, v):
        if out is not None:
            raise RuntimeError("vmonarch_amd: packed_attention writes into `out` only where no gradient is recorded")
        return _PackedAttention.apply(q, k, v, offsets, k_offsets, sm_scale, bool(causal))
    return _lib.host().packed_fwd(q, k, v, offsets, k_offsets, sm_scale, bool(causal), out, False)[0]
