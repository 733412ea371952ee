"""packed_attention, forward and backward, against 64 bits within derived bounds (tests/packed_ref.py): lengths from none
and one to several tiles, grouped heads, both memory orders, queries that continue after cached keys, rows without a key,
rows of no sequence, infinities and NaN wherever a row does not look."""
import pytest
import torch

from conftest import hip_library_loaded
from packed_ref import assert_within, reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def offsets(lengths):
    return torch.tensor([0] + list(lengths), device=DEV).cumsum(0).to(torch.int32)


def tensor(g, heads, tokens, D, dtype, layout, scale=1.0):
    x = torch.randn(tokens, heads, D, generator=g) * scale
    x = x.to(dtype).to(DEV)
    return x.transpose(0, 1) if layout == "nhd" else x.transpose(0, 1).contiguous()


CASES = [
    # lengths, key lengths (None: the same), H, Hkv, D, dtype, layout, causal
    ([1], None, 1, 1, 64, "bf16", "hnd", True),
    ([77, 1, 200, 33], None, 8, 2, 64, "bf16", "nhd", True),
    ([128], None, 2, 1, 128, "f16", "nhd", True),
    ([129, 63, 64, 65, 0, 127], None, 4, 4, 128, "bf16", "hnd", True),
    ([500, 3], None, 6, 2, 128, "bf16", "nhd", True),
    ([1000], None, 3, 1, 64, "f16", "nhd", True),
    ([700, 31], None, 12, 3, 128, "f16", "hnd", True),
    ([40, 7, 130], [168, 7, 900], 4, 2, 128, "bf16", "nhd", True),      # after cached keys
    ([40, 300, 5, 6], [0, 100, 1, 5], 2, 1, 64, "bf16", "nhd", True),   # rows that see no key
    ([65, 33, 300], None, 4, 2, 64, "f16", "nhd", False),
    ([40, 129, 9], [200, 65, 0], 2, 2, 128, "bf16", "hnd", False),
    ([0, 0], None, 2, 1, 64, "bf16", "hnd", True),
    ([5] * 70 + [150], None, 2, 1, 64, "f16", "nhd", True),             # more sequences than lanes
    ([3000], None, 2, 1, 64, "f16", "nhd", True),
    ([2000, 1300], None, 2, 2, 128, "bf16", "hnd", False),
    ([7000], None, 1, 1, 64, "bf16", "hnd", True),                      # heavy tiles in parts
    ([6500, 77], [7100, 77], 2, 2, 128, "bf16", "nhd", True),
    ([6200], None, 2, 1, 128, "f16", "hnd", False),
    ([9, 0, 140] * 40 + [4100] + [1] * 9, None, 2, 1, 64, "bf16", "nhd", True),   # both
    ([3, 200] * 50, [130, 0] * 50, 6, 2, 128, "f16", "hnd", True),
    ([1, 0, 17] * 300, None, 3, 3, 64, "f16", "nhd", False),
]


@pytest.mark.parametrize("lengths, k_lengths, H, KVH, D, dtype, layout, causal", CASES)
def test_forward_and_gradients(lengths, k_lengths, H, KVH, D, dtype, layout, causal):
    from vmonarch_amd import packed_attention
    print("packed", lengths[:6], k_lengths, H, KVH, D, dtype, layout, causal, flush=True)
    g = torch.Generator().manual_seed(sum(lengths) + H + D)
    dt, kl = DTYPES[dtype], k_lengths or lengths
    q = tensor(g, H, sum(lengths), D, dt, layout).requires_grad_()
    k, v = (tensor(g, KVH, sum(kl), D, dt, layout).requires_grad_() for _ in range(2))
    grad = tensor(g, H, sum(lengths), D, dt, layout)
    off, koff = offsets(lengths), offsets(kl)
    o = packed_attention(q, k, v, off, None if k_lengths is None else koff, causal=causal)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), grad)
    want = reference(q, k, v, lengths, kl, causal, D ** -0.5, grad)
    for name, got in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert_within(got.detach(), want[name], name)
    with torch.no_grad():
        plain = packed_attention(q, k, v, off, koff, causal=causal)
    assert torch.equal(plain, o)
    for a, b in ((o, q), (dq, q), (dk, k), (dv, v)):
        if b.shape[0] > 1 and b.shape[1] > 1:   # (a single head or row has no memory order to keep)
            assert a.stride() == b.stride()
    again = torch.autograd.grad(packed_attention(q, k, v, off, koff, causal=causal), (q, k, v), grad)
    assert all(torch.equal(a, b) for a, b in zip(again, (dq, dk, dv)))
    assert hip_library_loaded()


def test_what_a_row_does_not_see_has_no_part_in_it():
    """Infinities and NaN in later tokens, in another sequence and behind the last one: the rows before are bit for bit
    those of clean inputs, forward and backward; the rows that do see them are not finite."""
    from vmonarch_amd import packed_attention
    for D, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        print("unseen", D, dtype, flush=True)
        g = torch.Generator().manual_seed(5)
        lengths, H, KVH, T = [150, 200, 90], 4, 2, 460   # rows 440 .. 459 are of no sequence
        q, grad = (tensor(g, H, T, D, dtype, "nhd") for _ in range(2))
        k, v = (tensor(g, KVH, T, D, dtype, "nhd") for _ in range(2))
        off = offsets(lengths)

        def run(*x):
            leaves = [t.clone().requires_grad_() for t in x[:3]]
            o = packed_attention(*leaves, off)
            return [o.detach(), *torch.autograd.grad(o, leaves, x[3])]

        clean = run(q, k, v, grad)
        for t in clean:
            assert not bool(t[:, 440:].any()), "rows of no sequence are zeros"
        for at in (250, 349, 150, 288):                  # tokens of the second sequence
            for bad in (float("nan"), float("inf"), float("-inf")):
                x = [t.clone() for t in (q, k, v, grad)]
                for t in x:
                    t[:, at] = bad
                    t[:, 440:] = float("nan")
                dirty = run(*x)
                for a, b in zip(clean, dirty):
                    for rows in (slice(0, 150), slice(350, 460)):      # the other sequences
                        assert torch.equal(a[:, rows], b[:, rows])
                for i in (0, 1):                                       # o, dq: rows before the token
                    assert torch.equal(clean[i][:, 150:at], dirty[i][:, 150:at])
                    assert not torch.isfinite(dirty[i][:, at:350].float()).any()
                for i in (2, 3):                                       # dk, dv: keys behind it get nothing from its row
                    if at < 349:
                        assert dirty[i].shape == clean[i].shape
        # a token whose row alone is bad (its query and upstream gradient): keys behind it are as before
        x = [t.clone() for t in (q, k, v, grad)]
        x[0][:, 250] = x[3][:, 250] = float("nan")
        dirty = run(*x)
        for i in (2, 3):
            assert torch.equal(clean[i][:, 251:], dirty[i][:, 251:]) and torch.equal(clean[i][:, :150], dirty[i][:, :150])
            assert torch.isnan(dirty[i][:, 150:251].float()).all()
        # a value alone: the rows that see it take it, column by column
        x = [t.clone() for t in (q, k, v, grad)]
        x[2][:, 250, 5] = float("inf")
        o = run(*x)[0]
        assert torch.equal(o[:, :250], clean[0][:, :250]) and bool((o[:, 250:350, 5] == float("inf")).all())
        keep = [c for c in range(D) if c != 5]
        assert torch.equal(o[:, :, keep], clean[0][:, :, keep])


@pytest.mark.parametrize("scale, dtype", [(8.0, torch.bfloat16), (8.0, torch.float16), (40.0, torch.bfloat16)])
def test_sharp_rows(scale, dtype):
    """Logits whose maximum keeps growing along the row: the reference point of the weights moves again and again."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(9)
    n, D = 700, 64
    q = torch.ones(2, n, D).to(dtype).to(DEV)
    ramp = torch.linspace(-1, 1, n)[None, :, None] * scale / D ** 0.5
    k = (ramp + 0.01 * torch.randn(2, n, D, generator=g)).to(dtype).to(DEV)
    v = torch.randn(2, n, D, generator=g).to(dtype).to(DEV)
    for keys in (k, k.flip(1)):
        o = packed_attention(q, keys, v, offsets([n]))
        s = (q.double() @ keys.double().transpose(1, 2).contiguous() * D ** -0.5)
        p = torch.softmax(s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device=DEV).tril(), float("-inf")), -1)
        want, a = p @ v.double(), p @ v.double().abs()
        u = torch.finfo(dtype).eps / 2
        # logits up to 2^9 in size: 2^-24 of that in the exponent, twice (s and s c - m); fp16 weights' floor as elsewhere
        bound = u * a + u * want.abs() + 2 ** -13 * a + (n * 2.0 ** -25 * 5 if dtype == torch.float16 else 0)
        assert bool(((o.double() - want).abs() <= bound).all())


def test_rows_of_no_sequence_and_out():
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(3)
    q, k, v = tensor(g, 4, 400, 64, torch.bfloat16, "nhd"), *(tensor(g, 2, 300, 64, torch.bfloat16, "nhd") for _ in range(2))
    off, koff = torch.tensor([10, 60, 130], device=DEV, dtype=torch.int32), torch.tensor([5, 80, 250], device=DEV, dtype=torch.int32)
    fresh = packed_attention(q, k, v, off, koff)
    assert not bool(fresh[:, :10].any()) and not bool(fresh[:, 130:].any())
    alone = packed_attention(q[:, 10:130], k[:, 5:250], v[:, 5:250], off - 10, koff - 5)
    assert torch.equal(fresh[:, 10:130], alone)
    out = torch.full((400, 4, 64), 7.0, device=DEV, dtype=torch.bfloat16).transpose(0, 1)
    assert packed_attention(q, k, v, off, koff, out=out) is out
    assert torch.equal(out[:, 10:130], alone) and bool((out[:, :10] == 7).all()) and bool((out[:, 130:] == 7).all())
    own = q.clone()
    packed_attention(own, k, v, off, koff, out=own)      # in q's own memory
    assert torch.equal(own[:, 10:130], alone) and torch.equal(own[:, 130:], q[:, 130:])
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*leaves, off, koff).sum(), leaves)   # (an expanded upstream gradient)
    for t, (a, b) in zip(grads, ((10, 130), (5, 250), (5, 250))):
        assert not bool(t[:, :a].any()) and not bool(t[:, b:].any()) and torch.isfinite(t.float()).all()


def test_many_sequences_with_rows_outside():
    """More sequences than a workgroup looks through itself, rows before the first and behind the last one: zeros there, the
    rest as without them."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(8)
    lengths, before, behind = [17, 0, 130] * 40 + [1900], 300, 500
    n = sum(lengths)
    q, k, v, grad = (tensor(g, h, before + n + behind, 64, torch.bfloat16, "nhd") for h in (4, 2, 2, 4))
    inner = [t[:, before:before + n] for t in (q, k, v, grad)]
    want_leaves = [t.detach().requires_grad_() for t in inner[:3]]
    want = packed_attention(*want_leaves, offsets(lengths))
    want_grads = torch.autograd.grad(want, want_leaves, inner[3])
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = packed_attention(*leaves, offsets(lengths) + before)
    for got, x in zip((o, *torch.autograd.grad(o, leaves, grad)), (want, *want_grads)):
        assert torch.equal(got[:, before:before + n], x)
        assert not bool(got[:, :before].any()) and not bool(got[:, before + n:].any())


def test_offsets_that_lead_outside_are_cut():
    """Nothing outside the tensors is read or written, whatever the offsets hold: the tensors are the middle of larger
    buffers whose edges would show it."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(4)
    big = [torch.full((2, 600, 64), float("nan"), device=DEV, dtype=torch.bfloat16) for _ in range(4)]
    q, k, v, out = (b[:, 200:400] for b in big)
    for t in (q, k, v):
        t.copy_(torch.randn(2, 200, 64, generator=g).to(t.dtype))
    cut = packed_attention(q, k, v, offsets([200]))
    for off in ([-50, 900], [0, 1 << 30], [-(1 << 31), (1 << 31) - 1]):
        packed_attention(q, k, v, torch.tensor(off, device=DEV, dtype=torch.int32), out=out)
        assert torch.equal(out, cut)
        for b in big:
            assert torch.isnan(b[:, :200].float()).all() and torch.isnan(b[:, 400:].float()).all()
    packed_attention(q, k, v, torch.tensor([0, 150, 100, 300, 20], device=DEV, dtype=torch.int32), out=out)   # falling
    for b in big:
        assert torch.isnan(b[:, :200].float()).all() and torch.isnan(b[:, 400:].float()).all()


@pytest.mark.parametrize("more", [0, 100])   # sequences of no token behind them
def test_replays_with_other_lengths_from_a_graph(more):
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(6)
    q, k, v = tensor(g, 4, 500, 128, torch.bfloat16, "nhd"), *(tensor(g, 2, 500, 128, torch.bfloat16, "nhd") for _ in range(2))
    grad, off = tensor(g, 4, 500, 128, torch.bfloat16, "nhd"), offsets([100, 300, 50] + [0] * more)
    leaves = [t.requires_grad_() for t in (q, k, v)]

    def step():
        o = packed_attention(*leaves, off)
        return [o.detach(), *torch.autograd.grad(o, leaves, grad)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lengths in ([100, 300, 50], [1, 2, 3], [0, 499, 0], [250, 125, 125]):
        off.copy_(offsets(lengths + [0] * more))
        with torch.no_grad():
            q.copy_(q.roll(1, 1))
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), lengths
        _ = step()


def test_gradient_against_differences():
    """The directional derivative from 64-bit function values of the plain formula (the kernels' own roundings are far
    above a difference's step): dq, dk and dv give it within what their roundings allow."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(8)
    lengths, D = [70, 40], 64
    q, k, v = (tensor(g, h, 110, D, torch.float16, "hnd").requires_grad_() for h in (4, 2, 2))
    grad = tensor(g, 4, 110, D, torch.float16, "hnd")
    got = torch.autograd.grad(packed_attention(q, k, v, offsets(lengths)), (q, k, v), grad)
    want = reference(q, k, v, lengths, lengths, True, D ** -0.5, grad)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = [t.detach().double() for t in (q, k, v)]
        d = torch.randn(x[i].shape, generator=g).double().to(DEV)

        def value(step):
            y = [t + step * d if j == i else t for j, t in enumerate(x)]
            return float((reference(*y, lengths, lengths, True, D ** -0.5)["o"][0] * grad.double()).sum())

        diff = (value(1e-4) - value(-1e-4)) / 2e-4
        ours, allowed = float((got[i].double() * d).sum()), float((want[name][1] * d.abs()).sum())
        assert abs(ours - diff) <= allowed + 1e-5 * abs(diff)


def test_capture_beside_a_live_eager_graph_is_refused():
    """The leaf's gradient node belongs to the eager graph's stream: a captured backward would end the process."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(7)
    leaves = [tensor(g, h, 50, 64, torch.bfloat16, "hnd").requires_grad_() for h in (2, 1, 1)]
    grad, off = tensor(g, 2, 50, 64, torch.bfloat16, "hnd"), offsets([50])
    alive = packed_attention(*leaves, off)
    torch.cuda.synchronize()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="another stream"):
            packed_attention(*leaves, off)
        with torch.no_grad():
            o = packed_attention(*leaves, off)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, alive) and float(x[0]) == 1
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = packed_attention(*leaves, off)
        got = torch.autograd.grad(o, leaves, grad)
    del o
    graph.replay()
    torch.cuda.synchronize()
    want = torch.autograd.grad(packed_attention(*leaves, off), leaves, grad)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_on_another_stream():
    """Work and allocations on the stream that is current; the result of a call on one stream used on another after a wait."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(11)
    q, k, v = (tensor(g, h, 3000, 64, torch.bfloat16, "nhd") for h in (2, 1, 1))
    off = offsets([2000, 1000])
    want = packed_attention(q, k, v, off)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams * 2:                       # two calls at once, their workspaces apart
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(packed_attention(q, k, v, off))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_no_keys_and_no_sequences():
    from vmonarch_amd import packed_attention
    q = torch.ones(2, 30, 64, device=DEV, dtype=torch.bfloat16).requires_grad_()
    k = torch.ones(1, 0, 64, device=DEV, dtype=torch.bfloat16).requires_grad_()
    none = torch.zeros(2, device=DEV, dtype=torch.int32)
    for off, koff in ((offsets([30]), none), (none[:1], none[:1])):
        o = packed_attention(q, k, k, off, koff)
        assert not bool(o.any())
        dq, dk = torch.autograd.grad(o.sum(), (q, k))
        assert not bool(dq.any()) and dk.shape == k.shape
    kk = torch.ones(1, 40, 64, device=DEV, dtype=torch.bfloat16).requires_grad_()
    e = torch.ones(2, 0, 64, device=DEV, dtype=torch.bfloat16).requires_grad_()
    o = packed_attention(e, kk, kk, none, offsets([40]))
    assert o.shape == e.shape and not bool(torch.autograd.grad(o.sum(), kk)[0].any())
    assert not bool(torch.autograd.grad(packed_attention(q, kk, kk, none[:1], none[:1]).sum(), kk)[0].any())


def test_inputs_that_the_kernels_cannot_read_in_place():
    """Features apart, rows off 16 bytes, heads or rows expanded: copied, with the results of contiguous tensors."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(21)
    base = torch.randn(4, 90, 128, generator=g).bfloat16().to(DEV)
    off = offsets([90])
    apart = base[:, :, ::2]
    odd = torch.empty(4 * 90 * 64 + 3, device=DEV, dtype=torch.bfloat16)[3:].view(4, 90, 64).copy_(apart)
    heads, rows = base[:1, :, :64].expand(4, 90, 64), base[:, :1, :64].expand(4, 90, 64)
    for q in (apart, odd, heads, rows):
        for k in (apart, odd, heads, rows):
            leaves = [t.detach().requires_grad_() for t in (q, k, odd)]
            plain = [t.detach().contiguous().clone().requires_grad_() for t in (q, k, odd)]
            o, want = (packed_attention(*x, off) for x in (leaves, plain))
            assert torch.equal(o, want)
            for a, b in zip(torch.autograd.grad(o.sum(), leaves), torch.autograd.grad(want.sum(), plain)):
                assert torch.equal(a, b)


def test_a_buffer_that_is_written_counts_as_changed():
    from vmonarch_amd import packed_attention
    q = torch.ones(1, 10, 64, device=DEV, dtype=torch.bfloat16)
    out = torch.ones_like(q)
    y = (out * torch.ones_like(q).requires_grad_()).sum()
    packed_attention(q, q, q, offsets([10]), out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_rows_far_apart():
    """Tokens 2 MB apart, so a sequence's rows reach 6 GB from its first: bit for bit as rows beside each other."""
    from vmonarch_amd import packed_attention
    g = torch.Generator().manual_seed(23)
    T, D = 3000, 64
    buf = torch.empty(T, 1 << 20, device=DEV, dtype=torch.bfloat16)
    near = [tensor(g, h, T, D, torch.bfloat16, "nhd") for h in (2, 1, 1, 2)]
    far, at = [], 0
    for t in near:
        far.append(buf[:, at:at + t.shape[0] * D].view(T, t.shape[0], D).transpose(0, 1).copy_(t))
        at += t.shape[0] * D
    out = buf[:, at:at + 2 * D].view(T, 2, D).transpose(0, 1)
    off = offsets([40, T - 40])
    leaves = [[t.detach().requires_grad_() for t in x[:3]] for x in (near, far)]
    want, got = (packed_attention(*x, off) for x in leaves)
    assert torch.equal(want, got)
    for a, b in zip(torch.autograd.grad(want, leaves[0], near[3]), torch.autograd.grad(got, leaves[1], far[3])):
        assert torch.equal(a, b)
    with torch.no_grad():
        packed_attention(*far[:3], off, out=out)
    assert torch.equal(want, out)
