"""The paged cache: attention of new tokens against 64 bits within derived bounds (tests/packed_ref.py: a row that sees all
keys), rows into their pages, pages copied, and a run of them together with packed_attention."""
import pytest
import torch

from conftest import hip_library_loaded
from packed_ref import FP32, assert_within, half_step, one, reference, sees

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def cache(g, lengths, KVH, D, page, dtype, spare=3, order="phnd"):
    """Shuffled pages; every place that no token has holds NaN, unused places of the table -1."""
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    perm = torch.randperm(pages, generator=g).tolist()
    width = max(need + [1]) + 1
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    k, v = (torch.full((pages, KVH, page, D), float("nan")) for _ in range(2))
    rows = []
    for b, n in enumerate(lengths):
        mine = [perm.pop() for _ in range(need[b])]
        table[b, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        kb, vb = (torch.randn(KVH, n, D, generator=g).to(dtype) for _ in range(2))
        rows.append((kb.to(DEV), vb.to(DEV)))
        for i, p in enumerate(mine):
            for t, x in ((k, kb), (v, vb)):
                part = x[:, i * page:(i + 1) * page]
                t[p, :, :part.shape[1]] = part.float()
    k, v = (t.to(dtype).to(DEV) for t in (k, v))
    if order == "pnhd":   # token by token, the heads of one beside each other
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    return k, v, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), rows


def want_one(q, rows, sm, dtype):
    """(value, bound) of one sequence's (H, D) answer."""
    k, v = rows
    group, u = q.shape[0] // k.shape[0], half_step(dtype)
    got = [one(q[h:h + 1].double(), k[h // group].double(), v[h // group].double(), None,
               sees(1, k.shape[1], False, DEV), sm, dtype)["o"] for h in range(q.shape[0])]
    value, bound = (torch.cat([x[i] for x in got]) for i in (0, 1))
    return value, 1.02 * bound + (u + FP32) * value.abs() + 1e-30


CASES = [
    # lengths, H, Hkv, D, page, dtype, order
    ([1], 1, 1, 64, 8, "bf16", "phnd"),
    ([5, 0, 33, 16, 17], 8, 2, 128, 16, "bf16", "phnd"),
    ([300, 129, 1000], 6, 2, 64, 32, "f16", "pnhd"),
    ([2500, 1, 640], 12, 3, 128, 16, "f16", "phnd"),
    ([700], 40, 1, 64, 64, "bf16", "phnd"),          # more query heads a key / value head than the product has columns
    ([9000, 4100], 4, 4, 128, 1024, "bf16", "pnhd"),
    ([128, 256, 127, 129], 32, 1, 128, 8, "f16", "phnd"),
]


@pytest.mark.parametrize("lengths, H, KVH, D, page, dtype, order", CASES)
def test_attention_of_new_tokens(lengths, H, KVH, D, page, dtype, order):
    from vmonarch_amd import paged_attention
    print("paged", lengths, H, KVH, D, page, dtype, order, flush=True)
    g = torch.Generator().manual_seed(sum(lengths) + H)
    dt = DTYPES[dtype]
    k, v, table, lens, rows = cache(g, lengths, KVH, D, page, dt, order=order)
    q = torch.randn(len(lengths), H, D, generator=g).to(dt).to(DEV)
    o = paged_attention(q, k, v, table, lens)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not bool(o[b].any())
        else:
            assert_within(o[b], want_one(q[b], rows[b], D ** -0.5, dt), f"sequence {b}")
    # a wider table (more workgroups that find nothing, other pieces), a strided q and out, a given scale
    wide = torch.cat([table, torch.full((len(lengths), 300), -1, dtype=torch.int32, device=DEV)], 1)
    qs = torch.randn(H, len(lengths), D, device=DEV, dtype=dt).transpose(0, 1).copy_(q)
    out = torch.empty(len(lengths), H, 2 * D, device=DEV, dtype=dt)[..., :D]
    assert paged_attention(qs, k, v, wide, lens, sm_scale=0.3, out=out) is out
    for b, n in enumerate(lengths):
        if n:
            assert_within(out[b], want_one(q[b], rows[b], 0.3, dt), f"sequence {b}, wide table")
    assert torch.equal(o, paged_attention(q, k, v, table, lens))
    assert hip_library_loaded()


def test_pages_and_lengths_that_lead_outside():
    """Such a sequence's rows are NaN, the others as they were."""
    from vmonarch_amd import paged_attention
    g = torch.Generator().manual_seed(2)
    k, v, table, lens, _ = cache(g, [40, 900, 100, 20], 2, 64, 16, torch.bfloat16)
    q = torch.randn(4, 4, 64, generator=g).bfloat16().to(DEV)
    good = paged_attention(q, k, v, table, lens)
    for page in (-1, k.shape[0], 1 << 30, -(1 << 31)):
        bad = table.clone()
        bad[1, 40] = page
        o = paged_attention(q, k, v, bad, lens)
        assert torch.isnan(o[1].float()).all() and torch.equal(o[[0, 2, 3]], good[[0, 2, 3]])
    for n in (table.shape[1] * 16 + 1, (1 << 31) - 1):
        bad = lens.clone()
        bad[2] = n
        o = paged_attention(q, k, v, table, bad)
        assert torch.isnan(o[2].float()).all() and torch.equal(o[[0, 1, 3]], good[[0, 1, 3]])
    bad = lens.clone()
    bad[3] = -5
    assert not bool(paged_attention(q, k, v, table, bad)[3].any())


@pytest.mark.parametrize("new, past, KVH, D, page, order", [
    ([1, 1, 1], [0, 15, 16], 2, 64, 16, "phnd"), ([40, 1, 0, 100], [3, 16, 5, 0], 3, 128, 32, "pnhd"), ([9], [0], 1, 64, 8, "phnd")])
def test_append(new, past, KVH, D, page, order):
    from vmonarch_amd import append_pages
    g = torch.Generator().manual_seed(sum(new))
    total = [a + b for a, b in zip(new, past)]
    k, v, table, lens, rows = cache(g, total, KVH, D, page, torch.float16, order=order)
    want_k, want_v = k.clone(), v.clone()
    T = sum(new)
    kn, vn = (torch.randn(T + 4, KVH, D, generator=g).half().to(DEV).transpose(0, 1) for _ in range(2))   # 4 rows of no sequence
    at = 0
    for b, n in enumerate(new):
        for i in range(n):
            t = past[b] + i
            p = int(table[b, t // page])
            want_k[p, :, t % page], want_v[p, :, t % page] = kn[:, at], vn[:, at]
            at += 1
    off = torch.tensor([0] + new, device=DEV).cumsum(0).to(torch.int32)
    append_pages(kn, vn, k, v, table, lens, off)
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))   # noqa: E731  (NaN among them)
    assert same(k, want_k) and same(v, want_v)
    if all(n == 1 for n in new):
        k2, v2 = k.clone(), v.clone()
        append_pages(kn[:, :T], vn[:, :T], k2, v2, table, lens)
        assert same(k2, want_k) and same(v2, want_v)
    # pages and places outside are left out
    before = k.clone()
    append_pages(kn, vn, k, v, torch.full_like(table, k.shape[0]), lens, off)
    append_pages(kn, vn, k, v, torch.full_like(table, -1), lens, off)
    append_pages(kn, vn, k, v, table, torch.full_like(lens, (1 << 31) - 1), off)
    append_pages(kn, vn, k, v, table, torch.full_like(lens, -7), off)
    append_pages(kn, vn, k, v, table, lens, torch.full_like(off, -1))
    assert same(k, before)


@pytest.mark.parametrize("layers, pages, moves", [(None, 9, 4), (3, 40, 17), (1, 1100, 500)])
def test_copy(layers, pages, moves):
    from vmonarch_amd import copy_pages
    g = torch.Generator().manual_seed(moves)
    shape = (pages, 2, 8, 64) if layers is None else (layers, pages, 2, 8, 64)
    k, v = (torch.randn(shape, generator=g).bfloat16().to(DEV) for _ in range(2))
    perm = torch.randperm(pages, generator=g).tolist()
    src, dst = perm[:moves], perm[moves:2 * moves]
    src[1] = src[0]                                       # one page to two places
    want = [t.clone() for t in (k, v)]
    for t in want:
        x = t.transpose(0, 1) if layers is not None else t
        x[dst] = x[src]
    copy_pages(k, v, src, dst)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    copy_pages(k, v, [], [])
    assert torch.equal(k, want[0])


def test_copies_that_would_meet_are_refused():
    from vmonarch_amd import copy_pages
    k = torch.zeros(8, 1, 8, 64, device=DEV, dtype=torch.bfloat16)
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [1, 3]), ([0, 2], [2, 3]), ([0], [0]), ([2, 0], [3, 2])):
        with pytest.raises(RuntimeError, match="written twice"):
            copy_pages(k, k.clone(), src, dst)
    for src, dst in (([0], [8]), ([-1], [2]), ([1 << 40], [2])):
        with pytest.raises(ValueError, match="of 8"):
            copy_pages(k, k.clone(), src, dst)


def test_prompts_then_tokens_over_a_cache():
    """Prompts through packed_attention and into the cache; two sequences fork; every sequence's tokens then come one by
    one over two layers, a sequence ends, the cache is compacted: each step's answers are those of the whole sequence."""
    from vmonarch_amd import PagedKVCache, append_pages, packed_attention, paged_attention
    g = torch.Generator().manual_seed(12)
    H, KVH, D, page, L = 6, 2, 64, 16, 2
    dt, sm = torch.bfloat16, 64 ** -0.5
    kv = PagedKVCache(pages=64, page=page, heads=KVH, head_dim=D, layers=L, dtype=dt, device=DEV)
    prompts = [70, 16, 1]
    ids = [kv.open() for _ in prompts]
    table, lens = kv.grow(ids, prompts)
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt).to(DEV)   # noqa: E731
    history = {}
    off = torch.tensor([0] + prompts, device=DEV).cumsum(0).to(torch.int32)
    for i in range(L):
        q, k, v = rnd(sum(prompts), H, D).transpose(0, 1), *(rnd(sum(prompts), KVH, D).transpose(0, 1) for _ in range(2))
        o = packed_attention(q, k, v, off)
        assert_within(o, reference(q, k, v, prompts, prompts, True, sm)["o"], "prompts")
        append_pages(k, v, *kv.layer(i), table, lens, off)
        a = 0
        for s, n in zip(ids, prompts):
            history[s, i] = (k[:, a:a + n].clone(), v[:, a:a + n].clone())
            a += n
    for parent in (ids[0], ids[1]):                     # one with an unfilled last page, one with a full one
        child = kv.fork(parent)
        ids.append(child)
        for i in range(L):
            history[child, i] = history[parent, i]
    for step in range(20):
        if step == 7:
            kv.free(ids.pop(1))
        if step == 9:
            assert kv.compact() > 0
            assert sorted(p for s in ids for p in set(kv.pages_of(s)))[-1] < 64 - kv.free_pages
        table, lens = kv.grow(ids)
        for i in range(L):
            k, v = (rnd(len(ids), KVH, D).transpose(0, 1) for _ in range(2))
            append_pages(k, v, *kv.layer(i), table, lens)
            q = rnd(len(ids), H, D)
            o = paged_attention(q, *kv.layer(i), table, lens)
            for b, s in enumerate(ids):
                history[s, i] = tuple(torch.cat([old, new[:, b:b + 1]], 1) for old, new in zip(history[s, i], (k, v)))
                assert_within(o[b], want_one(q[b], history[s, i], sm, dt), f"step {step}, sequence {s}, layer {i}")
    for s in ids:
        kv.free(s)
    assert kv.free_pages == 64


def test_token_steps_replay_from_a_graph():
    """Append and attend captured once; table and lengths change between the replays."""
    from vmonarch_amd import append_pages, paged_attention
    g = torch.Generator().manual_seed(13)
    k, v, table, lens, _ = cache(g, [40, 1000, 100], 2, 128, 16, torch.bfloat16)
    wide = torch.cat([table, table], 1).contiguous()
    q, kn, vn = (torch.randn(*s, generator=g).bfloat16().to(DEV) for s in ((3, 8, 128), (2, 3, 128), (2, 3, 128)))

    def step(kp, vp):
        append_pages(kn, vn, kp, vp, wide, lens)
        return paged_attention(q, kp, vp, wide, lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(k.clone(), v.clone())
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(k, v)
    for change in range(4):
        lens.sub_(torch.tensor([1, 200, 0], device=DEV, dtype=torch.int32))
        kn.copy_(kn.roll(1, 1))
        k2, v2 = k.clone(), v.clone()
        want = step(k2, v2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(k.view(torch.int16), k2.view(torch.int16)), change
        _ = step(k2, v2)


def test_a_cache_beyond_32_bits_of_bytes():
    """Pages behind the first 4 GiB: written, copied and read where they are."""
    from vmonarch_amd import append_pages, copy_pages, paged_attention
    g = torch.Generator().manual_seed(31)
    pages, KVH, page, D = 150000, 8, 16, 128            # 32 KiB a page, 4.9 GB a tensor
    k, v = (torch.empty(pages, KVH, page, D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    table = torch.tensor([[pages - 1, 3, pages - 7]], device=DEV, dtype=torch.int32)
    n = 41
    kn, vn = (torch.randn(n, KVH, D, generator=g).bfloat16().to(DEV).transpose(0, 1) for _ in range(2))
    lens, off = torch.tensor([n], device=DEV, dtype=torch.int32), torch.tensor([0, n], device=DEV, dtype=torch.int32)
    append_pages(kn, vn, k, v, table, lens, off)
    assert torch.equal(k[pages - 1], kn[:, :16]) and torch.equal(v[pages - 7, :, :9], vn[:, 32:])
    q = torch.randn(1, 16, D, generator=g).bfloat16().to(DEV)
    o = paged_attention(q, k, v, table, lens)
    assert_within(o[0], want_one(q[0], (kn, vn), D ** -0.5, torch.bfloat16), "high pages")
    copy_pages(k, v, [pages - 1, pages - 7], [pages - 2, 5])
    assert torch.equal(k[pages - 2], kn[:, :16])
    assert torch.equal(paged_attention(q, k, v, table.new_tensor([[pages - 2, 3, 5]]), lens), o)


def test_many_sequences():
    """More sequences than a wave has lanes, many of them without tokens: each row whole or in parts."""
    from vmonarch_amd import paged_attention
    g = torch.Generator().manual_seed(33)
    lengths = [(7 * i) % 50 if i % 3 else 0 for i in range(700)] + [3000]
    k, v, table, lens, rows = cache(g, lengths, 1, 64, 16, torch.float16)
    q = torch.randn(len(lengths), 4, 64, generator=g).half().to(DEV)
    o = paged_attention(q, k, v, table, lens)
    for b in list(range(0, 700, 13)) + [700]:
        if lengths[b] == 0:
            assert not bool(o[b].any())
        else:
            assert_within(o[b], want_one(q[b], rows[b], 64 ** -0.5, torch.float16), f"sequence {b}")
    assert not bool(o[[i for i, n in enumerate(lengths) if n == 0]].any())


def test_values_that_are_not_finite_stay_in_their_sequence():
    from vmonarch_amd import paged_attention
    g = torch.Generator().manual_seed(35)
    k, v, table, lens, _ = cache(g, [50, 60, 70], 2, 64, 16, torch.bfloat16)
    q = torch.randn(3, 4, 64, generator=g).bfloat16().to(DEV)
    good = paged_attention(q, k, v, table, lens)
    v[int(table[1, 2]), 0, 3, 7] = float("inf")
    o = paged_attention(q, k, v, table, lens)
    assert torch.equal(o[[0, 2]], good[[0, 2]]) and torch.equal(o[1, 2:], good[1, 2:])
    assert bool((o[1, :2, 7] == float("inf")).all()) and torch.equal(o[1, :2, :7], good[1, :2, :7])
    q[1] = float("nan")
    o = paged_attention(q, k, v, table, lens)
    assert torch.equal(o[[0, 2]], good[[0, 2]]) and torch.isnan(o[1].float()).all()


@pytest.mark.parametrize("dtype, scale", [(torch.float16, 8.0), (torch.bfloat16, 40.0)])
def test_sharp_rows(dtype, scale):
    """Logits that keep growing (and falling) along the cache: the reference point moves in every wave's share."""
    from vmonarch_amd import paged_attention
    g = torch.Generator().manual_seed(37)
    n, D, page = 3000, 64, 16
    ramp = torch.linspace(-1, 1, n)[:, None] * scale / D ** 0.5
    u = torch.finfo(dtype).eps / 2
    for sign in (1, -1):
        kd = (sign * ramp + 0.01 * torch.randn(n, D, generator=g)).to(dtype)
        vd = torch.randn(n, D, generator=g).to(dtype)
        pages = -(-n // page)
        k, v = (torch.zeros(pages * page, D, dtype=dtype).index_copy_(0, torch.arange(n), t).view(pages, 1, page, D).to(DEV) for t in (kd, vd))
        q = torch.ones(1, 2, D, device=DEV, dtype=dtype)
        o = paged_attention(q, k, v, torch.arange(pages, device=DEV, dtype=torch.int32)[None], torch.tensor([n], device=DEV, dtype=torch.int32))
        p = torch.softmax(q[0].double() @ kd.double().to(DEV).t().contiguous() * D ** -0.5, -1)
        want, a = p @ vd.double().to(DEV), p @ vd.double().to(DEV).abs()
        # (as for whole prompts: logits up to 2^9, fp16 weights' floor)
        bound = u * a + u * want.abs() + 2 ** -13 * a + (n * 2.0 ** -25 * 5 if dtype == torch.float16 else 0)
        assert bool(((o[0].double() - want).abs() <= bound).all())


def test_calls_at_once_on_streams_of_their_own():
    """Two threads, each with its stream, its cache and its steps: results as one after the other; out may be q's memory."""
    import threading
    from vmonarch_amd import append_pages, copy_pages, paged_attention

    def steps(seed, stream, results):
        with torch.no_grad(), torch.cuda.stream(stream):
            g = torch.Generator().manual_seed(seed)
            k, v, table, lens, _ = cache(g, [100 * seed, 3000, 5], 2, 128, 16, torch.bfloat16)
            width = torch.full((3, 2), k.shape[0] - 1, dtype=torch.int32, device=DEV)
            for i in range(10):
                kn, vn, q = (torch.randn(n, 3, 128, generator=g).bfloat16().to(DEV) for n in (2, 2, 8))
                q = q.transpose(0, 1).contiguous()
                lens = torch.clamp(lens + 1, max=3008)
                append_pages(kn, vn, k, v, torch.cat([table, width], 1), lens)
                copy_pages(k, v, [0], [k.shape[0] - 2])
                assert paged_attention(q, k, v, torch.cat([table, width], 1), lens, out=q) is q
                results.append(q)
            stream.synchronize()

    alone, beside = [[], []], [[], []]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for j in range(2):
        steps(j + 2, streams[j], alone[j])
    threads = [threading.Thread(target=steps, args=(j + 2, streams[j], beside[j])) for j in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(alone, beside):
        assert len(b) == 10
        for x, y in zip(a, b):
            assert not bool(torch.isnan(x.float()).all()) and torch.equal(torch.nan_to_num(x), torch.nan_to_num(y))


@pytest.mark.parametrize("page", [8, 512])
def test_scale_zero_is_the_mean(page):
    from vmonarch_amd import paged_attention
    g = torch.Generator().manual_seed(41)
    k, v, table, lens, rows = cache(g, [77, 1, 2000], 2, 64, page, torch.float16)
    q = torch.randn(3, 6, 64, generator=g).half().to(DEV)
    o = paged_attention(q, k, v, table, lens, sm_scale=0.0)
    for b in range(3):
        assert_within(o[b], want_one(q[b], rows[b], 0.0, torch.float16), f"sequence {b}")


def test_several_new_tokens_of_one_sequence():
    """A row each, all with the sequence's pages and lengths that grow: the prompt's attention after cached keys."""
    from vmonarch_amd import paged_attention
    g = torch.Generator().manual_seed(43)
    past, new, H, D = 500, 70, 8, 128
    k, v, table, lens, rows = cache(g, [past + new], 2, D, 16, torch.bfloat16)
    q = torch.randn(new, H, D, generator=g).bfloat16().to(DEV)
    lengths = torch.arange(past + 1, past + new + 1, device=DEV, dtype=torch.int32)
    o = paged_attention(q, k, v, table.expand(new, -1), lengths)
    for i in range(0, new, 3):
        n = past + i + 1
        assert_within(o[i], want_one(q[i], tuple(x[:, :n] for x in rows[0]), D ** -0.5, torch.bfloat16), f"token {i}")


def test_in_inference_mode():
    """A cache made outside or inside of it, and weights that would record gradients elsewhere."""
    from vmonarch_amd import PagedKVCache, append_pages, packed_attention, paged_attention
    g = torch.Generator().manual_seed(47)
    q, k, v = (torch.randn(h, 60, 64, generator=g).bfloat16().to(DEV).requires_grad_() for h in (4, 2, 2))
    off = torch.tensor([0, 45, 60], device=DEV, dtype=torch.int32)
    outside = PagedKVCache(12, 16, 2, 64)
    with torch.inference_mode():
        want = packed_attention(q, k, v, off)
        for cache_ in (outside, PagedKVCache(12, 16, 2, 64)):
            ids = [cache_.open(), cache_.open()]
            table, lengths = cache_.grow(ids, [45, 15])
            append_pages(k, v, *cache_.layer(), table, lengths, off)
            twin = cache_.fork(ids[0])
            cache_.grow([twin])                            # copies the page that both would write
            o = paged_attention(q[:, [44, 59]].transpose(0, 1), *cache_.layer(), *cache_.tables(ids))
            for b, row in enumerate((44, 59)):
                a, n = (0, 45) if b == 0 else (45, 15)
                assert_within(o[b], want_one(q[:, row], (k[:, a:a + n], v[:, a:a + n]), 0.125, torch.bfloat16), f"sequence {b}")
                assert_within(want[:, row], want_one(q[:, row], (k[:, a:a + n], v[:, a:a + n]), 0.125, torch.bfloat16), f"row {row}")
