"""What packed_attention and the paged cache refuse before any launch, and the cache's books: no GPU needed."""
import pytest
import torch


def x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def i32(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("change, message", [
    (dict(k=x(2, 9, 64, dtype=torch.float16)), "one dtype"), (dict(q=x(4, 9, 64, dtype=torch.float32)), "one dtype"),
    (dict(k=x(3, 9, 64), v=x(3, 9, 64)), "multiple"), (dict(v=x(2, 8, 64)), "one shape"), (dict(k=x(2, 9, 32), v=x(2, 9, 32)), "head dim"),
    (dict(q=x(1, 4, 9, 64)), "heads, tokens, D"), (dict(offsets=torch.tensor([0, 9])), "int32"), (dict(offsets=i32()), "one more"),
    (dict(k_offsets=i32(0, 4, 9)), "one more"), (dict(out=x(4, 8, 64)), "shaped like q"), (dict(out=x(4, 9, 64, dtype=torch.float16)), "dtype"),
    (dict(k=torch.zeros(2, 9, 64, dtype=torch.bfloat16, device="meta")), "device"),
    ({n: x(h, 9, 64, dtype=torch.float32) for n, h in (("q", 4), ("k", 2), ("v", 2))}, "bf16 or fp16")])
def test_packed_attention_refuses(change, message):
    from vmonarch_amd import packed_attention
    args = dict(q=x(4, 9, 64), k=x(2, 9, 64), v=x(2, 9, 64), offsets=i32(0, 9))
    with pytest.raises(AssertionError, match=message):
        packed_attention(**{**args, **change})


def test_inputs_on_the_host_are_refused():
    from vmonarch_amd import append_pages, copy_pages, packed_attention, paged_attention
    pages, table = x(4, 2, 8, 64), i32(0).view(1, 1)
    for call in (lambda: packed_attention(x(4, 9, 64), x(2, 9, 64), x(2, 9, 64), i32(0, 9)),
                 lambda: paged_attention(x(1, 4, 64), pages, pages, table, i32(3)),
                 lambda: append_pages(x(2, 1, 64), x(2, 1, 64), pages, pages.clone(), table, i32(1)),
                 lambda: copy_pages(pages, pages.clone(), [0], [1])):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_out_with_gradients_is_refused():
    from vmonarch_amd import packed_attention
    with pytest.raises(RuntimeError, match="gradient"):
        packed_attention(x(4, 9, 64).requires_grad_(), x(2, 9, 64), x(2, 9, 64), i32(0, 9), out=x(4, 9, 64))


@pytest.mark.parametrize("change, message", [
    (dict(q=x(3, 64)), "sequences, heads, D"), (dict(k_pages=x(4, 2, 8, 32), v_pages=x(4, 2, 8, 32)), "head dim"),
    (dict(v_pages=x(4, 2, 16, 64)), "pages, heads"), (dict(page_table=i32(0, 1, 2)), "int32"), (dict(lengths=i32(1, 2)), "one length"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), "int32"), (dict(q=x(3, 3, 64)), "multiple"),
    (dict(q=x(3, 4, 64, dtype=torch.float16)), "dtype"), (dict(out=x(3, 4, 32)), "shaped like q")])
def test_paged_attention_refuses(change, message):
    from vmonarch_amd import paged_attention
    args = dict(q=x(3, 4, 64), k_pages=x(4, 2, 8, 64), v_pages=x(4, 2, 8, 64), page_table=torch.zeros(3, 2, dtype=torch.int32),
                lengths=i32(1, 2, 3))
    with pytest.raises(AssertionError, match=message):
        paged_attention(**{**args, **change})


@pytest.mark.parametrize("change, message", [
    (dict(v=x(2, 4, 64)), "one shape"), (dict(k=x(3, 3, 64), v=x(3, 3, 64)), "heads"), (dict(offsets=i32(0, 1, 3)), "one more"),
    (dict(k=x(2, 5, 64), v=x(2, 5, 64)), "one row a sequence"), (dict(lengths=i32(1, 2)), "one length")])
def test_append_pages_refuses(change, message):
    from vmonarch_amd import append_pages
    args = dict(k=x(2, 3, 64), v=x(2, 3, 64), k_pages=x(4, 2, 8, 64), v_pages=x(4, 2, 8, 64),
                page_table=torch.zeros(3, 2, dtype=torch.int32), lengths=i32(1, 2, 3))
    with pytest.raises(AssertionError, match=message):
        append_pages(**{**args, **change})


def test_pages_that_overlap_are_not_written():
    from vmonarch_amd import append_pages
    args = dict(k=x(2, 3, 64), v=x(2, 3, 64), page_table=torch.zeros(3, 2, dtype=torch.int32), lengths=i32(1, 2, 3))
    for pages in (x(1, 2, 8, 64).expand(4, 2, 8, 64), x(4, 2, 8, 68)[..., :64], x(4, 2, 8, 128)[..., ::2]):
        with pytest.raises(ValueError, match="aligned"):
            append_pages(k_pages=pages, v_pages=pages, **args)


def test_c_entries_refuse():
    """Each with its code and a message, before a launch."""
    import ctypes
    from test_capi import _addr
    from vmonarch_amd import _lib
    L = _lib.lib()

    def packed(**kw):
        a = _lib.PackedArgs()
        a.heads, a.kv_heads, a.n, a.tq, a.tk, a.d, a.sm_scale = 4, 2, 1, 16, 16, 64, 0.1
        a.q = a.k = a.v = a.o = a.grad_o = a.grad_q = a.grad_k = a.grad_v = _lib.View(_addr(), 0, 1024, 64)
        a.q_offsets = a.k_offsets = a.lse = _addr()
        a.stat_stride = 16
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    def paged(**kw):
        a = _lib.PagedArgs()
        a.batch, a.heads, a.kv_heads, a.d, a.pages, a.page_size, a.table_width, a.sm_scale = 2, 4, 2, 64, 8, 16, 300, 0.1
        a.q = a.k = a.v = a.o = _lib.View(_addr(), 2048, 1024, 64)
        a.table = a.lengths = _addr()
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    def append(**kw):
        a = _lib.AppendArgs()
        a.sequences, a.tokens, a.kv_heads, a.d, a.pages, a.page_size, a.table_width = 2, 2, 2, 64, 8, 16, 4
        a.k = a.v = a.k_pages = a.v_pages = _lib.View(_addr(), 2048, 1024, 64)
        a.table = a.lengths = _addr()
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    odd = _lib.View(_addr(2), 2048, 1024, 64)
    none = _lib.View(None, 2048, 1024, 64)
    calls = [
        (L.vmo_packed_fwd, packed, [dict(dtype=7), dict(kv_heads=3), dict(kv_heads=0), dict(n=-1), dict(tq=-1), dict(sm_scale=-1.0),
                                    dict(sm_scale=float("nan")), dict(q=odd), dict(k=none), dict(q_offsets=None)], 1),
        (L.vmo_packed_fwd, packed, [dict(d=48), dict(n=2049), dict(q=_lib.View(_addr(), 0, 1024, 1 << 27))], 2),
        (L.vmo_packed_bwd, packed, [dict(lse=None), dict(grad_q=none), dict(grad_v=odd)], 1),
        (L.vmo_packed_bwd, packed, [dict(), dict(workspace=_addr(), workspace_bytes=64)], 3),
        (L.vmo_paged_attention, paged, [dict(dtype=2), dict(kv_heads=3), dict(batch=-1), dict(pages=0), dict(table=None), dict(q=odd),
                                        dict(v=none), dict(sm_scale=float("inf"))], 1),
        (L.vmo_paged_attention, paged, [dict(d=96), dict(page_size=12), dict(page_size=4), dict(page_size=2048)], 2),
        (L.vmo_paged_attention, paged, [dict(), dict(workspace=_addr(), workspace_bytes=64)], 3),
        (L.vmo_append_pages, append, [dict(tokens=3), dict(tokens=-1), dict(d=12), dict(k=odd), dict(k_pages=none), dict(lengths=None),
                                      dict(pages=0)], 1),
        (L.vmo_append_pages, append, [dict(page_size=24)], 2),
    ]
    for f, make, changes, code in calls:
        for change in changes:
            assert f(ctypes.byref(make(**change)), None) == code, (f.__name__, change)
            assert L.vmo_last_error()
        assert f(None, None) == 1
    assert L.vmo_paged_attention(ctypes.byref(paged(batch=0)), None) == 0
    assert L.vmo_append_pages(ctypes.byref(append(tokens=0)), None) == 0

    def copy(src, dst, **kw):
        a = _lib.CopyArgs()
        a.layers, a.pages, a.pairs, a.k, a.v, a.page_bytes, a.layer_bytes = 1, 8, len(src), _addr(), _addr(), 1024, 8192
        a.src, a.dst = (ctypes.cast((ctypes.c_int32 * len(y))(*y), ctypes.c_void_p) for y in (src, dst))
        for n, v in kw.items():
            setattr(a, n, v)
        return L.vmo_copy_pages(ctypes.byref(a), None)

    for src, dst in (([0], [8]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3])):
        assert copy(src, dst) == 1
    assert copy([0], [1], page_bytes=24) == 1 and copy([0], [1], k=None) == 1 and copy([0], [1], pairs=-1) == 1
    assert copy([0], [1], pairs=0) == 0 and copy([0], [1], layers=0) == 0


def books(pages=6, page=8):
    from vmonarch_amd import PagedKVCache
    return PagedKVCache(pages, page, 1, 64, device="cpu")


def test_the_cache_hands_out_and_takes_back():
    c = books()
    a, b = c.open(), c.open()
    table, lengths = c.grow([a, b], [9, 8])
    assert table.tolist() == [[0, 1], [2, -1]] and lengths.tolist() == [9, 8] and lengths.dtype == table.dtype == torch.int32
    assert c.grow([b])[0].tolist() == [[2, 3]] and c.free_pages == 2
    with pytest.raises(RuntimeError, match="free"):
        c.grow([a, b], [8, 30])
    assert (c.length(a), c.length(b), c.free_pages) == (9, 9, 2)      # nothing changed
    d = c.fork(a)
    assert c.pages_of(d) == [0, 1] and c.free_pages == 2
    c.free(a)
    assert c.free_pages == 2 and c.pages_of(d) == [0, 1]              # the fork holds them
    c.grow([d], [3])                                                  # alone by now: no copy
    assert c.pages_of(d) == [0, 1] and c.length(d) == 12
    c.free(d)
    assert c.free_pages == 4 and c.grow([c.open()], [20])[0].tolist() == [[0, 1, 4]]
    assert c.grow([], [])[0].shape[0] == 0


def test_the_cache_refuses():
    c = books()
    a = c.open()
    for seqs, counts in (([a, a], [1, 1]), ([a], [1, 2]), ([a], [-1])):
        with pytest.raises(ValueError):
            c.grow(seqs, counts)
    with pytest.raises(KeyError):
        c.free(99)
    with pytest.raises(ValueError, match="powers of two"):
        books(page=12)
    with pytest.raises(ValueError):
        books(pages=0)
    from vmonarch_amd import PagedKVCache
    with pytest.raises(ValueError, match="bf16 and fp16"):
        PagedKVCache(4, 8, 1, 64, dtype=torch.float32, device="cpu")
    assert c.compact() == 0


def test_forks_copy_a_page_that_others_hold_when_they_write(monkeypatch):
    """Which pages are copied, and who keeps the first one: three sequences over one unfilled page."""
    import vmonarch_amd.paged as paged
    copies = []
    monkeypatch.setattr(paged, "copy_pages", lambda k, v, src, dst: copies.append((list(src), list(dst))))
    c = books(pages=10)
    a = c.open()
    c.grow([a], [11])                                  # pages 0, 1; 1 holds 3 tokens
    b, d = c.fork(a), c.fork(a)
    c.grow([b])                                        # one writes: a copy of its own
    assert copies == [([1], [2])] and c.pages_of(b) == [0, 2] and c.pages_of(a) == c.pages_of(d) == [0, 1]
    c.grow([a, d])                                     # both that are left: one copies, one keeps
    assert copies[1:] == [([1], [3])] and c.pages_of(a) == [0, 3] and c.pages_of(d) == [0, 1]
    c.grow([a, b, d])
    assert len(copies) == 2
    e = c.fork(a)
    c.grow([e], [0])                                   # nothing written: still shared
    assert c.pages_of(e) == c.pages_of(a) and len(copies) == 2
    full = c.open()
    c.grow([full], [8])
    other = c.fork(full)
    c.grow([full, other])                              # a filled page stays shared
    assert len(copies) == 2 and c.pages_of(full)[0] == c.pages_of(other)[0] and c.pages_of(full)[1] != c.pages_of(other)[1]
    for s in (a, b, d, e, full, other):
        c.free(s)
    assert c.free_pages == 10


def test_compaction_moves_the_held_pages_down(monkeypatch):
    import vmonarch_amd.paged as paged
    moves = []
    monkeypatch.setattr(paged, "copy_pages", lambda k, v, src, dst: moves.append(dict(zip(src, dst))))
    c = books(pages=12)
    a, b, d = c.open(), c.open(), c.open()
    for s in (a, b, d):
        c.grow([s], [24])                              # pages 0-2, 3-5, 6-8
    twin = c.fork(d)
    c.free(a)
    c.free(b)
    assert c.compact() == 3 and moves == [{6: 0, 7: 1, 8: 2}]
    assert c.pages_of(d) == c.pages_of(twin) == [0, 1, 2] and c.free_pages == 9
    assert c.compact() == 0
    c.free(d)
    assert c.free_pages == 9
    c.free(twin)
    assert c.free_pages == 12 and c.grow([c.open()], [8 * 12])[0].tolist() == [list(range(12))]


def test_the_cache_records_no_gradients():
    from vmonarch_amd import append_pages, copy_pages, paged_attention
    q, k, pages = x(2, 2, 64), x(2, 2, 64), x(3, 2, 8, 64)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: paged_attention(q.requires_grad_(), pages, pages, table, lens),
                 lambda: append_pages(k.requires_grad_(), k, pages, pages, table, lens),
                 lambda: copy_pages(pages.requires_grad_(), pages, [0], [1])):
        with pytest.raises(RuntimeError, match="no_grad"):
            call()
