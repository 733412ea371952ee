"""A paged key / value cache and the attention of new tokens over it (csrc/paged.hip).  No counterpart in the reference.

Pages are (pages, heads, page tokens, D) tensors; token t of a sequence lies at place t % page of page table[t // page] of
its row of the page table.  The functions take any such tensors; PagedKVCache keeps the books for a program that has no
allocator of its own.
"""
import heapq

import torch

from . import _lib


def paged_attention(q, k_pages, v_pages, page_table, lengths, sm_scale=None, out=None):
    """
    Attention of one new token a sequence over the cached tokens of it (the new one's own key and value among them:
    append_pages first).

    Args:
        q: (B, H, D), bf16 or fp16, D 64 or 128
        k_pages, v_pages: (pages, Hkv, page, D), page a power of two from 8 to 1024; H is a multiple of Hkv
        page_table: (B, W) int32 on the GPU: the page numbers of each sequence, in order
        lengths: (B,) int32 on the GPU: cached tokens of each sequence
        sm_scale: softmax scale, defaults to 1 / sqrt(D)
        out: written instead of a new tensor
    Returns:
        o: (B, H, D) in q's dtype; 0 for a sequence without tokens.

    Several new tokens of one sequence are that many rows with its pages (one row of a table, expanded) and growing
    lengths.  Table and lengths are read on the GPU when the kernels run (a captured graph replays with what they then hold).
    A page number outside the cache, or a length beyond W pages, is not followed: that sequence's rows are NaN.  Not
    differentiable: where gradients are recorded the call is refused, as those below are.
    """
    if sm_scale is None:
        sm_scale = q.shape[-1] ** -0.5
    return _lib.host().paged_attention(q, k_pages, v_pages, page_table, lengths, sm_scale, out)


def append_pages(k, v, k_pages, v_pages, page_table, lengths, offsets=None):
    """
    Put new keys and values into their pages.

    Args:
        k, v: (Hkv, T, D): the new rows of all sequences
        k_pages, v_pages: (pages, Hkv, page, D), written in place
        page_table, lengths: as paged_attention reads them, lengths with the new tokens counted
        offsets: (B + 1,) int32 on the GPU: sequence b's new rows are offsets[b] .. offsets[b + 1] - 1 of k and v, the last
            of them its token lengths[b] - 1; None: T = B, row b is sequence b's newest token

    A row of no sequence, or one whose place or page number is outside the cache, is left out.  Sequences must not share
    the pages that they are writing to (PagedKVCache copies such a page first).
    """
    _lib.host().append_pages(k, v, k_pages, v_pages, page_table, lengths, offsets)


def copy_pages(k_pages, v_pages, src, dst):
    """
    Copy page src[i] to page dst[i], in k_pages and v_pages; (pages, Hkv, page, D), or (layers, pages, Hkv, page, D) for the
    same pages of every layer.  src and dst are sequences of numbers on the host, which the launch carries (a captured
    graph repeats these very copies).  A page that is written twice, or written and read, is refused.
    """
    _lib.host().copy_pages(k_pages, v_pages, src, dst)


class PagedKVCache:
    """
    Pages for the keys and values of many sequences, and the books on who holds which: a sequence grows by pages as its
    tokens come, forks share their full pages, and a page goes back when its last holder does.

        cache = PagedKVCache(pages=4096, page=16, heads=8, head_dim=128, layers=32)
        ids = [cache.open() for _ in prompts]
        table, lengths = cache.grow(ids, [len(p) for p in prompts])
        for layer: append_pages(k, v, *cache.layer(layer), table, lengths, offsets)
        while decoding:
            table, lengths = cache.grow(ids)                       # room for one more token each
            for layer:
                append_pages(k, v, *cache.layer(layer), table, lengths)
                o = paged_attention(q, *cache.layer(layer), table, lengths)

    Page numbers are handed out lowest first.  All of it is work of the host, but for the pages that a fork's first write
    or `compact` copies and the two small tensors that `grow` sends to the GPU; calls belong on the stream that the
    cache is used on.
    """

    def __init__(self, pages, page, heads, head_dim, layers=1, dtype=torch.bfloat16, device="cuda"):
        if page < 8 or page > 1024 or page & (page - 1):
            raise ValueError(f"vmonarch_amd: pages of {page} tokens (powers of two from 8 to 1024)")
        if min(pages, heads, head_dim, layers) < 1:
            raise ValueError("vmonarch_amd: a cache has pages, heads, features and layers")
        if dtype not in _lib.DTYPES:
            raise ValueError(f"vmonarch_amd: a cache of {dtype} (bf16 and fp16 are built)")
        shape = (layers, pages, heads, page, head_dim)
        self.k_pages, self.v_pages = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.page = page
        self._free = list(range(pages))      # a heap
        self._holders = [0] * pages
        self._held = {}                      # sequence -> its page numbers
        self._tokens = {}                    # sequence -> its tokens
        self._next = 0

    def layer(self, i=0):
        """(k_pages, v_pages) of one layer."""
        return self.k_pages[i], self.v_pages[i]

    @property
    def free_pages(self):
        return len(self._free)

    def length(self, seq):
        return self._tokens[seq]

    def pages_of(self, seq):
        return list(self._held[seq])

    def open(self):
        """A new sequence without tokens."""
        seq, self._next = self._next, self._next + 1
        self._held[seq], self._tokens[seq] = [], 0
        return seq

    def fork(self, seq):
        """A new sequence that begins as `seq` is now.  Its pages are shared; the last, unfilled one is copied when either
        of them next grows."""
        new = self.open()
        self._held[new], self._tokens[new] = list(self._held[seq]), self._tokens[seq]
        for p in self._held[new]:
            self._holders[p] += 1
        return new

    def free(self, seq):
        """End a sequence; pages that nobody else holds go back."""
        for p in self._held.pop(seq):
            self._let_go(p)
        del self._tokens[seq]

    def _let_go(self, p):
        self._holders[p] -= 1
        if self._holders[p] == 0:
            heapq.heappush(self._free, p)

    def grow(self, seqs, counts=None):
        """
        Room for counts[i] more tokens of seqs[i] (default: one each), and the (page_table, lengths) that append_pages and
        paged_attention then take, in the order of `seqs`.  Raises, with nothing changed, if the cache has too few pages.
        """
        seqs = list(seqs)
        counts = [1] * len(seqs) if counts is None else [int(n) for n in counts]
        if len(counts) != len(seqs) or len(set(seqs)) != len(seqs):
            raise ValueError("vmonarch_amd: grow takes each sequence once, and a count for each")
        if any(n < 0 for n in counts):
            raise ValueError("vmonarch_amd: a sequence cannot grow by less than nothing")
        need, holders = 0, {}
        shared = []                                    # sequences whose unfilled last page others hold too
        for s, n in zip(seqs, counts):
            held, tokens = self._held[s], self._tokens[s]
            need += max(0, -(-(tokens + n) // self.page) - len(held))
            if n and tokens % self.page:
                p = held[-1]
                left = holders.setdefault(p, self._holders[p])
                if left > 1:                           # (the last holder that writes keeps the page itself)
                    shared.append(s)
                    holders[p] = left - 1
                    need += 1
        if need > len(self._free):
            raise RuntimeError(f"vmonarch_amd: {need} pages needed, {len(self._free)} free")
        src, dst = [], []
        for s in shared:
            p, new = self._held[s][-1], heapq.heappop(self._free)
            self._holders[p] -= 1
            self._holders[new] = 1
            self._held[s][-1] = new
            src.append(p)
            dst.append(new)
        if src:
            copy_pages(self.k_pages, self.v_pages, src, dst)
        for s, n in zip(seqs, counts):
            self._tokens[s] += n
            held = self._held[s]
            while len(held) * self.page < self._tokens[s]:
                p = heapq.heappop(self._free)
                self._holders[p] = 1
                held.append(p)
        return self.tables(seqs)

    def tables(self, seqs):
        """(page_table, lengths) of `seqs` as they are; unused places of the table hold -1."""
        held = [self._held[s] for s in seqs]
        width = max([1] + [len(h) for h in held])
        both = torch.tensor([n for s, h in zip(seqs, held) for n in [self._tokens[s]] + h + [-1] * (width - len(h))],
                            dtype=torch.int32).view(len(held), 1 + width).to(self.k_pages.device)
        return both[:, 1:], both[:, 0].contiguous()

    def compact(self):
        """Move the held pages to the lowest numbers, so that the rest of the cache is one piece; returns how many moved.
        Tables made before no longer hold."""
        used = sorted({p for h in self._held.values() for p in h})
        src = [p for p in used if p >= len(used)]
        taken = set(used)
        dst = [p for p in range(len(used)) if p not in taken]
        if not src:
            return 0
        copy_pages(self.k_pages, self.v_pages, src, dst)
        to = dict(zip(src, dst))
        for h in self._held.values():
            h[:] = [to.get(p, p) for p in h]
        for a, b in to.items():
            self._holders[b], self._holders[a] = self._holders[a], 0
        self._free = list(range(len(used), len(self._holders)))
        return len(src)
