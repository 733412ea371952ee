"""What is measured of the language-model side of the attention: packed causal prompts (forward, training), one new
token a sequence over a paged key / value cache, and the cache's own work (new rows into their pages, pages copied).

A case is a dict of plain values:
  op        "packed" (packed_attention), "paged" (paged_attention), "append" (append_pages) or "copy" (copy_pages)
  dtype     "bf16" or "f16";  D: head dim;  H: query heads;  KVH: key / value heads (each shared by H / KVH)
  lengths   "a+b+...": tokens of each sequence ("packed": the query tokens; "append": the new tokens)
  past      "a+b+...": cached tokens of each sequence that come before those ("packed": keys beyond the queries)
  train     "packed": forward and the gradients of q, k, v instead of the forward alone
  layout    "hnd": (heads, tokens, D) tensors; "nhd": (tokens, heads, D) buffers viewed so, as projections give them
  page      tokens a page;  pages: pages of the cache;  layers: layers that one cache holds ("copy")
  moves     "copy": pages copied to others, in every layer
"""
import math
import random

import torch

own = False   # True: run() calls the framework's operators; False: their plain forms

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _numbers(text):
    return [int(x) for x in text.split("+")]


def _text(numbers):
    return "+".join(str(int(x)) for x in numbers)


def _spread(n, low, high, seed):
    """n lengths between low and high, evenly over their logarithm, in a shuffled order that the seed gives."""
    rng = random.Random(seed)
    got = [int(round(low * (high / low) ** (i / max(1, n - 1)))) for i in range(n)]
    rng.shuffle(got)
    return got


def _packed(name, lengths, H, KVH, D, dtype="bf16", past=None, train=False, layout="nhd"):
    return {"name": name, "op": "packed", "lengths": _text(lengths), "past": _text(past or [0] * len(lengths)), "H": H,
            "KVH": KVH, "D": D, "dtype": dtype, "train": train, "layout": layout}


def _paged(name, lengths, H, KVH, D, page, dtype="bf16"):
    return {"name": name, "op": "paged", "past": _text(lengths), "H": H, "KVH": KVH, "D": D, "page": page, "dtype": dtype}


def _append(name, lengths, past, KVH, D, page, dtype="bf16"):
    return {"name": name, "op": "append", "lengths": _text(lengths), "past": _text(past), "KVH": KVH, "D": D, "page": page,
            "dtype": dtype}


def _copy(name, layers, pages, moves, KVH, D, page, dtype="bf16"):
    return {"name": name, "op": "copy", "layers": layers, "pages": pages, "moves": moves, "KVH": KVH, "D": D, "page": page,
            "dtype": dtype}


def listed():
    return [
        # a few short prompts, odd lengths, one of a single token: the smallest call, where latency counts
        _packed("prompt_short", [77, 1, 200, 33], 8, 2, 64),
        # an ordinary batch of prompts of very different lengths, some of them continued after cached tokens
        _packed("prompt_batch", _spread(12, 40, 2900, 1), 12, 4, 128, past=[0, 0, 512, 0, 1111, 0, 0, 64, 0, 0, 0, 999]),
        # one long context
        _packed("prompt_long", [16384], 12, 4, 128),
        # training on a packed batch of odd lengths
        _packed("train_batch", _spread(10, 50, 2048, 2), 8, 2, 64, dtype="f16", train=True, layout="hnd"),
        # training on long contexts: the largest case
        _packed("train_long", [12000, 4384], 8, 2, 128, train=True),
        # one sequence's next token: the smallest step
        _paged("token_one", [2000], 8, 2, 128, 16),
        # the next token of an ordinary serving batch, lengths from a few tokens to thousands
        _paged("token_batch", _spread(64, 16, 8192, 3), 24, 8, 128, 16),
        # few long sequences, heads not shared
        _paged("token_long", [32760, 16384, 30011, 25000], 12, 12, 64, 64, dtype="f16"),
        # the batch's new token goes into the cache
        _append("append_token", [1] * 64, _spread(64, 16, 4096, 4), 8, 128, 16),
        # prompts go into the cache
        _append("append_prompts", _spread(12, 40, 9000, 5), _spread(12, 1, 999, 6), 8, 128, 16),
        # sequences fork: the page that each of them is filling is copied, in all layers
        _copy("copy_fork", 12, 256, 32, 4, 128, 16),
        # a cache's live pages move together (compaction), in all its layers
        _copy("copy_compact", 12, 640, 256, 4, 128, 16),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        KVH = rng.choice([1, 2, 3, 4, 8])
        common = {"KVH": KVH, "D": rng.choice([64, 128]), "dtype": rng.choice(["bf16", "bf16", "f16"])}
        op = rng.choice(["packed", "packed", "paged", "append", "copy"])
        if op == "packed":
            lengths = [_log_int(rng, 1, 12000) for _ in range(_log_int(rng, 1, 16))]
            past = [rng.choice([0, 0, _log_int(rng, 1, 2000)]) for _ in lengths]
            case = {"op": op, "lengths": _text(lengths), "past": _text(past), "H": KVH * rng.choice([1, 2, 3, 4]),
                    "train": rng.random() < 0.4, "layout": rng.choice(["hnd", "nhd"]), **common}
            # (the plain form holds every score of the packed batch)
            if sum(lengths) * (sum(lengths) + sum(past)) * case["H"] > 1.6e9:
                continue
        elif op == "paged":
            past = [_log_int(rng, 1, 32760) for _ in range(_log_int(rng, 1, 96))]
            case = {"op": op, "past": _text(past), "H": KVH * rng.choice([1, 2, 3, 4, 6, 8]), "page": rng.choice([16, 32, 64]),
                    **common}
            if len(past) * max(past) * KVH > 4e6:
                continue
        elif op == "append":
            n = _log_int(rng, 1, 64)
            one = rng.random() < 0.4
            lengths = [1 if one else _log_int(rng, 1, 9000) for _ in range(n)]
            case = {"op": op, "lengths": _text(lengths), "past": _text(_log_int(rng, 1, 4096) - 1 for _ in range(n)),
                    "page": rng.choice([16, 32, 64]), **common}
            if sum(lengths) + sum(_numbers(case["past"])) > 150000:
                continue
        else:
            moves = _log_int(rng, 1, 256)
            case = {"op": op, "layers": rng.choice([1, 8, 12]), "pages": 2 * moves + _log_int(rng, 1, 128), "moves": moves,
                    "page": rng.choice([16, 32, 64]), **common}
            if case["layers"] * case["pages"] * case["page"] * KVH > 1.0e6:
                continue
        return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _offsets(lengths):
    got = [0]
    for n in lengths:
        got.append(got[-1] + n)
    return torch.tensor(got, dtype=torch.int32, device="cuda")


def _cache(case, g, lengths):
    """Pages in a shuffled order, as a cache that has served for a while hands them out, with a few unused."""
    page, dtype = case["page"], DTYPES[case["dtype"]]
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # unused places of the table hold page 0
    at = _offsets(need)[:-1].long()[:, None] + torch.arange(max(need), device="cuda")
    used = torch.arange(max(need), device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(used, order[at.clamp_max(pages - 1)], torch.zeros_like(order[:1]))
    shape = (pages, case["KVH"], page, case["D"])
    return {"k_pages": _normal(g, shape, dtype), "v_pages": _normal(g, shape, dtype), "table": table.contiguous(),
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g, dtype, D = _generator(seed), DTYPES[case["dtype"]], case["D"]
    state = {"op": case["op"]}
    if case["op"] == "packed":
        lengths, past = _numbers(case["lengths"]), _numbers(case["past"])

        def tensor(heads, tokens):
            if case["layout"] == "hnd":
                return _normal(g, (heads, tokens, D), dtype)
            return _normal(g, (tokens, heads, D), dtype).transpose(0, 1)

        nq, nk = sum(lengths), sum(lengths) + sum(past)
        state |= {"q": tensor(case["H"], nq), "k": tensor(case["KVH"], nk), "v": tensor(case["KVH"], nk),
                  "offsets": _offsets(lengths), "k_offsets": _offsets([a + b for a, b in zip(lengths, past)])}
        if case["train"]:
            state["grad"] = tensor(case["H"], nq)
            for name in "qkv":
                state[name].requires_grad_()
    elif case["op"] == "paged":
        lengths = _numbers(case["past"])
        state |= _cache(case, g, lengths)
        state["q"] = _normal(g, (len(lengths), case["H"], D), dtype)
    elif case["op"] == "append":
        new, past = _numbers(case["lengths"]), _numbers(case["past"])
        state |= _cache(case, g, [a + b for a, b in zip(new, past)])   # lengths: with the new tokens
        state["offsets"] = _offsets(new)
        state["k"] = _normal(g, (sum(new), case["KVH"], D), dtype).transpose(0, 1)
        state["v"] = _normal(g, (sum(new), case["KVH"], D), dtype).transpose(0, 1)
    else:
        rng = random.Random(int(seed))
        picked = rng.sample(range(case["pages"]), 2 * case["moves"])
        state["src"], state["dst"] = picked[: case["moves"]], picked[case["moves"]:]
        shape = (case["layers"], case["pages"], case["KVH"], case["page"], D)
        state["k_pages"], state["v_pages"] = _normal(g, shape, dtype), _normal(g, shape, dtype)
    return state


def _plain_packed(q, k, v, offsets, k_offsets):
    """Every score of the packed batch, those of other sequences and of later tokens masked."""
    group, dev = q.shape[0] // k.shape[0], q.device
    rows, cols = torch.arange(q.shape[1], device=dev), torch.arange(k.shape[1], device=dev)
    qs, ks = (torch.searchsorted(off[1:].contiguous(), x.int(), right=True) for off, x in ((offsets, rows), (k_offsets, cols)))
    q_end, k_end = offsets[1:].long()[qs], k_offsets[1:].long()[ks]
    seen = (qs[:, None] == ks[None, :]) & ((k_end - cols)[None, :] >= (q_end - rows)[:, None])   # counted from the end
    kf, vf = (t.float().repeat_interleave(group, 0) for t in (k, v))
    s = torch.matmul(q.float() * q.shape[-1] ** -0.5, kf.transpose(1, 2).contiguous()).masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    return (torch.matmul(p, vf.contiguous()) / p.sum(-1, keepdim=True).clamp_min(1e-30)).to(q.dtype)


def _plain_paged(q, k_pages, v_pages, table, lengths):
    """Every sequence's pages gathered to the longest one's length."""
    B, H, D = q.shape
    KVH = k_pages.shape[1]
    k, v = (t[table.long()].float().transpose(1, 2).reshape(B, KVH, -1, D) for t in (k_pages, v_pages))
    s = torch.matmul((q.float() * D ** -0.5).view(B, KVH, H // KVH, D), k.transpose(2, 3).contiguous())
    s = s.masked_fill(torch.arange(k.shape[2], device=q.device) >= lengths[:, None, None, None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(B, H, D).to(q.dtype)


def _plain_append(k, v, k_pages, v_pages, table, lengths, offsets):
    rows, page = torch.arange(k.shape[1], device=k.device), k_pages.shape[2]
    seq = torch.searchsorted(offsets[1:].contiguous(), rows.int(), right=True)
    at = lengths.long()[seq] - (offsets[1:].long()[seq] - rows)   # the last new token is the last of the sequence
    where = table[seq, at // page].long()
    k_pages[where, :, at % page] = k.transpose(0, 1)
    v_pages[where, :, at % page] = v.transpose(0, 1)


def _plain_copy(k_pages, v_pages, src, dst):
    src, dst = torch.tensor([src, dst], device=k_pages.device)
    k_pages[:, dst] = k_pages[:, src]
    v_pages[:, dst] = v_pages[:, src]


def run(state):
    if own:
        from vmonarch_amd import append_pages, copy_pages, packed_attention, paged_attention
    op = state["op"]
    if op == "packed":
        q, k, v, lengths = state["q"], state["k"], state["v"], (state["offsets"], state["k_offsets"])
        with torch.set_grad_enabled("grad" in state):
            o = packed_attention(q, k, v, *lengths) if own else _plain_packed(q, k, v, *lengths)
        if "grad" not in state:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), state["grad"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    cache = (state["k_pages"], state["v_pages"])
    if op == "paged":
        x = (state["q"], *cache, state["table"], state["lengths"])
        return {"o": paged_attention(*x) if own else _plain_paged(*x)}
    if op == "append":
        x = (state["k"], state["v"], *cache, state["table"], state["lengths"], state["offsets"])
        append_pages(*x) if own else _plain_append(*x)
    else:
        copy_pages(*cache, state["src"], state["dst"]) if own else _plain_copy(*cache, state["src"], state["dst"])
    return {"k_pages": cache[0], "v_pages": cache[1]}


def work(case):
    D, KVH = case["D"], case["KVH"]
    if case["op"] == "packed":
        lengths, past = _numbers(case["lengths"]), _numbers(case["past"])
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(lengths, past))
        rows, keys = sum(lengths) * case["H"], (sum(lengths) + sum(past)) * KVH
        nbytes, flops = (2 * rows + 2 * keys) * D * 2, 4.0 * D * pairs * case["H"]
        if case["train"]:   # the upstream gradient read, three gradients written; five products for the forward's two
            nbytes, flops = nbytes + (2 * rows + 2 * keys) * D * 2, 3.5 * flops
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "paged":
        tokens, rows = sum(_numbers(case["past"])), len(_numbers(case["past"])) * case["H"]
        return {"bytes": (2 * tokens * KVH + 2 * rows) * D * 2, "flops": 4.0 * D * tokens * case["H"]}
    if case["op"] == "append":
        return {"bytes": 2 * 2 * sum(_numbers(case["lengths"])) * KVH * D * 2, "flops": 0}
    return {"bytes": 2 * 2 * case["layers"] * case["moves"] * case["page"] * KVH * D * 2, "flops": 0}


def _exact_head(q, k, v, past, grad, rows=2048):
    """One head of one sequence in 64 bits, some rows at a time: o, and with an upstream gradient dq, dk and dv."""
    scale, n = q.shape[-1] ** -0.5, q.shape[0]
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for a in range(0, n, rows):
        b = min(n, a + rows)
        end = b + past                                   # keys that some of these rows see
        x = torch.mm(q[a:b], k[:end].t().contiguous()) * scale
        x += torch.full_like(x, -math.inf).triu(a + past + 1)
        p = torch.softmax(x, -1)
        o[a:b] = torch.mm(p, v[:end])
        if grad is not None:
            dp = torch.mm(grad[a:b], v[:end].t().contiguous())
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
            dv[:end] += torch.mm(p.t().contiguous(), grad[a:b])
            dk[:end] += torch.mm(ds.t().contiguous(), q[a:b])
            dq[a:b] = torch.mm(ds, k[:end])
    return o, dq, dk, dv


def _exact_packed(case, state):
    lengths, past = _numbers(case["lengths"]), _numbers(case["past"])
    q, k, v = (state[n].detach().double() for n in "qkv")
    grad, group = (state["grad"].double() if case["train"] else None), case["H"] // case["KVH"]
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    at = kat = 0
    for n, p in zip(lengths, past):
        rows, keys = slice(at, at + n), slice(kat, kat + n + p)
        for h in range(case["H"]):
            got = _exact_head(q[h, rows], k[h // group, keys], v[h // group, keys], p, None if grad is None else grad[h, rows])
            o[h, rows], dq[h, rows] = got[0], got[1]
            dk[h // group, keys] += got[2]
            dv[h // group, keys] += got[3]
        at, kat = at + n, kat + n + p
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"o": o}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "packed":
        return _exact_packed(case, state)
    kp, vp = state["k_pages"].double(), state["v_pages"].double()
    if case["op"] == "copy":
        source = list(range(case["pages"]))
        for s, d in zip(state["src"], state["dst"]):
            source[d] = s
        source = torch.tensor(source, device="cuda")
        return {"k_pages": kp.index_select(1, source), "v_pages": vp.index_select(1, source)}
    page, table = case["page"], state["table"].cpu()
    if case["op"] == "append":
        at = 0
        for b, (n, past) in enumerate(zip(_numbers(case["lengths"]), _numbers(case["past"]))):
            done = 0
            while done < n:   # the rows that go into one page
                first = (past + done) % page
                take = min(page - first, n - done)
                which = int(table[b, (past + done) // page])
                rows = slice(at + done, at + done + take)
                kp[which, :, first:first + take] = state["k"][:, rows].double()
                vp[which, :, first:first + take] = state["v"][:, rows].double()
                done += take
            at += n
        return {"k_pages": kp, "v_pages": vp}
    q, out = state["q"].double(), []
    group = case["H"] // case["KVH"]
    for b, n in enumerate(_numbers(case["past"])):
        mine = table[b, : -(-n // page)].long().cuda()
        heads = []
        for h in range(case["KVH"]):
            k, v = (t[mine, h].reshape(-1, case["D"])[:n] for t in (kp, vp))
            x = torch.mm(q[b, h * group:(h + 1) * group], k.t().contiguous()) * case["D"] ** -0.5
            heads.append(torch.mm(torch.softmax(x, -1), v))
        out.append(torch.cat(heads, 0))
    return {"o": torch.stack(out)}
