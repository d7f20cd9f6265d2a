"""Generation from a paged key-value cache, as cases that can be timed: keys and values written to
pages, attention of one new token per sequence over them, eviction by accumulated attention weight,
beam search's selection, and the beams' reordering of the cache.

``listed()`` holds the named cases, ``draw(rng)`` gives further ones of the same ranges.
``prepare(case, seed)`` makes the inputs on the GPU and ``run(state)`` is one pass: through the
framework's entry points where ``own`` is true, else in elementary torch operations.
``exact(case, seed)`` is the same pass in 64 bits, ``work(case)`` the bytes and operations that it
cannot do without.

A cache is a pool of pages [pages, key-value heads, slots, D] for the keys and one for the values, a
table [rows, pages of a row] that names each row's pages, and the rows' lengths.  The largest case
reads about 1 GB.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EOS = 2  # the token that ends a sequence


def listed():
    return [
        # One decoding step of a serving batch writes each sequence's new key and value: the
        # smallest of the calls, once per layer and token.
        dict(name="append_step_bf16", kind="append", rows=64, heads=8, D=128, page=16, new=1, before=1500,
             ragged=True, meta=True, dtype="bf16"),
        # The prompts of a batch, padded to the longest, go into the cache after the prefill.
        dict(name="append_prompts_f32", kind="append", rows=8, heads=12, D=64, page=32, new=1024, before=0,
             ragged=True, meta=False, dtype="f32"),
        # One sequence, one new token, a cache of ragged length: latency.
        dict(name="decode_one_f32", kind="decode", rows=1, heads=12, group=1, D=64, page=16, length=1000,
             ragged=False, weigh=False, dtype="f32"),
        # The batch that the contiguous decode is benchmarked on, out of pages.
        dict(name="decode_batch_f32", kind="decode", rows=32, heads=12, group=1, D=64, page=64, length=2048,
             ragged=False, weigh=False, dtype="f32"),
        # Serving with shared key-value heads, sequences of all lengths up to 8 thousand.
        dict(name="decode_ragged_bf16", kind="decode", rows=64, heads=8, group=4, D=128, page=16, length=8191,
             ragged=True, weigh=False, dtype="bf16"),
        # Two long documents with few key-value heads; each position's attention weight is added
        # up for the eviction.
        dict(name="decode_long_bf16", kind="decode", rows=2, heads=2, group=8, D=128, page=128, length=131071,
             ragged=False, weigh=True, dtype="bf16"),
        # A batch at the end of its context is cut to half, the last 256 positions kept.
        dict(name="evict_half_f32", kind="evict", rows=32, heads=12, D=64, page=64, length=2048, keep=1024,
             recent=256, dtype="f32"),
        # A long cache loses its least used positions, in steps of 64.
        dict(name="evict_few_bf16", kind="evict", rows=2, heads=8, D=128, page=16, length=32832, keep=32768,
             recent=4096, dtype="bf16"),
        # First step of one search: all beams but one start at -inf.
        dict(name="select_first_f32", kind="select", groups=1, beams=4, vocab=8192, first=True, dtype="f32"),
        # A batch of searches over an odd vocabulary, some beams finished.
        dict(name="select_batch_bf16", kind="select", groups=32, beams=8, vocab=50257, first=False, dtype="bf16"),
        # The cache of one search follows its beams: the last, partly filled page is copied.
        dict(name="reorder_one_f32", kind="reorder", groups=1, beams=4, layers=2, heads=12, D=64, page=16,
             length=1001, dtype="f32"),
        # A batch of searches on a model of 12 layers.
        dict(name="reorder_batch_bf16", kind="reorder", groups=32, beams=8, layers=12, heads=12, D=64, page=32,
             length=1500, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over their logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "evict", "select", "reorder"])
    dtype, D = rng.choice(["f32", "bf16"]), rng.choice([32, 64, 128])
    page = rng.choice([8, 16, 32, 64, 128])
    e = 4 if dtype == "f32" else 2
    if kind == "append":
        rows, heads = _log(rng, 1, 64), rng.randint(1, 16)
        new = _log(rng, 1, max(1, min(2048, (100 << 20) // (4 * rows * heads * D * e))))
        return dict(kind=kind, rows=rows, heads=heads, D=D, page=page, new=new, before=rng.randint(0, 2000),
                    ragged=rng.random() < 0.5, meta=rng.random() < 0.5, dtype=dtype)
    if kind == "decode":
        rows, heads, group = _log(rng, 1, 64), rng.randint(1, 16), rng.choice([1, 1, 2, 3, 4, 5, 8, 12, 16])
        length = _log(rng, 1, max(1, min(131072, (800 << 20) // (2 * rows * heads * D * 4))))
        return dict(kind=kind, rows=rows, heads=heads, group=group, D=D, page=page, length=length,
                    ragged=rng.random() < 0.5, weigh=rng.random() < 0.5, dtype=dtype)
    if kind == "evict":
        rows, heads = _log(rng, 1, 32), rng.randint(1, 12)
        length = _log(rng, 2, max(2, min(65536, (400 << 20) // (2 * rows * heads * D * 4))))
        keep = rng.randint(1, length)
        return dict(kind=kind, rows=rows, heads=heads, D=D, page=page, length=length, keep=keep,
                    recent=rng.randint(0, keep), dtype=dtype)
    if kind == "select":
        groups, beams = _log(rng, 1, 32), rng.randint(1, 16)
        return dict(kind=kind, groups=groups, beams=beams,
                    vocab=_log(rng, 16, min(131072, (12 << 20) // (groups * beams))), first=rng.random() < 0.2,
                    dtype=dtype)
    groups, beams, layers, heads = _log(rng, 1, 32), rng.randint(1, 8), rng.randint(1, 12), rng.randint(1, 12)
    pages = max(2, min(40, (400 << 20) // (groups * beams * layers * heads * page * D * 2 * e)))
    return dict(kind=kind, groups=groups, beams=beams, layers=layers, heads=heads, D=D, page=page,
                length=rng.randint(1, (pages - 1) * page), dtype=dtype)


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _normal(gen, shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).to(dtype)


def _lengths(gen, rows, longest, ragged):
    """The rows' lengths: all of them `longest`, or spread from 1 to it, the first row's being it."""
    if not ragged:
        return torch.full((rows,), longest, dtype=torch.int32, device="cuda")
    n = (torch.rand(rows, generator=gen, device="cuda") * longest).to(torch.int32) + 1
    n = n.clamp_(max=longest)
    n[0] = longest
    return n


def _cache(gen, case, rows, longest, layers=None, spare=0):
    """Pools, table and page count of a cache whose rows hold up to `longest` positions each; a row's
    pages lie anywhere in the pool."""
    per_row = -(-longest // case["page"])
    pages = rows * per_row + spare
    shape = (pages, case["heads"], case["page"], case["D"])
    shape = shape if layers is None else (layers, *shape)
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    return {"k": _normal(gen, shape, _type(case)), "v": _normal(gen, shape, _type(case)),
            "table": order[:rows * per_row].reshape(rows, per_row).contiguous(), "spare": order[rows * per_row:].clone()}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, s = case["kind"], {"case": case}
    if kind == "append":
        rows, heads, D, new = case["rows"], case["heads"], case["D"], case["new"]
        s["counts"] = _lengths(gen, rows, new, True) if case["ragged"] and new > 1 else None
        before = _lengths(gen, rows, case["before"], case["ragged"]) if case["before"] else 0
        added = s["counts"] if s["counts"] is not None else torch.full((rows,), new, dtype=torch.int32, device="cuda")
        s["lens"] = (added + before).to(torch.int32)  # the lengths with the new tokens
        s.update(_cache(gen, case, rows, case["before"] + new))
        # the projection's output holds a token's keys and values of all heads beside its queries
        qkv = _normal(gen, (rows, new, 3, heads, D), _type(case))
        s["k_new"], s["v_new"] = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
        if case["meta"]:
            cap = s["table"].shape[1] * case["page"]
            s["weights"] = torch.rand((rows, heads, cap), generator=gen, device="cuda")
            s["positions"] = torch.full((rows, heads, cap), -1, dtype=torch.int32, device="cuda")
            s["seen"] = s["lens"] + 100  # a hundred positions were evicted before
    elif kind == "decode":
        rows, heads = case["rows"], case["heads"]
        s["lens"] = _lengths(gen, rows, case["length"], case["ragged"])
        s.update(_cache(gen, case, rows, case["length"]))
        s["q"] = _normal(gen, (rows, heads * case["group"], 1, case["D"]), _type(case), 1.5)
        if case["weigh"]:
            cap = s["table"].shape[1] * case["page"]
            s["weights"] = _normal(gen, (rows, heads, cap)).mul_(1.5).exp_().div_(cap)
            s["weights_out"] = s["weights"].clone()
    elif kind == "evict":
        rows, heads, n = case["rows"], case["heads"], case["length"]
        s["lens"] = _lengths(gen, rows, n, False)
        s.update(_cache(gen, case, rows, n))
        cap = s["table"].shape[1] * case["page"]
        # sums of softmax weights: a few large, most small, some that never had any
        w = _normal(gen, (rows, heads, cap)).mul_(1.5).exp_().div_(cap)
        s["weights"] = w.mul_((torch.rand(w.shape, generator=gen, device="cuda") > 0.05).float())
        # earlier evictions left the positions in about their order
        late = torch.arange(cap, device="cuda") + torch.rand(w.shape, generator=gen, device="cuda") * (0.1 * n)
        s["positions"] = (late.argsort(dim=2).argsort(dim=2) * 2).to(torch.int32)
        s["weights_out"], s["positions_out"] = s["weights"].clone(), s["positions"].clone()
    elif kind == "select":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        s["logits"] = _normal(gen, (groups * beams, vocab), _type(case), 2.0)
        scores = _normal(gen, (groups, beams)) - 20.0
        s["finished"] = (torch.rand((groups, beams), generator=gen, device="cuda") < 0.2).to(torch.int32)
        if case["first"]:
            scores.fill_(-math.inf)
            scores[:, 0] = 0.0
            s["finished"].zero_()
        s["scores"] = scores
    else:
        groups, beams, n = case["groups"], case["beams"], case["length"]
        rows = groups * beams
        s["lens"] = _lengths(gen, rows, n, False)
        s.update(_cache(gen, case, rows, n + case["page"], case["layers"], spare=rows))
        s["parents"] = torch.randint(0, beams, (groups, beams), generator=gen, device="cuda", dtype=torch.int32)
        full = n // case["page"]  # full pages are shared with the beam of the same group that wrote them
        if full:
            writer = torch.randint(0, beams, (groups, beams, full), generator=gen, device="cuda")
            s["table"][:, :full] = s["table"].view(groups, beams, -1)[:, :, :full].gather(1, writer).reshape(rows, full)
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program keeps beside its data: the cache's handle and the calls' workspaces."""
    import inferno_amd as ia

    case, kind = s["case"], s["case"]["kind"]
    if kind == "select":
        s["ws"] = ia.beam_select_workspace(case["groups"], case["beams"], case["vocab"], device="cuda")
        return
    s["cache"] = ia.PagedKV(s["k"], s["v"], s["table"], s["lens"])
    if kind == "decode":
        s["ws"] = ia.attn_decode_paged_workspace(s["cache"], case["heads"] * case["group"], max_len=case["length"],
                                                 weights=case["weigh"])
    if kind == "evict":
        s["ws"] = ia.kv_evict_workspace(s["cache"], case["keep"], max_len=case["length"])


def run(state):
    return (_run_own if own else _PLAIN[state["case"]["kind"]])(state)


def _run_own(s):
    import inferno_amd as ia

    case, kind = s["case"], s["case"]["kind"]
    if kind == "append":
        if not case["meta"]:
            ia.kv_append(s["cache"], s["k_new"], s["v_new"], counts=s["counts"])
            return {"k": s["k"], "v": s["v"]}
        ia.kv_append(s["cache"], s["k_new"], s["v_new"], counts=s["counts"], weights=s["weights"],
                     positions=s["positions"], seen=s["seen"])
        return {"k": s["k"], "v": s["v"], "weights": s["weights"], "positions": s["positions"]}
    if kind == "decode":
        if not case["weigh"]:
            return {"o": ia.attn_decode_paged(s["q"], s["cache"], max_len=case["length"], workspace=s["ws"])}
        o = ia.attn_decode_paged(s["q"], s["cache"], max_len=case["length"], weights=s["weights"],
                                 weights_out=s["weights_out"], workspace=s["ws"])
        return {"o": o, "weights": s["weights_out"]}
    if kind == "evict":
        lens = ia.kv_evict(s["cache"], s["weights"], s["positions"], case["keep"], recent=case["recent"],
                           weights_out=s["weights_out"], positions_out=s["positions_out"], max_len=case["length"],
                           workspace=s["ws"])
        return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "positions": s["positions_out"], "lens": lens}
    if kind == "select":
        tokens, parents, scores, finished = ia.beam_select(s["logits"], s["scores"], finished=s["finished"], eos=EOS,
                                                           workspace=s["ws"])
        return {"tokens": tokens, "parents": parents, "scores": scores, "finished": finished}
    table, spare = ia.beam_reorder(s["cache"], s["parents"], s["spare"])
    return {"k": s["k"], "v": s["v"], "table": table, "spare": spare}


# ---- plain forms ---------------------------------------------------------------------------------


def _plain_append(s):
    rows, heads, new, _ = s["k_new"].shape
    page, cap = s["case"]["page"], s["table"].shape[1] * s["case"]["page"]
    lens = s["lens"].long()[:, None]
    t = torch.arange(new, device="cuda")
    counts = s["counts"].long()[:, None] if s["counts"] is not None else new
    there = t < counts
    slot = lens - counts + t
    row, col = torch.nonzero(there & (slot >= 0) & (slot < cap), as_tuple=True)
    at = slot[row, col]
    where = s["table"].long()[row, at // page]
    s["k"][where, :, at % page] = s["k_new"][row, :, col]
    s["v"][where, :, at % page] = s["v_new"][row, :, col]
    if not s["case"]["meta"]:
        return {"k": s["k"], "v": s["v"]}
    s["weights"][row, :, at] = 0.0
    s["positions"][row, :, at] = (s["seen"].long()[:, None] - counts + t)[row, col][:, None].to(torch.int32)
    return {"k": s["k"], "v": s["v"], "weights": s["weights"], "positions": s["positions"]}


def _rows_of(pool, table, n):
    """The first n positions of every row, [rows, heads, n, D]."""
    pages = table[:, :-(-n // pool.shape[2])].long()
    x = pool[pages]  # [rows, pages, heads, slots, D]
    return x.permute(0, 2, 1, 3, 4).reshape(x.shape[0], x.shape[2], -1, x.shape[4])[:, :, :n]


def _scale(D):
    """1 / sqrt(D) as the library takes it by default (32 bits)."""
    return float(np.float32(1.0) / np.sqrt(np.float32(D)))


def _plain_decode(s):
    n, heads, D = s["case"]["length"], s["case"]["heads"], s["case"]["D"]
    k, v = (_rows_of(s[x], s["table"], n).float() for x in ("k", "v"))
    q = s["q"].float().reshape(-1, heads, s["case"]["group"], D)
    hidden = (torch.arange(n, device="cuda") >= s["lens"][:, None])[:, None, None, :]
    x = torch.matmul(q, k.transpose(2, 3)) * _scale(D)
    x = x.masked_fill(hidden, -math.inf)
    p = torch.exp(x - x.amax(dim=3, keepdim=True))
    p = p / p.sum(dim=3, keepdim=True)
    o = torch.matmul(p, v).reshape(s["q"].shape).to(s["q"].dtype)
    if not s["case"]["weigh"]:
        return {"o": o}
    s["weights_out"][:, :, :n] = torch.where(hidden[:, 0], s["weights_out"][:, :, :n],
                                             s["weights"][:, :, :n] + p.sum(dim=2))
    return {"o": o, "weights": s["weights_out"]}


def _plain_evict(s):
    n, keep, recent, page = s["case"]["length"], s["case"]["keep"], s["case"]["recent"], s["case"]["page"]
    w, pos = s["weights"][:, :, :n], s["positions"][:, :, :n]
    rows, heads = w.shape[:2]
    safe = pos >= pos.amax(dim=2, keepdim=True) + 1 - recent
    # best first: the recent ones, then by weight, the lower slot where weights are equal
    order = torch.where(safe, math.inf, w).argsort(dim=2, descending=True, stable=True)
    kept = torch.zeros((rows, heads, n), dtype=torch.bool, device="cuda").scatter_(2, order[:, :, :min(keep, n)], True)
    # the kept ones behind the cut fill the holes before it, both in their order
    r, h, hole = torch.nonzero(~kept[:, :, :keep], as_tuple=True)
    _, _, src = torch.nonzero(kept[:, :, keep:], as_tuple=True)
    src = src + keep
    table = s["table"].long()
    for pool in (s["k"], s["v"]):
        pool[table[r, hole // page], h, hole % page] = pool[table[r, src // page], h, src % page]
    for x, out in ((s["weights"], s["weights_out"]), (s["positions"], s["positions_out"])):
        out[:, :, :keep] = x[:, :, :keep]
        out[r, h, hole] = x[r, h, src]
    return {"k": s["k"], "v": s["v"], "weights": s["weights_out"], "positions": s["positions_out"],
            "lens": s["lens"].clamp(max=keep)}


def _plain_select(s):
    groups, beams = s["scores"].shape
    vocab = s["logits"].shape[1]
    x = s["logits"].double()  # candidates of different beams can lie close together
    x = x - x.amax(dim=1, keepdim=True)
    x = x - torch.exp(x).sum(dim=1, keepdim=True).log()
    done = s["finished"].reshape(-1, 1) != 0
    x = x.masked_fill(done, -math.inf)
    x[:, EOS] = torch.where(done[:, 0], 0.0, x[:, EOS])  # a finished beam goes on as it is
    x = (x + s["scores"].double().reshape(-1, 1)).reshape(groups, beams * vocab)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    best, at = best[:, :beams], at[:, :beams]
    tokens, parents = (at % vocab).to(torch.int32), (at // vocab).to(torch.int32)
    finished = (s["finished"].gather(1, parents.long()) != 0) | (tokens == EOS)
    return {"tokens": tokens, "parents": parents, "scores": best.float(), "finished": finished.to(torch.int32)}


def _plain_reorder(s):
    n, page = s["case"]["length"], s["case"]["page"]
    groups, beams = s["parents"].shape
    full, part = n // page, n % page
    me = torch.arange(groups * beams, device="cuda")
    parent = (s["parents"].long() + torch.arange(groups, device="cuda")[:, None] * beams).reshape(-1)
    table, spare = s["table"].clone(), s["spare"].clone()
    table[:, :full] = s["table"][parent, :full]
    if part:
        moves = torch.nonzero(parent != me)[:, 0]
        src, dst = s["table"][parent[moves], full].long(), s["spare"][moves].long()
        for pool in (s["k"], s["v"]):
            pool[:, dst, :, :part] = pool[:, src, :, :part]
        table[moves, full] = s["spare"][moves]
        spare[moves] = s["table"][moves, full]
    return {"k": s["k"], "v": s["v"], "table": table, "spare": spare}


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "evict": _plain_evict, "select": _plain_select,
          "reorder": _plain_reorder}


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    kind, e = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind == "append":
        # ragged counts spread evenly from 1 to `new`
        tokens = case["rows"] * ((case["new"] + 1) / 2 if case["ragged"] else case["new"])
        return {"bytes": tokens * case["heads"] * (4 * case["D"] * e + (8 if case["meta"] else 0)), "flops": 0}
    if kind == "decode":
        keys = case["rows"] * case["heads"] * ((case["length"] + 1) / 2 if case["ragged"] else case["length"])
        ends = 2 * case["rows"] * case["heads"] * case["group"] * case["D"] * e
        return {"bytes": keys * (2 * case["D"] * e + (8 if case["weigh"] else 0)) + ends,
                "flops": 4 * keys * case["group"] * case["D"]}
    if kind == "evict":
        n, keep = case["length"], case["keep"]
        # the evicted ones that lie before the cut, if they are spread evenly over the old positions,
        # which are mostly those before the last `recent`
        old = max(n - case["recent"], 1)
        holes = (n - keep) * min(keep, old) / old
        per_head = 8 * (n + keep) + holes * 4 * case["D"] * e
        return {"bytes": case["rows"] * case["heads"] * per_head, "flops": case["rows"] * case["heads"] * n}
    if kind == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * e, "flops": 4 * n}
    rows, part = case["groups"] * case["beams"], case["length"] % case["page"]
    moved = case["groups"] * (case["beams"] - 1)  # one beam in `beams` stays its own parent
    pages = rows * (case["length"] // case["page"] + 2)
    return {"bytes": 4 * case["layers"] * moved * case["heads"] * part * case["D"] * e + 8 * pages, "flops": 0}


# ---- the same in 64 bits -------------------------------------------------------------------------


def exact(case, seed):
    return _EXACT[case["kind"]](case, prepare(case, seed))


def _exact_append(case, s):
    k, v = s["k"].double(), s["v"].double()
    out = {"k": k, "v": v}
    if case["meta"]:
        out.update(weights=s["weights"].double(), positions=s["positions"])
    lens, table = s["lens"].tolist(), s["table"].tolist()
    for row in range(case["rows"]):
        count = case["new"] if s["counts"] is None else int(s["counts"][row])
        first, t = lens[row] - count, 0
        while t < count:  # page by page
            at = (first + t) % case["page"]
            m = min(count - t, case["page"] - at)
            where = table[row][(first + t) // case["page"]]
            k[where, :, at:at + m] = s["k_new"][row, :, t:t + m].double()
            v[where, :, at:at + m] = s["v_new"][row, :, t:t + m].double()
            t += m
        if case["meta"]:
            out["weights"][row, :, first:first + count] = 0.0
            out["positions"][row, :, first:first + count] = torch.arange(
                int(s["seen"][row]) - count, int(s["seen"][row]), device="cuda", dtype=torch.int32)
    return out


def _exact_decode(case, s):
    # row by row, head by head, page after page
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights_out"].double() if case["weigh"] else None
    for row, n in enumerate(s["lens"].tolist()):
        pages = s["table"][row, :-(-n // case["page"])].long()
        for h in range(case["heads"]):
            k = s["k"][pages, h].reshape(-1, case["D"])[:n].double()
            v = s["v"][pages, h].reshape(-1, case["D"])[:n].double()
            mine = slice(h * case["group"], (h + 1) * case["group"])
            p = torch.softmax((s["q"][row, mine].double() * k).sum(-1) * _scale(case["D"]), dim=-1)
            o[row, mine, 0] = (p[:, :, None] * v).sum(1)
            if case["weigh"]:
                weights[row, h, :n] = s["weights"][row, h, :n].double() + p.sum(0)
    return {"o": o, "weights": weights} if case["weigh"] else {"o": o}


def _exact_evict(case, s):
    n, keep, page = case["length"], case["keep"], case["page"]
    w, pos = s["weights"].cpu().numpy(), s["positions"].cpu().numpy()
    k, v = s["k"].double(), s["v"].double()
    w_out, pos_out = s["weights_out"].double().cpu().numpy(), s["positions_out"].cpu().numpy()
    table = s["table"].cpu().numpy().astype(np.int64)
    for row in range(case["rows"]):
        for h in range(case["heads"]):
            wn, pn = w[row, h, :n].astype(np.float64), pos[row, h, :n].astype(np.int64)
            old = pn <= pn.max() - case["recent"]
            worst = np.lexsort((-np.arange(n), wn, ~old))  # the old before the recent, then the least weight
            gone = set(worst[:max(n - keep, 0)].tolist())
            holes = [i for i in range(min(keep, n)) if i in gone]
            src = [i for i in range(keep, n) if i not in gone]
            w_out[row, h, :keep], pos_out[row, h, :keep] = w[row, h, :keep], pos[row, h, :keep]
            if not holes:
                continue
            a, b = np.array(holes), np.array(src)
            w_out[row, h, a], pos_out[row, h, a] = w[row, h, b], pos[row, h, b]
            to, at = (torch.from_numpy(x).cuda() for x in (table[row, a // page], a % page))
            of, by = (torch.from_numpy(x).cuda() for x in (table[row, b // page], b % page))
            for pool in (k, v):
                pool[to, h, at] = pool[of, h, by]
    return {"k": k, "v": v, "weights": torch.from_numpy(w_out).cuda(), "positions": torch.from_numpy(pos_out).cuda(),
            "lens": torch.full((case["rows"],), min(n, keep), dtype=torch.int32, device="cuda")}


def _exact_select(case, s):
    groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
    logits = s["logits"].float().cpu().numpy().astype(np.float64).reshape(groups, beams, vocab)
    scores, done = s["scores"].cpu().numpy().astype(np.float64), s["finished"].cpu().numpy()
    out = {name: np.zeros((groups, beams), t) for name, t in
           (("tokens", np.int32), ("parents", np.int32), ("scores", np.float64), ("finished", np.int32))}
    for g in range(groups):
        found = []
        for b in range(beams):
            if done[g, b]:
                found.append((-scores[g, b], b, EOS))
                continue
            row = logits[g, b]
            lse = row.max() + np.log(np.exp(row - row.max()).sum())
            best = np.argsort(-row, kind="stable")[:beams]
            found += [(-(scores[g, b] + row[t] - lse), b, int(t)) for t in best]
        for i, (score, b, t) in enumerate(sorted(found)[:beams]):
            out["tokens"][g, i], out["parents"][g, i], out["scores"][g, i] = t, b, -score
            out["finished"][g, i] = int(bool(done[g, b]) or t == EOS)
    return {name: torch.from_numpy(x).cuda() for name, x in out.items()}


def _exact_reorder(case, s):
    n, page, beams = case["length"], case["page"], case["beams"]
    k, v = s["k"].double(), s["v"].double()
    table, spare = s["table"].tolist(), s["spare"].tolist()
    table_out, spare_out = [list(r) for r in table], list(spare)
    for row, p in enumerate(s["parents"].reshape(-1).tolist()):
        parent = row // beams * beams + p
        for i in range(n // page):
            table_out[row][i] = table[parent][i]
        if parent != row and n % page:
            src, dst = table[parent][n // page], spare[row]
            for pool, given in ((k, s["k"]), (v, s["v"])):
                pool[:, dst, :, :n % page] = given[:, src, :, :n % page].double()
            table_out[row][n // page], spare_out[row] = dst, table[row][n // page]
    return {"k": k, "v": v, "table": torch.tensor(table_out, dtype=torch.int32, device="cuda"),
            "spare": torch.tensor(spare_out, dtype=torch.int32, device="cuda")}


_EXACT = {"append": _exact_append, "decode": _exact_decode, "evict": _exact_evict, "select": _exact_select,
          "reorder": _exact_reorder}
