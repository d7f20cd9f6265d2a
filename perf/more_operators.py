"""Generation with weights in 8 bits and a paged key-value cache in 4 bits, as cases that can be timed: the
linear layer whose inputs are quantised token by token, keys and values written to the cache and read back, and
attention of one new token per sequence over it.

``listed()`` holds the named cases, ``draw(rng)`` gives further ones of the same ranges.
``prepare(case, seed)`` makes the inputs on the GPU and ``run(state)`` is one pass: through the
framework's entry points where ``own`` is true, else in elementary torch operations.
``exact(case, seed)`` is the same pass in 64 bits, ``work(case)`` the bytes and operations that it
cannot do without.

8 bits: a row's scale is its largest magnitude times 1/127, its values are whole multiples of it.
4 bits: blocks of 32 channels share a power of two, 2^(byte - 127); a value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6
times it, with a sign (bit 3).  Byte i of a row holds channel 2 i in its low half, 2 i + 1 in its high one.
A cache is pools of pages [pages, key-value heads, slots, D / 2] of such bytes and [pages, heads, D / 32, slots]
of scales for the keys and for the values, a table [rows, pages of a row] that names each row's pages, and the
rows' lengths.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

INV127 = float(np.float32(1.0) / np.float32(127.0))


def listed():
    return [
        # The projection to queries, keys and values of one sequence's new token: the smallest call.
        dict(name="linear_one_f32", kind="linear", M=1, K=768, N=2304, bias=True, dtype="f32"),
        # A serving batch's new tokens through the up-projection of a larger model: the weights' bytes count.
        dict(name="linear_step_bf16", kind="linear", M=32, K=4096, N=16384, bias=False, dtype="bf16"),
        # A few prompts of odd lengths through the same width.
        dict(name="linear_chunk_bf16", kind="linear", M=333, K=4096, N=4096, bias=True, dtype="bf16"),
        # The prompts of a batch of 8 x 1024 tokens on the small model.
        dict(name="linear_prompt_f32", kind="linear", M=8192, K=768, N=2304, bias=True, dtype="f32"),
        # Long prompts on a large model: the matrix cores.
        dict(name="linear_large_bf16", kind="linear", M=16384, K=8192, N=8192, bias=False, dtype="bf16"),
        # One decoding step of a serving batch writes each sequence's new key and value; what was written is read.
        dict(name="kv4_step_bf16", kind="kv4", rows=64, heads=8, D=128, page=16, new=1, before=1500, ragged=True,
             whole=False, dtype="bf16"),
        # The prompts of a batch go into the cache, and out again for the attention of what follows them.
        dict(name="kv4_prompts_f32", kind="kv4", rows=8, heads=12, D=64, page=32, new=1024, before=0, ragged=True,
             whole=True, dtype="f32"),
        # The next 512 tokens of long prompts go in; all that is before them comes out for their attention.
        dict(name="kv4_prefix_bf16", kind="kv4", rows=16, heads=8, D=128, page=64, new=512, before=4000, ragged=False,
             whole=True, dtype="bf16"),
        # One sequence, one new token: latency.
        dict(name="kv4_decode_one_f32", kind="decode", rows=1, heads=12, group=1, D=64, page=16, length=1000,
             ragged=False, dtype="f32"),
        # A batch of the small model at the end of its context.
        dict(name="kv4_decode_batch_f32", kind="decode", rows=32, heads=12, group=1, D=64, page=64, length=2048,
             ragged=False, dtype="f32"),
        # Serving with shared key-value heads, sequences of all lengths up to 8 thousand.
        dict(name="kv4_decode_ragged_bf16", kind="decode", rows=64, heads=8, group=4, D=128, page=16, length=8191,
             ragged=True, dtype="bf16"),
        # Long documents with few key-value heads.
        dict(name="kv4_decode_long_bf16", kind="decode", rows=4, heads=2, group=8, D=128, page=128, length=131071,
             ragged=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over their logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "kv4", "decode", "decode"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "linear":
        K, N = _log(rng, 64, 16384), _log(rng, 64, 16384)
        if rng.random() < 0.6:  # most layers are multiples of 64 wide
            K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
        # the largest product and the most bytes are the largest listed case's
        most = min(16384, (1 << 40) // (K * N), (800 << 20) // (4 * (K + N)))
        return dict(kind=kind, M=_log(rng, 1, max(1, most)), K=K, N=N, bias=rng.random() < 0.5, dtype=dtype)
    D, page = rng.choice([32, 64, 128]), rng.choice([16, 32, 64, 128])
    rows, heads = _log(rng, 1, 64), rng.randint(1, 16)
    if kind == "kv4":
        new = _log(rng, 1, max(1, min(2048, (16 << 20) // (rows * heads * D))))
        before = _log(rng, 1, max(1, min(8000, (48 << 20) // (rows * heads * D)))) if rng.random() < 0.8 else 0
        return dict(kind=kind, rows=rows, heads=heads, D=D, page=page, new=new, before=before,
                    ragged=rng.random() < 0.5, whole=rng.random() < 0.5, dtype=dtype)
    length = _log(rng, 1, max(1, min(131072, (512 << 20) // (rows * heads * D))))
    return dict(kind=kind, rows=rows, heads=heads, group=rng.choice([1, 1, 2, 3, 4, 5, 8, 12, 16]), D=D, page=page,
                length=length, ragged=rng.random() < 0.5, dtype=dtype)


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


def _hidden(gen, shape, dtype):
    """A layer's activations: normal, a few channels far larger than the others, tokens of different sizes."""
    x = _normal(gen, shape)
    x *= torch.exp(_normal(gen, (shape[0], 1), std=0.5))
    x *= 1 + 15 * (torch.rand(shape[1], generator=gen, device="cuda") < 0.004)
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = _hidden(gen, (M, K), _type(case))
        weight = _normal(gen, (K, N), std=K ** -0.5)  # as a layer trained in 32 bits holds it
        s["bias"] = _normal(gen, (N,), _type(case), 0.1) if case["bias"] else None
        if own:  # the weights are laid out once, the workspace is kept
            import inferno_amd as ia

            s["w"], s["w_scale"] = ia.quantize_i8(weight, transpose=True)
            s["ws"] = ia.linear_i8_workspace(M, N, K, device="cuda")
        else:
            s["w"], s["w_scale"] = _quantize(weight.t())
        return s
    rows, heads, D, page = case["rows"], case["heads"], case["D"], case["page"]
    if case["kind"] == "kv4":
        before = _lengths(gen, rows, case["before"], case["ragged"]) if case["before"] else 0
        s["counts"] = _lengths(gen, rows, case["new"], True) if case["ragged"] and case["new"] > 1 else None
        added = s["counts"] if s["counts"] is not None else torch.full((rows,), case["new"], dtype=torch.int32,
                                                                       device="cuda")
        s["lens"] = (added + before).to(torch.int32)  # the lengths with the new tokens
        s["first"] = None if case["whole"] else s["lens"] - added
        longest = case["before"] + case["new"]
        # the projection's output holds a token's keys and values of all heads beside its queries
        qkv = _normal(gen, (rows, case["new"], 3, heads, D), _type(case))
        s["k_new"], s["v_new"] = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    else:
        s["lens"] = _lengths(gen, rows, case["length"], case["ragged"])
        longest = case["length"]
        s["q"] = _normal(gen, (rows, heads * case["group"], 1, D), _type(case), 1.5)
    # a row's pages lie anywhere in the pool
    per_row = -(-longest // page)
    order = torch.randperm(rows * per_row, generator=gen, device="cuda").to(torch.int32)
    s["table"] = order.reshape(rows, per_row).contiguous()
    for name in ("k", "v"):
        codes = torch.empty((rows * per_row, heads, page, D // 2), dtype=torch.uint8, device="cuda")
        scales = torch.empty((rows * per_row, heads, D // 32, page), dtype=torch.uint8, device="cuda")
        for i in range(0, rows * per_row, 1 + (64 << 20) // (heads * page * D)):
            part = slice(i, i + 1 + (64 << 20) // (heads * page * D))
            codes[part], scale = _encode(_normal(gen, (*codes[part].shape[:3], D)))
            scales[part] = scale.transpose(2, 3)
        s[name], s[name + "_scale"] = codes, scales
    if own:
        import inferno_amd as ia

        s["cache"] = ia.PagedKV4(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["lens"])
        if case["kind"] == "decode":
            s["ws"] = ia.attn_decode_kv4_workspace(s["cache"], heads * case["group"], max_len=case["length"])
    return s


def run(state):
    return (_run_own if own else _PLAIN[state["case"]["kind"]])(state)


def _run_own(s):
    import inferno_amd as ia

    case = s["case"]
    if case["kind"] == "linear":
        return {"y": ia.linear_i8(s["x"], s["w"], s["w_scale"], bias=s["bias"], workspace=s["ws"])}
    if case["kind"] == "kv4":
        ia.kv4_append(s["cache"], s["k_new"], s["v_new"], counts=s["counts"])
        k, v = ia.kv4_read(s["cache"], _positions(case), first=s["first"], dtype=_type(case))
        return {"k": k, "v": v}
    return {"o": ia.attn_decode_kv4(s["q"], s["cache"], max_len=case["length"], workspace=s["ws"])}


def _positions(case):
    """How many positions of a row are read back."""
    return case["new"] + (case["before"] if case["whole"] else 0)


# ---- plain forms ---------------------------------------------------------------------------------


def _quantize(x):
    """Rows in 8 bits: whole numbers (as int8) and the rows' scales."""
    x = x.float()
    scale = x.abs().amax(dim=1) * INV127
    # values next to the middle between two whole numbers need more than 32 bits
    q = torch.round(x.double() / scale.double()[:, None]).clamp(-127, 127)
    return q.to(torch.int8), scale


def _plain_linear(s):
    q, scale = _quantize(s["x"])
    y = torch.matmul(q.float(), s["w"].float().t()) * scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"y": y.to(s["x"].dtype)}


def _power(e):
    """2^e in 32 bits, -126 <= e <= 127."""
    return ((e + 127) << 23).view(torch.float32)


def _encode(x):
    """[..., D] in 4 bits: bytes [..., D / 2] and scales [..., D / 32]."""
    x = x.float().reshape(*x.shape[:-1], -1, 32)
    top = x.abs().amax(dim=-1)
    e = (torch.frexp(top).exponent - 3).clamp(min=-125)  # the largest comes to lie in [4, 8)
    y = x.abs() * _power(-e)[..., None]
    # the grid 0, 0.5, 1, 1.5, 2, 3, 4, 6: to the nearest, ties to the even code
    code = ((y > 0.25).byte() + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = (code | (torch.signbit(x).byte() << 3)).reshape(*x.shape[:-2], -1)
    return code[..., ::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _decode(codes, scales):
    """The values of bytes and scales, in 32 bits."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    grid = torch.cat((grid, -grid))
    x = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), dim=-1)
    x = x.reshape(*scales.shape, 32) * _power(scales.int() - 127)[..., None]
    return x.reshape(*scales.shape[:-1], -1)


def _rows_of(s, name, n):
    """The first n positions of every row, [rows, heads, n, D]."""
    pages = s["table"][:, :-(-n // s["case"]["page"])].long()
    codes = s[name][pages].permute(0, 2, 1, 3, 4)  # [rows, heads, pages, slots, bytes]
    scales = s[name + "_scale"][pages].permute(0, 2, 1, 4, 3)
    return _decode(*(x.reshape(*x.shape[:2], -1, x.shape[4])[:, :, :n] for x in (codes, scales)))


def _plain_kv4(s):
    case, page = s["case"], s["case"]["page"]
    lens = s["lens"].long()[:, None]
    t = torch.arange(case["new"], device="cuda")
    counts = s["counts"].long()[:, None] if s["counts"] is not None else case["new"]
    row, col = torch.nonzero((t < counts).expand(case["rows"], -1), as_tuple=True)
    at = (lens - counts + t)[row, col]
    where = s["table"].long()[row, at // page]
    for name in ("k", "v"):
        codes, scales = _encode(s[name + "_new"][row, :, col])
        s[name][where, :, at % page] = codes
        s[name + "_scale"][where, :, :, at % page] = scales
    j = torch.arange(_positions(case), device="cuda")
    j = j if case["whole"] else j + s["first"].long()[:, None]
    there = (j < lens).expand(case["rows"], -1)
    j = torch.where(there, j, 0)
    out = {}
    for name in ("k", "v"):
        pages = s["table"].long().gather(1, j // page)
        x = _decode(s[name][pages, :, j % page], s[name + "_scale"][pages, :, :, j % page])  # [rows, T, heads, D]
        x = x.masked_fill(~there[:, :, None, None], 0.0)  # nothing behind a row's end
        out[name] = x.transpose(1, 2).to(s[name + "_new"].dtype).contiguous()
    return out


def _scale(D):
    """1 / sqrt(D) as the library takes it by default (32 bits)."""
    return float(np.float32(1.0) / np.sqrt(np.float32(D)))


def _plain_decode(s):
    n, heads, D = s["case"]["length"], s["case"]["heads"], s["case"]["D"]
    k, v = (_rows_of(s, x, n) for x in ("k", "v"))
    q = s["q"].float().reshape(-1, heads, s["case"]["group"], D)
    hidden = (torch.arange(n, device="cuda") >= s["lens"][:, None])[:, None, None, :]
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * _scale(D)
    x = x.masked_fill(hidden, -math.inf)
    p = torch.exp(x - x.amax(dim=3, keepdim=True))
    p = p / p.sum(dim=3, keepdim=True)
    return {"o": torch.matmul(p, v).reshape(s["q"].shape).to(s["q"].dtype)}


_PLAIN = {"linear": _plain_linear, "kv4": _plain_kv4, "decode": _plain_decode}


# ---- the passes' needs -----------------------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": e * M * (K + N) + N * (K + 4) + (e * N if case["bias"] else 0), "flops": 2 * M * K * N}
    rows, heads, D = case["rows"], case["heads"], case["D"]
    held = D // 2 + D // 32  # bytes of a position's key or value of one head
    if case["kind"] == "kv4":
        # ragged rows lie evenly between one position and the most
        n, m = case["new"], _positions(case)
        if case["ragged"]:
            n, m = (1 if x == 1 else (x + 1) / 2 for x in (n, m))
        moved = n * (e * D + held) + m * (held + e * D)
        return {"bytes": int(2 * rows * heads * moved), "flops": int(2 * rows * heads * D * (2 * n + m))}
    n = case["length"] if not case["ragged"] else (case["length"] + 1) / 2
    qo = 2 * e * rows * heads * case["group"] * D
    return {"bytes": int(2 * rows * heads * n * held) + qo, "flops": int(4 * rows * heads * case["group"] * D * n)}


# ---- the passes in 64 bits, from the formulas ---------------------------------------------------------


def exact(case, seed):
    global own
    mine, own = own, False  # the inputs alone
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return _EXACT[case["kind"]](case, s)


def _exact_linear(case, s):
    # value by value: |x| / scale lies between whole numbers a and a + 1, and goes to the nearer, the even one of two
    w, sw = s["w"].double(), s["w_scale"].double()
    y = torch.empty((case["M"], case["N"]), dtype=torch.float64, device="cuda")
    for i in range(0, case["M"], 2048):
        x = s["x"][i:i + 2048].double()
        scale = (x.abs().max(dim=1).values.float() * torch.tensor(INV127, device="cuda")).double()[:, None]
        a = torch.floor(x.abs() / scale)
        over = x.abs() - a * scale - scale / 2  # exact: all three are multiples of one small power of two
        a = a + ((over > 0) | ((over == 0) & (a % 2 == 1))).double()
        q = a.clamp(max=127) * torch.sign(x)
        y[i:i + 2048] = torch.matmul(q, w.t()) * scale * sw
    return {"y": y if s["bias"] is None else y + s["bias"].double()}


def _nearest(x):
    """Blocks [..., 32] on their 4-bit grids, in 64 bits: the values that they are held as."""
    x = x.double()
    top = x.abs().amax(dim=-1, keepdim=True)
    e = torch.floor(torch.log2(top))
    # log2 may round across a whole number
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, torch.where(torch.exp2(e) > top, e - 1, e))
    unit = torch.exp2((e - 2).clamp(min=-125))
    y = (x.abs() / unit).clamp(max=6.0)
    # steps of a half below 2, of one below 4, of two from there on; torch.round takes ties to even
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    return torch.round(y / step) * step * unit * torch.sign(x)


def _values(codes, scales):
    """What bytes and scales stand for, in 64 bits: sign, two bits of exponent, one of mantissa."""
    c = torch.stack((codes % 16, codes // 16), dim=-1).reshape(*codes.shape[:-1], -1).long()
    exponent, mantissa = (c % 8) // 2, (c % 2).double()
    x = torch.where(exponent > 0, torch.exp2(exponent.double() - 1) * (1 + mantissa / 2), mantissa / 2)
    x = torch.where(c >= 8, -x, x)
    return x * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def _exact_kv4(case, s):
    T = _positions(case)
    out = {name: torch.zeros((case["rows"], case["heads"], T, case["D"]), dtype=torch.float64, device="cuda")
           for name in ("k", "v")}
    for row, n in enumerate(s["lens"].tolist()):
        count = case["new"] if s["counts"] is None else int(s["counts"][row])
        first = 0 if case["whole"] else n - count
        pages = s["table"][row].long()
        for name in ("k", "v"):
            if n - count > first:  # what was there before
                x = _values(s[name][pages], s[name + "_scale"][pages].transpose(2, 3))
                x = x.permute(1, 0, 2, 3).reshape(case["heads"], -1, case["D"])
                out[name][row, :, :n - count - first] = x[:, first:n - count]
            new = s[name + "_new"][row, :, :count]
            x = _nearest(new.reshape(case["heads"], count, -1, 32)).reshape(new.shape)
            out[name][row, :, n - count - first:n - first] = x
    return out


def _exact_decode(case, s):
    # row by row, head by head, page after page
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for row, n in enumerate(s["lens"].tolist()):
        pages = s["table"][row, :-(-n // case["page"])].long()
        for h in range(case["heads"]):
            k, v = (_values(s[x][pages, h].reshape(-1, case["D"] // 2)[:n],
                            s[x + "_scale"][pages, h].transpose(1, 2).reshape(-1, case["D"] // 32)[:n])
                    for x in ("k", "v"))
            mine = slice(h * case["group"], (h + 1) * case["group"])
            p = torch.softmax((s["q"][row, mine].double() * k).sum(-1) * _scale(case["D"]), dim=-1)
            o[row, mine, 0] = (p[:, :, None] * v).sum(1)
    return {"o": o}


_EXACT = {"linear": _exact_linear, "kv4": _exact_kv4, "decode": _exact_decode}
