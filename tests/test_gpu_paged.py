"""Generation from a paged key-value cache on the GPU against plain implementations in 64 bits on the
CPU: append, attention of one new token, eviction, beam selection and reordering, each at the
sizes, masks and layouts where it can go wrong, and a beam search of all of them together.

Tolerances.  A score's fp32 error: D products summed in any order, each sum off by at most 2^-24
of the products' absolute sum A = sum |q_d k_d| scale, so (D + 2) 2^-24 A; scaling and the
exponent's argument round it twice more.  A probability moves by that times itself, twice
(its own and the sum's); v_exp_f32 adds 2^-22, sums over n keys in chains of at most n / 16 + 64 additions
2^-24 each.  bf16 probabilities are held in two parts (2^-16), bf16 results round by 2^-8.  What is
copied, selected or counted has to be equal.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ia():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_amd

    inferno_amd.lib()
    return inferno_amd


def rnd(gen, shape, dtype=F32, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(dtype)


def make_cache(ia, gen, lens, heads, D, page, dtype, max_pages=None, spare=3, layout="heads", layers=None):
    """A cache of random rows on the GPU, its unused slots and pages NaN and the table entries behind
    a row's length no page at all; also the rows' keys and values in 64 bits, per row [heads, len, D]."""
    rows = len(lens)
    max_pages = max_pages or max(1, -(-max(lens) // page))
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((rows, max_pages), -7, dtype=torch.int32)
    shape = (pages, heads, page, D) if layers is None else (layers, pages, heads, page, D)
    k, v = torch.full(shape, math.nan, dtype=dtype), torch.full(shape, math.nan, dtype=dtype)
    ks, vs = [], []
    for r, n in enumerate(lens):
        mine = [order.pop() for _ in range(need[r])]
        table[r, :need[r]] = torch.tensor(mine, dtype=torch.int32)
        kr, vr = (rnd(gen, (*shape[:-4], heads, n, D), dtype) for _ in range(2))
        for i, p in enumerate(mine):
            m = min(page, n - i * page)
            k[..., p, :, :m, :], v[..., p, :, :m, :] = (x[..., i * page:i * page + m, :] for x in (kr, vr))
        ks.append(kr.double())
        vs.append(vr.double())
    if layout == "slots":  # [pages, slots, heads, D] in memory
        k, v = (x.transpose(-2, -3).contiguous().cuda().transpose(-2, -3) for x in (k, v))
    elif layout == "joint":  # keys and values of a page side by side
        both = torch.stack((k, v), dim=k.dim() - 3).cuda()
        k, v = both.unbind(dim=k.dim() - 3)
    else:
        k, v = k.cuda(), v.cuda()
    c = ia.PagedKV(k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    return c, ks, vs, torch.tensor(order, dtype=torch.int32)


def ref_decode(q, ks, vs, heads, scale):
    """(o, p per row [q_heads, len], bound per row and head) in 64 bits."""
    rows, hq, _, D = q.shape
    g = hq // heads
    o, ps, err = torch.zeros(rows, hq, D, dtype=torch.float64), [], torch.zeros(rows, hq, 1, dtype=torch.float64)
    for r in range(rows):
        n = ks[r].shape[1]
        kk, vv = ks[r].repeat_interleave(g, 0), vs[r].repeat_interleave(g, 0)
        s = (q[r].double() @ kk.transpose(1, 2))[:, 0] * scale
        p = torch.softmax(s, dim=1) if n else s
        ps.append(p)
        if n:
            o[r] = (p[:, None] @ vv)[:, 0]
            a = ((q[r].double().abs() @ kk.abs().transpose(1, 2))[:, 0] * scale).nan_to_num(posinf=0.0)
            a = a.amax(1)[:, None]
            rel = 2 * ((D + 2) * 2.0**-24 * a + 3 * 2.0**-24 * 1.5 * a) + 2.0**-22 + (n / 16 + 64) * 2.0**-24
            err[r] = rel * (p[:, None] @ vv.abs())[:, 0].amax(1)[:, None]
            ps[-1] = (p, rel)
    return o, ps, err


def check_decode(q, out, ks, vs, heads, scale, dtype, skip=()):
    o, ps, err = ref_decode(q, ks, vs, heads, scale)
    got = out[:, :, 0].double().cpu()
    if dtype == BF16:
        # 2^-16 of the sum of |p v|, bounded as err's own factor is (>= 64 2^-24 of it)
        err = err * (1 + 2.0**-16 / (64 * 2.0**-24)) + o.abs() * 2.0**-8
    bad = (got - o).abs() > err + 1e-30
    for r in range(q.shape[0]):
        if r not in skip:
            assert not bad[r].any(), (r, ks[r].shape, float((got[r] - o[r]).abs().max()), float(err[r].max()))
    return ps


DECODE = [
    # heads, group, page, max_pages, lengths
    (2, 1, 16, 9, (0, 1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 144)),
    (1, 4, 1, None, (1, 5, 40, 131)),
    (3, 2, 2, None, (3, 64, 65)),
    (2, 3, 4, 70, (277, 100, 0)),
    (2, 5, 8, None, (7, 8, 9, 300)),
    (1, 16, 32, None, (50, 1000)),
    (2, 17, 64, None, (65, 200)),      # two tiles of query heads
    (1, 33, 16, None, (100,)),
    (12, 1, 16, 80, (1000,)),
    (2, 8, 128, 40, (5000, 3, 0, 1111)),
    (1, 2, 1024, 2, (1, 1025, 2048)),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("heads,group,page,max_pages,lens", DECODE)
def test_decode(ia, heads, group, page, max_pages, lens, D, dtype):
    print(f"[case] paged decode {heads}x{group} page {page} {lens} D{D} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(len(lens) * 100 + D)
    c, ks, vs, _ = make_cache(ia, gen, list(lens), heads, D, page, dtype, max_pages)
    q = rnd(gen, (len(lens), heads * group, 1, D), dtype, 1.5)
    scale = ia.default_scale(D)
    w_in = torch.rand(c.rows, heads, c.capacity, generator=gen)
    w_out = torch.full((c.rows, heads, c.capacity), -5.0, device="cuda")
    out = ia.attn_decode_paged(q.cuda(), c)
    out_w = ia.attn_decode_paged(q.cuda(), c, weights=w_in.cuda(), weights_out=w_out)
    ps = check_decode(q, out, ks, vs, heads, scale, dtype)
    check_decode(q, out_w, ks, vs, heads, scale, dtype)
    w_out = w_out.double().cpu()
    for r, n in enumerate(lens):
        assert (w_out[r, :, n:] == -5.0).all()
        if not n:
            assert (out[r] == 0).all() and (out_w[r] == 0).all()
            continue
        p, rel = ps[r]
        want = w_in[r, :, :n].double() + p.view(heads, group, n).sum(1)
        bound = (rel * p).view(heads, group, n).sum(1) + (group + 1) * 2.0**-24 * want
        assert ((w_out[r, :, :n] - want).abs() <= bound).all(), r
    # in place, and this step's weights alone
    w = w_in.cuda()
    ia.attn_decode_paged(q.cuda(), c, weights=w, weights_out=w)
    for r, n in enumerate(lens):
        assert torch.equal(w[r, :, :n].cpu().double(), w_out[r, :, :n])
        assert torch.equal(w[r, :, n:].cpu(), w_in[r, :, n:])
    w.fill_(7.0)
    ia.attn_decode_paged(q.cuda(), c, weights_out=w)
    for r, n in enumerate(lens):
        if n:
            sums = w[r, :, :n].double().sum(1).cpu()
            assert ((sums - group).abs() <= group * (ps[r][1].max() + n * 2.0**-24)).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,group,D,page,longest,weigh", [
    (150, 2, 1, 64, 16, 700, False),    # three blocks of rows, in shares
    (130, 1, 17, 32, 8, 1100, True),    # two tiles of query heads, with weights
    (64, 3, 2, 128, 32, 400, False),    # a block that is just full
    (65, 1, 1, 128, 16, 300, True),
    (700, 4, 1, 32, 16, 520, False),    # many short rows: whole ones to the workgroups
    (600, 2, 18, 64, 64, 100, False),   # ... of one step, in two tiles of query heads
])
def test_decode_many_rows(ia, rows, heads, group, D, page, longest, weigh, dtype):
    """Rows of random lengths, a third of them empty, some next to each other."""
    print(f"[case] paged decode {rows} rows {heads}x{group} D{D} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(rows)
    lens = (torch.rand(rows, generator=gen) * longest).long() + 1
    lens[torch.rand(rows, generator=gen) < 0.3] = 0
    lens[-5:] = 0
    lens[1] = longest
    lens = lens.tolist()
    c, ks, vs, _ = make_cache(ia, gen, lens, heads, D, page, dtype)
    q = rnd(gen, (rows, heads * group, 1, D), dtype, 1.5)
    w = torch.full(c.meta_shape, -5.0, device="cuda") if weigh else None
    out = ia.attn_decode_paged(q.cuda(), c, max_len=longest, weights_out=w)
    ps = check_decode(q, out, ks, vs, heads, ia.default_scale(D), dtype)
    for r, n in enumerate(lens):
        if not n:
            assert (out[r] == 0).all()
        elif weigh:
            p, rel = ps[r]
            want, bound = p.view(heads, group, n).sum(1), (rel * p).view(heads, group, n).sum(1)
            assert ((w[r, :, :n].double().cpu() - want).abs() <= bound + (group + 1) * 2.0**-24 * want).all(), r
        if weigh:
            assert (w[r, :, n:] == -5.0).all()
    c.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")  # nothing in any row
    assert (ia.attn_decode_paged(q.cuda(), c, max_len=longest, weights_out=w) == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,group,D,lens", [
    (96, 16, 32, (2500, 1, 1800)), (96, 4, 64, (4000, 3000)), (128, 12, 128, (900, 0, 1500)),
])
def test_decode_weights_of_long_shares(ia, heads, group, D, lens, dtype):
    """Workgroups with many steps of several rows: the weights as from a cache of one head, whose workgroups have
    one step each.  Scores and maxima are the same bits; sums of up to n probabilities, in any order and joined
    from parts, are n 2^-24 off at most on either side, and so is each probability relative to itself."""
    print(f"[case] paged decode long shares {heads}x{group} D{D} {lens} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(heads + D)
    rows = len(lens)
    c, _, _, _ = make_cache(ia, gen, list(lens), heads, D, 16, dtype)
    q = rnd(gen, (rows, heads * group, 1, D), dtype, 1.5).cuda()
    w = torch.full(c.meta_shape, -5.0, device="cuda")
    out = ia.attn_decode_paged(q, c, weights_out=w)
    assert out.isfinite().all()
    rel = 2 * max(lens) * 2.0**-24
    for h in (0, 1, heads // 2, heads - 1):
        one = ia.PagedKV(c.k[:, h:h + 1], c.v[:, h:h + 1], c.table, c.lens)
        w1 = torch.full(one.meta_shape, -5.0, device="cuda")
        o1 = ia.attn_decode_paged(q[:, h * group:(h + 1) * group], one, weights_out=w1)
        assert ((w[:, h] - w1[:, 0]).abs() <= (rel + group * 2.0**-23) * w1[:, 0].abs()).all()
        o = out[:, h * group:(h + 1) * group].float()
        # the outputs: the same, of sums of |p v|, and bf16's own rounding on both sides
        top = c.v[:, h].float().nan_to_num(0.0).abs().max()
        err = 2 * rel * top + (2.0**-7 * o1.float().abs() if dtype == BF16 else 0.0)
        assert ((o - o1.float()).abs() <= err).all()
    for r, n in enumerate(lens):
        assert (w[r, :, n:] == -5.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout", ["slots", "joint"])
def test_decode_layouts(ia, layout, dtype):
    """Pools of other orders, queries out of a packed projection, a strided output, a wide table."""
    print(f"[case] paged decode layout {layout} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(3)
    heads, group, D, lens = 2, 2, 64, [70, 9, 33]
    c, ks, vs, _ = make_cache(ia, gen, lens, heads, D, 16, dtype, 6, layout=layout)
    wide = torch.full((3, 11), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:8] = c.table
    c.table = wide[:, 2:8]
    packed = rnd(gen, (3, 1, 3, heads * group, D), dtype).cuda()
    q = packed[:, :, 1].transpose(1, 2)  # [rows, q_heads, 1, D]
    out = torch.full((heads * group, 3, 1, D + 32), 9.0, dtype=dtype, device="cuda").transpose(0, 1)[..., :D]
    ia.attn_decode_paged(q, c, out=out)
    check_decode(q.cpu(), out, ks, vs, heads, ia.default_scale(D), dtype)
    ref = ia.attn_decode_paged(q.contiguous(), c, max_len=96)
    assert torch.equal(ref, out.contiguous())
    assert (torch.as_strided(out, (4, 3, 32), (3 * (D + 32), D + 32, 1), D) == 9.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decode_bad_rows_are_nan(ia, dtype):
    """Pages outside the pool and lengths past max_len make their row NaN and no other."""
    print(f"[case] paged decode bad rows {dtype}", flush=True)
    gen = torch.Generator().manual_seed(4)
    heads, group, D, page = 2, 2, 64, 16
    lens = [200, 40, 200, 150, 16]
    for weigh in (False, True):
        c, ks, vs, _ = make_cache(ia, gen, lens, heads, D, page, dtype, 20)
        q = rnd(gen, (5, heads * group, 1, D), dtype)
        t = c.table.clone()
        t[0, 12] = c.k.shape[0]           # the last page of row 0
        t[2, 3] = -1
        c.table = t
        c.lens = torch.tensor([200, 40, 200, 290, -3], dtype=torch.int32, device="cuda")
        w = torch.zeros(5, heads, c.capacity, device="cuda") if weigh else None
        out = ia.attn_decode_paged(q.cuda(), c, max_len=256, weights_out=w)
        assert out[0].isnan().all() and out[2].isnan().all() and out[3].isnan().all()
        assert (out[4] == 0).all()
        check_decode(q, out, ks, vs, heads, ia.default_scale(D), dtype, skip=(0, 2, 3, 4))
        if weigh:
            assert w[0, :, :200].isnan().all() and w[1].isfinite().all() and (w[4] == 0).all()
    c.lens = torch.tensor([16, 17, 15, 0, 300], dtype=torch.int32, device="cuda")
    out = ia.attn_decode_paged(q.cuda(), c, max_len=16)  # one split
    assert out[1].isnan().all() and out[4].isnan().all() and (out[3] == 0).all()
    assert out[0].isfinite().all() and out[2].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decode_infinite_scores(ia, dtype):
    """A key at -inf has probability 0; a row of such keys, of a key at +inf or of a NaN one is NaN."""
    print(f"[case] paged decode infinities {dtype}", flush=True)
    gen = torch.Generator().manual_seed(5)
    D, page, lens = 64, 16, [100, 60, 40, 40]
    c, ks, vs, _ = make_cache(ia, gen, lens, 1, D, page, dtype)
    q = rnd(gen, (4, 2, 1, D), dtype).abs_() + 0.1

    def set_key(r, j, value):
        c.k[int(c.table[r, j // page]), 0, j % page, 3] = value
        ks[r][0, j, 3] = value

    for j in (0, 17, 99):
        set_key(0, j, -math.inf)
    for j in range(60):
        set_key(1, j, -math.inf)
    set_key(2, 5, math.inf)
    set_key(3, 39, math.nan)
    w = torch.full((4, 1, c.capacity), 3.0, device="cuda")
    for args in (dict(), dict(weights_out=w)):
        out = ia.attn_decode_paged(q.cuda(), c, **args)
        check_decode(q, out, ks, vs, 1, ia.default_scale(D), dtype, skip=(1, 2, 3))
        assert out[1].isnan().all() and out[2].isnan().all() and out[3].isnan().all()
    assert (w[0, 0, [0, 17, 99]] == 0).all() and (w[0, 0, :100].sum() - 2).abs() < 1e-4


def test_decode_far_offsets(ia):
    """Elements past 2^31 in one pool (bf16, 5 GB), and the same bits on every run."""
    print("[case] paged decode far offsets", flush=True)
    heads, D, page = 2, 128, 64
    pages = (5 << 29) // (heads * D * page)
    pool = torch.empty(pages, heads, page, D, dtype=BF16, device="cuda")
    gen = torch.Generator().manual_seed(6)
    lens, per = [300, 520], 9
    far = torch.tensor([[pages - 1 - i for i in range(per)], [pages // 2 - 4 + i for i in range(per)]])
    ks = []
    for r, n in enumerate(lens):
        x = rnd(gen, (heads, per * page, D), BF16)
        pool[far[r].cuda()] = x.view(heads, per, page, D).transpose(0, 1).cuda()
        ks.append(x[:, :n].double())
    c = ia.PagedKV(pool, pool, far.to(torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    q = rnd(gen, (2, 4, 1, D), BF16)
    out = ia.attn_decode_paged(q.cuda(), c)
    check_decode(q, out, ks, ks, heads, ia.default_scale(D), BF16)
    for _ in range(3):
        assert torch.equal(out, ia.attn_decode_paged(q.cuda(), c))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_writes_far_offsets(ia, dtype):
    """Append, eviction and reordering on pages past 2^31 elements (2 x 5 GB in bf16, 10 in fp32)."""
    print(f"[case] paged writes far offsets {dtype}", flush=True)
    heads, D, page = 2, 64, 16
    pages = (5 << 29) // (heads * D * page)
    k = torch.empty(pages, heads, page, D, dtype=dtype, device="cuda")
    v = torch.empty_like(k)
    gen = torch.Generator().manual_seed(16)
    table = torch.tensor([[pages - 1, pages - 7, pages - 3], [pages - 2, pages - 5, pages - 4]], dtype=torch.int32)
    c = ia.PagedKV(k, v, table.cuda(), torch.full((2,), 40, dtype=torch.int32, device="cuda"))
    kn, vn = (rnd(gen, (2, heads, 40, D), dtype) for _ in range(2))
    ia.kv_append(c, kn.cuda(), vn.cuda())

    def row(pool, pages_of_row, n):
        return pool[pages_of_row.long().cuda()].transpose(0, 1).reshape(heads, -1, D)[:, :n].cpu()

    for r in range(2):
        assert torch.equal(row(k, table[r], 40), kn[r]) and torch.equal(row(v, table[r], 40), vn[r])
    spare = torch.tensor([pages - 9, pages - 8], dtype=torch.int32)
    new, _ = ia.beam_reorder(c, torch.tensor([[1, 0]], dtype=torch.int32).cuda(), spare.cuda())
    assert new.tolist() == [[pages - 2, pages - 5, pages - 9], [pages - 1, pages - 7, pages - 8]]
    for r in range(2):
        assert torch.equal(row(k, new[r].cpu(), 40), kn[1 - r]) and torch.equal(row(v, new[r].cpu(), 40), vn[1 - r])
    w = torch.rand(2, heads, 48, generator=gen)
    pos = torch.arange(48, dtype=torch.int32).expand(2, heads, 48).contiguous()
    ia.kv_evict(c, w.cuda(), pos.cuda(), 25, 3, max_len=40)
    for r in range(2):
        for h in range(heads):
            holes, src = ref_evict(w[r, h].numpy(), pos[r, h].numpy(), 40, 25, 3)
            kr, vr = kn[r, h].clone(), vn[r, h].clone()
            kr[holes], vr[holes] = kn[r, h][src], vn[r, h][src]
            assert torch.equal(row(k, table[r], 25)[h], kr[:25]) and torch.equal(row(v, table[r], 25)[h], vr[:25])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decode_long(ia, dtype):
    """A long row on many splits beside a short one; weights over all of it."""
    print(f"[case] paged decode long {dtype}", flush=True)
    gen = torch.Generator().manual_seed(7)
    heads, group, D, lens = 1, 4, 64, [70001, 5]
    c, ks, vs, _ = make_cache(ia, gen, lens, heads, D, 32, dtype)
    q = rnd(gen, (2, heads * group, 1, D), dtype, 2.0)
    w = torch.zeros(2, heads, c.capacity, device="cuda")
    out = ia.attn_decode_paged(q.cuda(), c, weights=w, weights_out=w)
    ps = check_decode(q, out, ks, vs, heads, ia.default_scale(D), dtype)
    for r, n in enumerate(lens):
        want, rel = ps[r][0].sum(0), ps[r][1]
        assert ((w[r, 0, :n].double().cpu() - want).abs() <= (rel.max() + 5 * 2.0**-24) * want + 1e-30).all()
        assert (w[r, 0, n:] == 0).all()


# ---- append ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("heads,D,page,T,layout,offset", [
    (3, 64, 16, 1, "heads", 0), (2, 32, 1, 7, "heads", 0), (2, 128, 4, 21, "slots", 0), (1, 64, 64, 40, "joint", 0),
    (5, 32, 8, 3, "heads", 4),  # bf16 rows aligned to 8 bytes only
])
def test_append(ia, heads, D, page, T, layout, offset, dtype):
    print(f"[case] append {heads} D{D} page {page} T{T} {layout} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(T)
    rows, max_pages = 6, -(-60 // page)
    cap = max_pages * page
    before = [0, 5, 17, 3, cap - 1, 2]
    counts = [T, max(T - 1, 0), 0, T, T, min(T, 2)]
    lens = [b + n for b, n in zip(before, counts)]  # row 4 runs past the capacity where T > 1
    c, _, _, _ = make_cache(ia, gen, [min(n, cap) for n in lens], heads, D, page, dtype, max_pages, layout=layout)
    c.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    t = c.table.clone()
    if lens[3] > 4:
        t[3, 3 // page] = -1  # the page of the first new token of row 3 is not in the pool
    c.table = t
    flat = rnd(gen, (offset + rows * T * 3 * heads * D,), dtype).cuda()[offset:]
    qkv = flat.view(rows, T, 3, heads, D)
    kn, vn = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    k0, v0 = c.k.cpu().clone(), c.v.cpu().clone()
    w = torch.full((rows, heads, cap), 0.5, device="cuda")
    pos = torch.full((rows, heads, cap), -9, dtype=torch.int32, device="cuda")
    seen = (c.lens + 1000).to(torch.int32)
    ia.kv_append(c, kn, vn, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"), weights=w, positions=pos,
                 seen=seen)
    wr, pr = torch.full_like(w.cpu(), 0.5), torch.full_like(pos.cpu(), -9)
    table = c.table.cpu()
    for r in range(rows):
        for i in range(counts[r]):
            a = lens[r] - counts[r] + i
            if a >= cap or not 0 <= int(table[r, a // page]) < c.k.shape[0]:
                continue
            p = int(table[r, a // page])
            k0[p, :, a % page], v0[p, :, a % page] = kn[r, :, i].cpu(), vn[r, :, i].cpu()
            wr[r, :, a], pr[r, :, a] = 0.0, lens[r] + 1000 - counts[r] + i
    assert torch.equal(c.k.cpu().nan_to_num(7.5), k0.nan_to_num(7.5))
    assert torch.equal(c.v.cpu().nan_to_num(7.5), v0.nan_to_num(7.5))
    assert torch.equal(w.cpu(), wr) and torch.equal(pos.cpu(), pr)


def test_append_without_counts(ia):
    print("[case] append without counts", flush=True)
    gen = torch.Generator().manual_seed(9)
    c, _, _, _ = make_cache(ia, gen, [10, 32, 4], 2, 64, 16, F32, 2)
    kn, vn = rnd(gen, (3, 2, 4, 64)).cuda(), rnd(gen, (3, 2, 4, 64)).cuda()
    pos = c.meta(torch.int32)
    ia.kv_append(c, kn, vn, positions=pos)
    for r, n in enumerate([10, 32, 4]):
        for i in range(4):
            a = n - 4 + i
            p = int(c.table[r, a // 16])
            assert torch.equal(c.k[p, :, a % 16], kn[r, :, i]) and torch.equal(c.v[p, :, a % 16], vn[r, :, i])
            assert (pos[r, :, a] == a).all()
    ia.kv_append(c, kn[:, :, :0], vn[:, :, :0])  # nothing to write


# ---- eviction ---------------------------------------------------------------------------------------


def ref_evict(w, pos, n, keep, recent):
    """(holes, sources) of one (row, head), both ascending."""
    w, pos = w[:n].astype(np.float64), pos[:n].astype(np.int64)
    if n <= keep:
        return [], []
    safe = pos >= pos.max() + 1 - recent
    rank = [(0 if safe[j] else 1, 1 if not safe[j] and np.isnan(w[j]) else 0,
             0.0 if safe[j] or np.isnan(w[j]) else -w[j], j) for j in range(n)]
    kept = {r[3] for r in sorted(rank)[:keep]}
    return [j for j in range(keep) if j not in kept], [j for j in range(keep, n) if j in kept]


def weights_of(kind, gen, shape):
    if kind == "ties":
        return torch.randint(0, 3, shape, generator=gen).float()
    if kind == "equal":
        return torch.full(shape, 0.25)
    w = torch.randn(shape, generator=gen).mul_(2.0).exp_()
    if kind == "odd":  # signs, both zeros, infinities, NaN, subnormal numbers
        pick = torch.randint(0, 10, shape, generator=gen)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1e-42)):
            w[pick == i] = x
        w[pick == 7] *= -1
    return w


EVICT = [
    # lengths, max_len, keep, recent, page
    ([100, 41, 40, 39, 0, 1], 112, 40, 10, 16),
    ([100, 64, 99], 112, 99, 99, 16),     # one of each at most
    ([100, 3, 2], 112, 1, 0, 4),
    ([100, 3, 2], 100, 1, 1, 4),
    ([1500, 1025, 1024], 2000, 1024, 0, 32),
    ([1500, 700, 2000], 1600, 200, 64, 1),  # 2000 > max_len: left alone
    ([5000], 5000, 4936, 512, 64),
    ([36864, 100], 36864, 20000, 1000, 64),  # the longest whose keys are held on the chip
    ([36865, 36000], 36865, 36000, 1000, 64),
    ([70000, 20], 70000, 30000, 100, 128),
]


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,max_len,keep,recent,page", EVICT)
def test_evict(ia, lens, max_len, keep, recent, page, kind):
    print(f"[case] evict {lens} keep {keep} recent {recent} {kind}", flush=True)
    gen = torch.Generator().manual_seed(keep)
    rows, heads, D = len(lens), 2, 32
    dtype = BF16 if keep % 2 else F32
    c, ks, vs, _ = make_cache(ia, gen, lens, heads, D, page, dtype, -(-max(max(lens), max_len) // page))
    w = weights_of(kind, gen, (rows, heads, c.capacity))
    pos = (torch.rand(w.shape, generator=gen) * 20 + torch.arange(c.capacity)).argsort(2).argsort(2).to(torch.int32) * 3
    k0, v0, w0, p0 = c.k.cpu().clone(), c.v.cpu().clone(), w.clone(), pos.clone()
    wr, pr = torch.full_like(w, -3.0), torch.full_like(pos, -4)
    table = c.table.cpu()
    for r, n in enumerate(lens):
        for h in range(heads):
            m = min(n, keep) if n <= max_len else n
            wr[r, h, :m], pr[r, h, :m] = w[r, h, :m], pos[r, h, :m]
            holes, src = ref_evict(w[r, h].numpy(), pos[r, h].numpy(), n, keep, recent) if n <= max_len else ([], [])
            assert len(holes) == len(src)
            for a, b in zip(holes, src):
                pa, pb = int(table[r, a // page]), int(table[r, b // page])
                k0[pa, h, a % page], v0[pa, h, a % page] = k0[pb, h, b % page], v0[pb, h, b % page]
                wr[r, h, a], pr[r, h, a] = w[r, h, b], pos[r, h, b]
    w_out, p_out = torch.full_like(w, -3.0).cuda(), torch.full_like(pos, -4).cuda()
    wd, pd = w.cuda(), pos.cuda()
    new = ia.kv_evict(c, wd, pd, keep, recent, weights_out=w_out, positions_out=p_out, max_len=max_len)
    want = [n if n > max_len else min(n, keep) for n in lens]
    assert new.tolist() == want
    same = lambda a, b: torch.equal(a.cpu().nan_to_num(1e9), b.nan_to_num(1e9))  # noqa: E731
    assert same(c.k, k0) and same(c.v, v0)
    assert same(w_out, wr) and torch.equal(p_out.cpu(), pr)
    assert same(wd, w0) and torch.equal(pd.cpu(), p0)
    # all in place: nothing that is kept differs, the slots past the cut stay
    lens_in = c.lens
    got = ia.kv_evict(c, wd, pd, keep, recent, lens_out=lens_in, max_len=max_len)
    assert got is lens_in and lens_in.tolist() == want
    for r, n in enumerate(lens):
        m = want[r]
        assert same(wd[r, :, :m], wr[r, :, :m]) and torch.equal(pd[r, :, :m].cpu(), pr[r, :, :m])
        assert same(wd[r, :, m:], w0[r, :, m:]) and torch.equal(pd[r, :, m:].cpu(), p0[r, :, m:])
    assert same(c.k, k0) and same(c.v, v0)


def test_evict_extreme_positions(ia):
    """Positions at both ends of their type, and a cache whose pages are partly outside the pool."""
    print("[case] evict extreme positions", flush=True)
    gen = torch.Generator().manual_seed(11)
    c, _, _, _ = make_cache(ia, gen, [64, 64], 1, 32, 16, F32)
    t = c.table.clone()
    t[1, 0] = 1 << 20
    c.table = t
    w = torch.rand(2, 1, 64, generator=gen)
    pos = torch.randperm(64, generator=gen).to(torch.int32).expand(2, 1, 64).contiguous()
    pos[pos == 63] = 2**31 - 1
    pos[pos == 0] = -2**31
    k0 = c.k.cpu().clone()
    wd, pd = w.cuda(), pos.cuda()
    new = ia.kv_evict(c, wd, pd, 20, 20)
    assert new.tolist() == [20, 20]
    for r in range(2):
        holes, src = ref_evict(w[r, 0].numpy(), pos[r, 0].numpy(), 64, 20, 20)
        want = w[r, 0, :20].clone()
        want[holes] = w[r, 0, src]
        assert torch.equal(wd[r, 0, :20].cpu(), want)
    bad = (k0.nan_to_num(1e9) != c.k.cpu().nan_to_num(1e9)).any(dim=3).any(dim=1).any(dim=1).nonzero().flatten()
    mine = {int(x) for x in c.table[0, :2]} | {int(x) for x in c.table[1, 1:2]}
    assert set(bad.tolist()) <= mine


# ---- beam selection -----------------------------------------------------------------------------------


def ref_select(logits, scores, finished, eos):
    """The best candidates of each group, by (score, beam, token) in 64 bits."""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    x = logits.double().numpy().reshape(groups, beams, vocab)
    out = []
    for g in range(groups):
        found = []
        for b in range(beams):
            s = float(scores[g, b])
            if finished is not None and finished[g, b]:
                found.append((s, b, eos))
                continue
            row = x[g, b]
            fine = math.isfinite(s) and not np.isnan(row).any() and row.max() < math.inf and row.max() > -math.inf
            if not fine:
                found += [(math.nan if math.isfinite(s) else s, b, t) for t in range(min(beams, vocab))]
                continue
            lse = row.max() + math.log(np.exp(row - row.max()).sum())
            found += [(s + (row[t] - lse), b, int(t)) for t in np.argsort(-row, kind="stable")[:beams]]
        found.sort(key=lambda f: (math.isnan(f[0]), -f[0] if not math.isnan(f[0]) else 0.0, f[1], f[2]))
        out.append(found[:beams])
    return out


def check_select(ia, logits, scores, finished=None, eos=None, dev_logits=None):
    got = ia.beam_select(logits.cuda() if dev_logits is None else dev_logits, scores.cuda(),
                         None if finished is None else finished.cuda(), eos)
    tokens, parents, out, done = (None if t is None else t.cpu() for t in got)
    ref = ref_select(logits, scores, finished, eos)
    for g, found in enumerate(ref):
        for i, (s, b, t) in enumerate(found):
            assert (int(parents[g, i]), int(tokens[g, i])) == (b, t), (g, i, found, parents[g], tokens[g])
            v = float(out[g, i])
            if math.isnan(s) or math.isinf(s):
                assert math.isnan(v) if math.isnan(s) else v == s
            else:
                # the result's rounding, and the exponentials' (2^-23 each) in the lse
                assert abs(v - s) <= 2.0**-24 * abs(s) + 2.0**-21
            if done is not None:
                assert int(done[g, i]) == int(bool(finished is not None and finished[g, b]) or t == eos)
    return got


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab", [
    (1, 1, 1), (1, 1, 2), (2, 4, 1), (1, 3, 3), (3, 4, 5), (2, 32, 33), (1, 32, 31), (5, 2, 255), (2, 5, 256),
    (1, 4, 8192), (2, 8, 8193), (3, 7, 20011), (1, 32, 50257), (40, 3, 1000),
])
def test_select(ia, groups, beams, vocab, dtype):
    print(f"[case] select {groups}x{beams} V{vocab} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab + beams)
    logits = rnd(gen, (groups * beams, vocab), dtype, 2.0)
    scores = rnd(gen, (groups, beams)) - 10.0
    check_select(ia, logits, scores)
    eos = min(2, vocab - 1)
    finished = (torch.rand(groups, beams, generator=gen) < 0.4).to(torch.int32) * 5
    check_select(ia, logits, scores, finished, eos)
    check_select(ia, logits, scores, None, eos)
    first = torch.full((groups, beams), -math.inf)
    first[:, 0] = 0.0
    check_select(ia, logits, first)
    check_select(ia, logits, scores, torch.ones(groups, beams, dtype=torch.int32), eos)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab,pad,shift", [(1001, 0, 0), (1001, 7, 1), (5003, 2, 3), (9000, 0, 5), (64, 3, 7)])
def test_select_alignment(ia, vocab, pad, shift, dtype):
    """Rows at any alignment; what lies around them is not read into the result."""
    print(f"[case] select alignment V{vocab} pad {pad} shift {shift} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    groups, beams = 2, 6
    wide = torch.full((groups * beams * (vocab + pad) + shift + 16,), math.inf, dtype=dtype, device="cuda")
    view = torch.as_strided(wide, (groups * beams, vocab), (vocab + pad, 1), shift)
    logits = rnd(gen, (groups * beams, vocab), dtype, 3.0)
    view.copy_(logits)
    check_select(ia, logits, rnd(gen, (groups, beams)), dev_logits=view)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_select_ties_and_odd_values(ia, dtype):
    print(f"[case] select ties {dtype}", flush=True)
    gen = torch.Generator().manual_seed(1)
    beams, vocab = 8, 20000
    same = torch.zeros(2 * beams, vocab, dtype=dtype)             # every candidate equal: lowest first
    check_select(ia, same, torch.zeros(2, beams))
    check_select(ia, same - 3.5, torch.arange(2.0 * beams).view(2, beams))
    few = torch.randint(0, 2, (2 * beams, vocab), generator=gen).to(dtype)
    check_select(ia, few, torch.zeros(2, beams))
    twins = rnd(gen, (1, vocab), dtype).expand(2 * beams, vocab).contiguous()
    check_select(ia, twins, torch.zeros(2, beams))                # equal beams: the lower one first
    masked = rnd(gen, (2 * beams, vocab), dtype)
    masked[:, 5:] = -math.inf                                     # five tokens allowed
    check_select(ia, masked, torch.randn(2, beams, generator=gen))
    one = masked.clone()
    one[:, 1:] = -math.inf                                        # one: the others follow at -inf
    check_select(ia, one, torch.zeros(2, beams))
    low = torch.full((2 * beams, vocab), torch.finfo(dtype).min, dtype=dtype)  # masks of the lowest value
    low[:, 77] = 1.0
    check_select(ia, low, torch.zeros(2, beams))
    odd = rnd(gen, (2 * beams, vocab), dtype)
    odd[0, 3], odd[1, 19999], odd[2], odd[3, 0] = math.nan, math.inf, -math.inf, -math.inf
    odd[8:] = math.nan                                            # a group without a finite beam
    check_select(ia, odd, torch.zeros(2, beams))
    scores = torch.zeros(2, beams)
    scores[0, :4] = torch.tensor([math.nan, math.inf, -math.inf, -1e30])
    check_select(ia, rnd(gen, (2 * beams, vocab), dtype), scores)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("beams,vocab,allowed", [
    (32, 9001, (8999,)), (32, 9001, range(0, 40)), (32, 9001, (0, 64, 65, 200, 8191, 8192, 9000)), (5, 300, range(3, 300, 7)),
    (8, 20000, range(8192, 8200)), (16, 4099, (1, 2, 3, 4096, 4098)), (32, 40000, range(100, 131)),
])
def test_select_allowed_tokens(ia, beams, vocab, allowed, dtype):
    """All tokens but a few at -inf, wherever they lie: with fewer candidates than beams the lowest tokens follow."""
    print(f"[case] select allowed {beams} V{vocab} {len(allowed)} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.full((2 * beams, vocab), -math.inf, dtype=dtype)
    logits[:, list(allowed)] = rnd(gen, (2 * beams, len(allowed)), dtype, 2.0)
    check_select(ia, logits, rnd(gen, (2, beams)))
    first = torch.full((2, beams), -math.inf)
    first[:, 0] = 0.0
    check_select(ia, logits, first)


def test_select_in_place(ia):
    """The results may be the inputs, and a workspace may hold anything."""
    print("[case] select in place", flush=True)
    gen = torch.Generator().manual_seed(2)
    groups, beams, vocab, eos = 3, 6, 3001, 4
    logits, scores = rnd(gen, (groups * beams, vocab)).cuda(), rnd(gen, (groups, beams)).cuda()
    fin = (torch.rand(groups, beams, generator=gen) < 0.3).to(torch.int32).cuda()
    want = ia.beam_select(logits, scores, fin, eos)
    ws = ia.beam_select_workspace(groups, beams, vocab)
    ws.fill_(255)
    tok, par = torch.empty_like(fin), torch.empty_like(fin)
    st = ia.lib().inf_beam_select(logits.data_ptr(), vocab, scores.data_ptr(), fin.data_ptr(), groups, beams, vocab, eos,
                                  tok.data_ptr(), par.data_ptr(), scores.data_ptr(), fin.data_ptr(), ia.INF_F32,
                                  ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert st == 0
    for a, b in zip((tok, par, scores, fin), want):
        assert torch.equal(a, b)


# ---- reordering ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,layers,heads,D,page,length,layout", [
    (1, 4, 1, 2, 64, 16, 41, "heads"), (3, 3, 2, 3, 32, 8, 16, "heads"), (2, 5, 3, 1, 128, 32, 31, "slots"),
    (2, 2, 2, 2, 64, 1, 5, "heads"), (2, 4, 1, 2, 64, 16, 0, "heads"), (1, 8, 2, 12, 64, 128, 511, "joint"),
    (4, 1, 1, 2, 32, 16, 20, "heads"),
])
def test_reorder(ia, groups, beams, layers, heads, D, page, length, layout, dtype):
    print(f"[case] reorder {groups}x{beams} L{layers} page {page} len {length} {layout} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(length)
    rows = groups * beams
    c, _, _, spare = make_cache(ia, gen, [length] * rows, heads, D, page, dtype, length // page + 2, spare=rows,
                                layers=layers, layout=layout)
    spare = spare[:rows].cuda()
    parents = torch.randint(0, beams, (groups, beams), generator=gen, dtype=torch.int32)
    k0, v0, table0 = c.k.cpu().clone(), c.v.cpu().clone(), c.table.cpu().clone()
    table, new_spare = ia.beam_reorder(c, parents.cuda(), spare)
    full, part = length // page, length % page
    tr, sr, kr, vr = table0.clone(), spare.cpu().clone(), k0.clone(), v0.clone()
    for row in range(rows):
        p = row // beams * beams + int(parents.view(-1)[row])
        tr[row, :full] = table0[p, :full]
        if part and p != row:
            a, b = int(table0[p, full]), int(spare[row])
            kr[:, b, :, :part], vr[:, b, :, :part] = k0[:, a, :, :part], v0[:, a, :, :part]
            tr[row, full], sr[row] = b, table0[row, full]
    assert torch.equal(table.cpu(), tr) and torch.equal(new_spare.cpu(), sr)
    assert torch.equal(c.k.cpu().nan_to_num(7.5), kr.nan_to_num(7.5))
    assert torch.equal(c.v.cpu().nan_to_num(7.5), vr.nan_to_num(7.5))
    assert torch.equal(c.table.cpu(), table0)
    # the tails are apart, and the spare pages too
    if part:
        tails = table[:, full].tolist() + new_spare.tolist()
        assert len(set(tails)) == 2 * rows
    # the other rows' and layers' copies read the tables and spare pages: not in place
    with pytest.raises(ia.InfernoError):
        ia.beam_reorder(c, parents.cuda(), spare, spare_out=spare)
    with pytest.raises(ia.InfernoError):
        ia.beam_reorder(c, parents.cuda(), spare, table_out=c.table)


def test_reorder_bad_parent(ia):
    """A parent outside the group gives a row without pages, which reads as NaN; pages outside the pool
    are not copied."""
    print("[case] reorder bad parent", flush=True)
    gen = torch.Generator().manual_seed(8)
    c, _, _, spare = make_cache(ia, gen, [21] * 4, 1, 32, 16, F32, spare=4)
    t = c.table.clone()
    t[3, 1] = -1
    c.table = t
    sp = spare[:4].clone()
    sp[1] = 10**6
    k0 = c.k.cpu().clone()
    parents = torch.tensor([[2, 0], [0, 1]], dtype=torch.int32)
    table, _ = ia.beam_reorder(c, parents.cuda(), sp.cuda())
    assert (table[0] == -1).all() and table[1].tolist() == [int(c.table[0, 0]), 10**6]
    assert torch.equal(c.k.cpu().nan_to_num(5.5), k0.nan_to_num(5.5))
    c.table = table
    out = ia.attn_decode_paged(torch.ones(4, 1, 1, 32, device="cuda"), c)
    assert out[0].isnan().all() and out[1].isnan().all() and out[2].isfinite().all() and out[3].isnan().all()


def test_reorder_from_a_bad_page(ia):
    """A parent whose last page is not in the pool passes its number on: the row reads as NaN too, not as
    what its spare page held."""
    print("[case] reorder from a bad page", flush=True)
    gen = torch.Generator().manual_seed(9)
    c, _, _, spare = make_cache(ia, gen, [21] * 4, 1, 32, 16, F32, spare=4)
    t = c.table.clone()
    t[1, 1], t[3, 1] = -1, 10**6
    c.table = t
    c.k.nan_to_num_(0.5)
    c.v.nan_to_num_(0.5)
    sp = spare[:4].cuda()
    table, spare_out = ia.beam_reorder(c, torch.tensor([[1, 0], [0, 0]], dtype=torch.int32, device="cuda"), sp)
    assert table[0].tolist() == [int(t[1, 0]), -1] and int(spare_out[0]) == int(sp[0])
    assert table[1].tolist() == [int(t[0, 0]), int(sp[1])]
    assert table[3].tolist() == [int(t[2, 0]), int(sp[3])]
    c.table = table
    out = ia.attn_decode_paged(torch.ones(4, 1, 1, 32, device="cuda"), c)
    assert out[0].isnan().all() and out[1:].isfinite().all()


# ---- together -----------------------------------------------------------------------------------------


class Toy:
    """Two layers of attention with shared key-value heads and tied logits; fp32 weights."""

    def __init__(self, heads=2, group=2, D=32, vocab=61, layers=2, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.heads, self.group, self.D, self.vocab, self.layers = heads, group, D, vocab, layers
        C = heads * group * D
        self.emb = torch.randn(vocab, C, generator=gen)
        self.wq = [torch.randn(C, C, generator=gen) / C**0.5 for _ in range(layers)]
        self.wkv = [torch.randn(C, 2 * heads * D, generator=gen) / C**0.5 for _ in range(layers)]
        self.wo = [torch.randn(C, C, generator=gen) / C**0.5 for _ in range(layers)]

    def to(self, f):
        t = Toy.__new__(Toy)
        t.__dict__.update(self.__dict__)
        t.emb, t.wq, t.wkv, t.wo = f(self.emb), *([f(w) for w in ws] for ws in (self.wq, self.wkv, self.wo))
        return t

    def heads_of(self, x, n):  # [B, T, n D] -> [B, n, T, D]
        return x.view(x.shape[0], x.shape[1], n, self.D).transpose(1, 2)

    def full(self, tokens):
        """Logits of the last position of [B, T] tokens, everything anew."""
        x = self.emb[tokens]
        T = tokens.shape[1]
        hide = torch.ones(T, T, dtype=torch.bool, device=x.device).triu(1)
        for wq, wkv, wo in zip(self.wq, self.wkv, self.wo):
            q = self.heads_of(x @ wq, self.heads * self.group)
            kv = self.heads_of(x @ wkv, 2 * self.heads).repeat_interleave(self.group, 1)
            n = self.heads * self.group
            s = (q @ kv[:, :n].transpose(2, 3)) / self.D**0.5
            o = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ kv[:, n:]
            x = x + o.transpose(1, 2).reshape(x.shape) @ wo
        return x[:, -1] @ self.emb.t()


def test_beam_search(ia):
    """Prompts of different lengths, beam search with pages and reordering: every step's beams against the
    search over whole sequences in 64 bits."""
    print("[case] beam search", flush=True)
    toy = Toy()
    ref, dev = toy.to(lambda w: w.double()), toy.to(lambda w: w.cuda())
    groups, beams, page, steps, eos = 3, 4, 8, 21, 5
    rows, prompt = groups * beams, [13, 8, 3]
    T = max(prompt)
    gen = torch.Generator().manual_seed(3)
    prompts = torch.randint(6, toy.vocab, (groups, T), generator=gen)
    max_pages = -(-(T + steps) // page) + 1
    pages = rows * (max_pages + 1)
    k = torch.full((toy.layers, pages, toy.heads, page, toy.D), math.nan, device="cuda")
    v = torch.full_like(k, math.nan)
    table = torch.arange(rows * max_pages, dtype=torch.int32, device="cuda").view(rows, max_pages)
    spare = torch.arange(rows * max_pages, pages, dtype=torch.int32, device="cuda")
    for g in range(groups):  # the beams of a prompt share its full pages
        f = (prompt[g] - 1) // page
        table[g * beams:(g + 1) * beams, :f] = table[g * beams, :f]
    lens = torch.tensor(prompt, dtype=torch.int32).repeat_interleave(beams).cuda() - 1
    cache = ia.PagedKV(k, v, table, lens)
    layers = [cache.layer(i) for i in range(toy.layers)]
    # the prompts but for their last token, padded to the longest: every row writes its own pages
    x = dev.emb[prompts[:, :T - 1].cuda()].repeat_interleave(beams, 0)
    hide = torch.ones(T - 1, T - 1, dtype=torch.bool, device="cuda").triu(1)
    for i in range(toy.layers):
        kv = toy.heads_of(x @ dev.wkv[i], 2 * toy.heads)
        ia.kv_append(layers[i], kv[:, :toy.heads], kv[:, toy.heads:], counts=lens.clone())
        q = toy.heads_of(x @ dev.wq[i], toy.heads * toy.group)
        kk, vv = (t.repeat_interleave(toy.group, 1).contiguous() for t in (kv[:, :toy.heads], kv[:, toy.heads:]))
        s = (q @ kk.transpose(2, 3).contiguous()) / toy.D**0.5
        o = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ vv
        x = x + o.transpose(1, 2).reshape(x.shape) @ dev.wo[i]
    tokens = torch.tensor([int(prompts[g, prompt[g] - 1]) for g in range(groups)]).repeat_interleave(beams).cuda()
    scores = torch.full((groups, beams), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    done = torch.zeros(groups, beams, dtype=torch.int32, device="cuda")
    seqs = [[prompts[g, :prompt[g]].tolist() for _ in range(beams)] for g in range(groups)]
    for step in range(steps):
        lens += 1
        x = dev.emb[tokens][:, None]
        for i in range(toy.layers):
            kv = toy.heads_of(x @ dev.wkv[i], 2 * toy.heads)
            ia.kv_append(layers[i], kv[:, :toy.heads], kv[:, toy.heads:])
            o = ia.attn_decode_paged(toy.heads_of(x @ dev.wq[i], toy.heads * toy.group), layers[i])
            x = x + o.reshape(x.shape) @ dev.wo[i]
        logits = x[:, 0] @ dev.emb.t()
        # every row's logits, finished ones' too, against the sequence that it stands for
        want = torch.cat([ref.full(torch.tensor(seqs[g])) for g in range(groups)])
        assert (logits.double().cpu() - want).abs().max() <= 1e-4 * want.abs().max()
        before, was = scores.double().cpu(), done.cpu().clone()
        tok, par, scores, done = ia.beam_select(logits, scores, done, eos)
        for g in range(groups):
            # each pick's score is that of its place in the ranking over everything
            lp = torch.log_softmax(want[g * beams:(g + 1) * beams], 1)
            lp[was[g] != 0] = -math.inf
            lp[was[g] != 0, eos] = 0.0
            all_scores = lp + before[g][:, None]
            best = torch.sort(all_scores.flatten(), descending=True).values[:beams]
            mine = all_scores[par[g].long().cpu(), tok[g].long().cpu()]
            # a score is off by twice the logits' error at most, the best ones' order by as much again: 4e-4 of the
            # largest logit, which is over 5
            assert (mine - best).abs().max() <= 2e-3 and (scores[g].double().cpu() - mine).abs().max() <= 2e-3
            seqs[g] = [seqs[g][int(p)] + [int(t)] for p, t in zip(par[g], tok[g])]
            assert len({tuple(s) for s in seqs[g]}) == beams or bool(done[g].any())
        table, spare = ia.beam_reorder(cache, par, spare)
        cache.table = table
        for c in layers:
            c.table = table
        tokens = tok.flatten().long()
    assert (lens.cpu() == torch.tensor(prompt).repeat_interleave(beams) - 1 + steps).all()


def test_bounded_cache(ia):
    """Generation in a cache cut to 24 positions whenever it holds 32: the attention of every step against
    64 bits over the positions that the same rule leaves."""
    print("[case] bounded cache", flush=True)
    gen = torch.Generator().manual_seed(12)
    rows, heads, group, D, page, cap, keep, recent = 2, 2, 2, 64, 8, 32, 24, 6
    k = torch.full((rows * cap // page + 1, heads, page, D), math.nan, device="cuda")
    v = torch.full_like(k, math.nan)
    table = torch.randperm(rows * cap // page, generator=gen).to(torch.int32).view(rows, -1).cuda()
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    seen = torch.zeros_like(lens)
    c = ia.PagedKV(k, v, table, lens)
    w, pos = c.meta(F32), c.meta(torch.int32)
    held = [[[] for _ in range(heads)] for _ in range(rows)]  # (position, k, v, weight) by slot
    scale = ia.default_scale(D)
    for step in range(70):
        kn, vn = rnd(gen, (rows, heads, 1, D)), rnd(gen, (rows, heads, 1, D))
        q = rnd(gen, (rows, heads * group, 1, D), std=2.0)
        lens += 1
        seen += 1
        ia.kv_append(c, kn.cuda(), vn.cuda(), weights=w, positions=pos, seen=seen)
        out = ia.attn_decode_paged(q.cuda(), c, weights=w, weights_out=w).double().cpu()
        n = int(lens[0])
        wn, pn = w.double().cpu(), pos.cpu()
        for r in range(rows):
            for h in range(heads):
                mine = held[r][h]
                mine.append([step, kn[r, h, 0].double(), vn[r, h, 0].double(), 0.0])
                kk, vv = (torch.stack([m[i] for m in mine]) for i in (1, 2))
                qq = q[r, h * group:(h + 1) * group, 0].double()
                p = torch.softmax(qq @ kk.t() * scale, 1)
                o = p @ vv
                assert (out[r, h * group:(h + 1) * group, 0] - o).abs().max() <= 1e-4 * o.abs().max()
                assert [m[0] for m in mine] == pn[r, h, :n].tolist()
                for j, m in enumerate(mine):
                    m[3] += float(p[:, j].sum())
                    assert abs(m[3] - float(wn[r, h, j])) <= 1e-4 * (1 + m[3])
        if n == cap:
            raw, rawp = w.cpu().numpy(), pos.cpu().numpy()
            ia.kv_evict(c, w, pos, keep, recent, lens_out=lens)
            for r in range(rows):
                for h in range(heads):
                    holes, src = ref_evict(raw[r, h], rawp[r, h], n, keep, recent)
                    for a, b in zip(holes, src):
                        held[r][h][a] = held[r][h][b]
                    del held[r][h][keep:]
                    for m, j in zip(held[r][h], range(keep)):
                        m[3] = float(w[r, h, j])
            assert lens.tolist() == [keep] * rows


def test_graph_replays_follow_the_lengths(ia):
    """One captured step (append, attention with weights, selection, reordering) replayed while lengths, tables
    and inputs change in place; each replay against the eager calls.  The lengths only grow: a row cut back
    into a full page, which it may share with its parent, would write where another row reads."""
    print("[case] paged graph", flush=True)
    gen = torch.Generator().manual_seed(13)
    groups, beams, heads, group, D, page, max_pages, vocab = 2, 3, 2, 2, 64, 16, 6, 3000
    rows = groups * beams
    pages = rows * (max_pages + 1)
    order = torch.randperm(pages, generator=gen).to(torch.int32)

    def state():
        g2 = torch.Generator().manual_seed(14)
        s = dict(k=rnd(g2, (pages, heads, page, D)).cuda(), v=rnd(g2, (pages, heads, page, D)).cuda(),
                 table=order[:rows * max_pages].view(rows, max_pages).cuda(),
                 spare=order[rows * max_pages:].cuda(), lens=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                 kn=torch.zeros(rows, heads, 1, D, device="cuda"), q=torch.zeros(rows, heads * group, 1, D, device="cuda"),
                 logits=torch.zeros(rows, vocab, device="cuda"), scores=torch.zeros(groups, beams, device="cuda"))
        s["cache"] = ia.PagedKV(s["k"], s["v"], s["table"], s["lens"])
        s["w"] = s["cache"].meta(F32)
        s["out"] = torch.zeros(rows, heads * group, 1, D, device="cuda")
        s["ws"] = ia.attn_decode_paged_workspace(s["cache"], heads * group, weights=True)
        s["ws2"] = ia.beam_select_workspace(groups, beams, vocab)
        s["t2"], s["s2"] = torch.zeros_like(s["table"]), torch.zeros_like(s["spare"])
        return s

    def step(s):
        c = s["cache"]
        ia.kv_append(c, s["kn"], s["kn"], weights=s["w"])
        ia.attn_decode_paged(s["q"], c, weights=s["w"], weights_out=s["w"], out=s["out"], workspace=s["ws"])
        s["sel"] = ia.beam_select(s["logits"], s["scores"], workspace=s["ws2"])
        ia.beam_reorder(c, s["sel"][1], s["spare"], table_out=s["t2"], spare_out=s["s2"])

    gs, es = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(gs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for name in ("k", "v", "w"):
        es[name].copy_(gs[name])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(gs)
    for rep, n in enumerate((1, 17, 40, 90, 96)):
        kn, q, lg = (rnd(gen, es[x].shape).cuda() for x in ("kn", "q", "logits"))
        for s in (gs, es):
            s["kn"].copy_(kn)
            s["q"].copy_(q)
            s["logits"].copy_(lg)
            s["lens"].copy_(torch.tensor([n, n, n, n // 2 + 1, n // 2 + 1, n // 2 + 1], dtype=torch.int32))
        gs["out"].fill_(math.nan)
        step(es)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("k", "v", "w", "out", "t2", "s2"):
            assert torch.equal(gs[name], es[name]), (rep, name)
        for a, b in zip(gs["sel"][:3], es["sel"][:3]):
            assert torch.equal(a, b), rep
        for s in (gs, es):
            s["table"].copy_(s["t2"])
            s["spare"].copy_(s["s2"])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_graph_replays_of_a_bounded_cache(ia, dtype):
    """A captured step that counts, appends, attends and cuts in place, replayed while rows reach the limit at
    different times; every replay against the eager calls, bit for bit."""
    print(f"[case] paged graph of a bounded cache {dtype}", flush=True)
    gen = torch.Generator().manual_seed(21)
    rows, heads, group, D, page, max_pages, keep, recent = 3, 2, 3, 64, 8, 5, 33, 4
    pages = rows * max_pages + 2
    table = torch.randperm(pages, generator=gen)[:rows * max_pages].to(torch.int32).view(rows, max_pages)
    k, v = rnd(gen, (pages, heads, page, D), dtype), rnd(gen, (pages, heads, page, D), dtype)

    def state():
        s = dict(c=ia.PagedKV(k.cuda(), v.cuda(), table.cuda(), torch.tensor([0, 20, 33], dtype=torch.int32).cuda()),
                 kn=torch.zeros(rows, heads, 1, D, dtype=dtype, device="cuda"),
                 q=torch.zeros(rows, heads * group, 1, D, dtype=dtype, device="cuda"),
                 out=torch.zeros(rows, heads * group, 1, D, dtype=dtype, device="cuda"))
        s["w"], s["pos"], s["seen"] = s["c"].meta(F32), s["c"].meta(torch.int32), s["c"].lens.clone()
        s["pos"].copy_(torch.arange(s["c"].capacity, device="cuda"))
        s["ws"] = ia.attn_decode_paged_workspace(s["c"], heads * group, weights=True)
        s["ws2"] = ia.kv_evict_workspace(s["c"], keep)
        return s

    def step(s):
        s["c"].lens.add_(1)
        s["seen"].add_(1)
        ia.kv_append(s["c"], s["kn"], s["kn"], weights=s["w"], positions=s["pos"], seen=s["seen"])
        ia.attn_decode_paged(s["q"], s["c"], weights=s["w"], weights_out=s["w"], out=s["out"], workspace=s["ws"])
        ia.kv_evict(s["c"], s["w"], s["pos"], keep, recent, lens_out=s["c"].lens, workspace=s["ws2"])

    gs, es = state(), state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(gs)
    for rep in range(18):
        kn, q = rnd(gen, gs["kn"].shape, dtype).cuda(), rnd(gen, gs["q"].shape, dtype, 1.5).cuda()
        for s in (gs, es):
            s["kn"].copy_(kn)
            s["q"].copy_(q)
        step(es)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("w", "pos", "out", "seen"):
            assert torch.equal(gs[name], es[name]), (rep, name)
        for name in ("k", "v", "lens"):
            assert torch.equal(getattr(gs["c"], name), getattr(es["c"], name)), (rep, name)
        assert gs["c"].lens.tolist() == [rep + 1, min(21 + rep, keep), keep]


def test_other_stream(ia):
    """Calls with a stream of their own, as an object and as a handle."""
    print("[case] paged other stream", flush=True)
    gen = torch.Generator().manual_seed(15)
    c, ks, vs, _ = make_cache(ia, gen, [500, 100], 2, 64, 16, F32)
    q = rnd(gen, (2, 4, 1, 64)).cuda()
    want = ia.attn_decode_paged(q, c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for st in (s, s.cuda_stream):
        out = ia.attn_decode_paged(q, c, stream=st)
        s.synchronize()
        assert torch.equal(out, want)
