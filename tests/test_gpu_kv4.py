"""A paged key-value cache in 4 bits on the GPU against plain implementations in 64 bits on the CPU: append
and read, attention of one new token, and the steps of a generation that uses them with weights in 8 bits.

What is written and read back has to be equal.  Attention: as over a cache of full precision that holds the values the
codes stand for.  A score's fp32 error: D products (three parts of each in fp32), each sum off by at most 2^-24 of
the products' absolute sum A = sum |q_d k_d| scale, so (3 D + 2) 2^-24 A; scaling and the exponent's argument round it twice
more.  A probability moves by that times itself, twice (its own and the sum's); v_exp_f32 adds 2^-22, sums over n
keys in chains of at most n / 16 + 64 additions 2^-24 each.  Probabilities are held in two bf16 parts for bf16 (2^-16), in
three for fp32 (2^-24); bf16 results round by 2^-8.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


@pytest.fixture(scope="module")
def ia():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_amd

    inferno_amd.lib()
    return inferno_amd


def held(x):
    """The values that x [..., D] is held as, in 64 bits."""
    b = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = torch.frexp(torch.where(bad, torch.ones((), dtype=torch.float64), top)).exponent.double() - 1
    e = torch.where(top == 0, torch.full_like(e, -200.0), e)
    unit = torch.exp2((e - 2).clamp(min=-125))[..., None]
    y = (b.abs() / unit).clamp(max=6.0)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    v = torch.round(y / step) * step * unit * torch.sign(b)
    v[bad] = math.nan
    return v.reshape(x.shape)


def stored(codes, scales):
    """What pools on the CPU stand for: codes [..., slots, D / 2], scales [..., D / 32, slots]."""
    c = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2).long()
    x = torch.cat((GRID, -GRID))[c]
    s = torch.exp2(scales.double() - 127)
    s[scales == 255] = math.nan
    return x * s.transpose(-1, -2).repeat_interleave(32, dim=-1)


def encode(x):
    """Bytes [..., D / 2] and scales [..., D / 32] of values on the grid's lattice."""
    b = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    e = torch.frexp(b.abs().amax(-1)).exponent - 3
    y = b / torch.exp2(e.double())[..., None]
    idx = (y.abs()[..., None] - GRID).abs().argmin(-1)
    c = (idx + 8 * (y < 0)).reshape(x.shape).to(torch.uint8)
    return c[..., ::2] | (c[..., 1::2] << 4), (e + 127).to(torch.uint8)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def make_cache(ia, gen, lens, heads, D, page, max_pages=None, spare=2, layout="heads"):
    """A cache of random rows on the GPU; every unused slot, page and table entry holds what must not count (codes of 6,
    scales of NaN, pages far outside).  Also the rows' keys and values in 64 bits, per row [heads, len, D]."""
    rows = len(lens)
    max_pages = max_pages or max(1, -(-max(lens) // page))
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).tolist()
    table = torch.full((rows, max_pages), -7, dtype=torch.int32)
    pools = [torch.full((pages, heads, page, D // 2), 0x77, dtype=torch.uint8) for _ in range(2)]
    scales = [torch.full((pages, heads, D // 32, page), 255, dtype=torch.uint8) for _ in range(2)]
    values = ([], [])
    for r, n in enumerate(lens):
        mine = [order.pop() for _ in range(need[r])]
        table[r, :need[r]] = torch.tensor(mine, dtype=torch.int32)
        for pool, scale, out in zip(pools, scales, values):
            x = held(torch.randn((heads, n, D), generator=gen) * torch.exp(torch.randn((heads, n, 1), generator=gen)))
            codes, byte = encode(x)
            for i, p in enumerate(mine):
                m = min(page, n - i * page)
                pool[p, :, :m] = codes[:, i * page:i * page + m]
                scale[p, :, :, :m] = byte[:, i * page:i * page + m].transpose(1, 2)
            out.append(x)
    if layout == "slots":  # [pages, slots, heads, bytes] in memory
        pools = [x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in pools]
        scales = [x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in scales]
    elif layout == "joint":  # keys and values of a page side by side
        pools = list(torch.stack(pools, dim=1).cuda().unbind(1))
        scales = list(torch.stack(scales, dim=1).cuda().unbind(1))
    else:
        pools, scales = [x.cuda() for x in pools], [x.cuda() for x in scales]
    lens = torch.tensor(lens, dtype=torch.int32).cuda()
    return ia.PagedKV4(*pools, *scales, table.cuda(), lens), *values, torch.tensor(order, dtype=torch.int32)


# ---- append and read -----------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,heads,page,layout", [(32, 3, 16, "heads"), (64, 2, 32, "slots"), (128, 1, 64, "joint"),
                                                 (128, 5, 16, "slots"), (64, 4, 128, "heads")])
def test_append_and_read(ia, D, heads, page, layout, dtype):
    gen = torch.Generator().manual_seed(D + heads + page)
    before, counts, T = [0, 5, page, 3 * page - 1, 40], [7, 1, 0, page, 20], max(20, page)
    lens = [b + c for b, c in zip(before, counts)]
    cache, ks, vs, _ = make_cache(ia, gen, lens, heads, D, page, layout=layout)
    pools = [t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    qkv = (torch.randn((5, T, 3, heads, D), generator=gen) * 3).to(dtype)
    new = [qkv[:, :, i].transpose(1, 2) for i in (1, 2)]
    dev = qkv.cuda()
    ia.kv4_append(cache, dev[:, :, 1].transpose(1, 2), dev[:, :, 2].transpose(1, 2),
                  counts=torch.tensor(counts, dtype=torch.int32).cuda())
    # every slot of the pools: the new tokens', and the others as they were
    table = cache.table.cpu()
    want = [stored(pools[i], pools[2 + i]) for i in range(2)]
    for r in range(5):
        for i in range(counts[r]):
            at = before[r] + i
            for w, x in zip(want, new):
                w[table[r, at // page], :, at % page] = held(x[r, :, i])
    assert same(stored(cache.k.cpu(), cache.k_scale.cpu()), want[0])
    assert same(stored(cache.v.cpu(), cache.v_scale.cpu()), want[1])
    # and as rows, from the start and from anywhere
    for first in (None, [0, 3, page - 1, -2, 10**6]):
        T2 = max(lens) + 3
        f = None if first is None else torch.tensor(first, dtype=torch.int32).cuda()
        for out in (F32, BF16):
            k, v = ia.kv4_read(cache, T2, first=f, dtype=out)
            for r, n in enumerate(lens):
                f0 = 0 if first is None else first[r]
                for got, w in ((k, want[0]), (v, want[1])):
                    exp = torch.zeros((heads, T2, D), dtype=torch.float64)
                    for t in range(T2):
                        j = f0 + t
                        if 0 <= j < n:
                            exp[:, t] = w[table[r, j // page], :, j % page]
                    assert same(got[r].cpu().double(), exp)


def test_every_middle(ia):
    """Every tie of the grid and its neighbours, at every power of two of either type, and what no block holds."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.cat((mids, torch.nextafter(mids, torch.tensor(9.0)), torch.nextafter(mids, torch.tensor(0.0)),
                      torch.tensor([4.0, 0.0, -0.0, 6.0, 7.9, 0.1, 1.0, 3.0, 0.125, 2.0, 0.5])))
    near = near * torch.where(torch.arange(32) % 3 == 0, -1.0, 1.0)
    scale = torch.exp2(torch.arange(-149, 126).double())
    x = (near.double() * scale[:, None]).float()
    x = x[torch.isfinite(x).all(1)]
    special = torch.stack([near * f for f in (0.0, -0.0, math.inf, math.nan)] + [near.clone() for _ in range(4)])
    for i, v in enumerate((math.inf, -math.inf, math.nan, 3.4e38)):
        special[4 + i, 7 * i] = v
    x = torch.cat((x, special))
    x = torch.cat((x, x[:(-x.shape[0]) % 4])).reshape(-1, 128)
    n = x.shape[0]
    for dtype in (F32, BF16):
        y = x.to(dtype).reshape(1, 1, n, 128)
        table = torch.arange(-(-n // 16), dtype=torch.int32).cuda()[None]
        cache = ia.PagedKV4.empty(table.shape[1], 1, 16, 128, table, torch.tensor([n], dtype=torch.int32).cuda())
        ia.kv4_append(cache, y.cuda(), -y.cuda())
        k, v = ia.kv4_read(cache, n)
        assert same(k.cpu().double(), held(y))
        assert same(v.cpu().double(), -held(y))


def test_append_drops_what_has_no_place(ia):
    """Positions outside the row's pages, pages outside the pool, counts past T."""
    gen = torch.Generator().manual_seed(1)
    cache, _, _, _ = make_cache(ia, gen, [16, 16, 16, 16], 2, 64, 16, max_pages=2, spare=0)
    cache.table[1, 0], cache.table[2, 0] = 4, -1
    cache.lens.copy_(torch.tensor([3, 16, 16, 40], dtype=torch.int32))
    pools = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    k = torch.randn((4, 2, 8, 64), generator=gen)
    ia.kv4_append(cache, k.cuda(), k.cuda(), counts=torch.tensor([8, 8, 99, 8], dtype=torch.int32).cuda())
    now = stored(cache.k.cpu(), cache.k_scale.cpu())
    was = stored(pools[0].cpu(), pools[2].cpu())
    p = int(cache.table[0, 0])
    was[p, :, :3] = held(k[0, :, 5:])  # positions -5 .. 2: the last three
    assert same(now, was)
    assert ia.kv4_read(cache, 4)[0][1:3].isnan().all()
    assert (ia.kv4_read(cache, 4, first=torch.full((4,), 40, dtype=torch.int32).cuda())[1] == 0).all()


def test_read_into_views(ia):
    """Rows of a larger tensor; what lies beside them stays."""
    gen = torch.Generator().manual_seed(2)
    cache, ks, vs, _ = make_cache(ia, gen, [9, 30], 2, 32, 16)
    store = torch.full((2, 40, 3, 2, 32), 5.0, device="cuda")
    k, v = store[:, :30, 1].transpose(1, 2), store[:, :30, 2].transpose(1, 2)
    ia.kv4_read(cache, 30, k_out=k, v_out=v)
    assert torch.equal(k[1].cpu().double(), ks[1]) and torch.equal(v[0, :, :9].cpu().double(), vs[0])
    assert (k[0, :, 9:] == 0).all() and (store[:, :, 0] == 5).all() and (store[:, 30:] == 5).all()


# ---- attention -------------------------------------------------------------------------------------------


def ref_decode(q, ks, vs, heads, scale):
    """(o, bound) in 64 bits."""
    rows, hq, _, D = q.shape
    g = hq // heads
    o, err = torch.zeros(rows, hq, D, dtype=torch.float64), torch.zeros(rows, hq, 1, dtype=torch.float64)
    for r in range(rows):
        n = ks[r].shape[1]
        if not n:
            continue
        kk, vv = ks[r].repeat_interleave(g, 0), vs[r].repeat_interleave(g, 0)
        p = torch.softmax((q[r].double() @ kk.transpose(1, 2))[:, 0] * scale, dim=1)
        o[r] = (p[:, None] @ vv)[:, 0]
        a = ((q[r].double().abs() @ kk.abs().transpose(1, 2))[:, 0] * scale).amax(1)[:, None]
        rel = 2 * ((3 * D + 2) * 2.0**-24 * a + 3 * 2.0**-24 * 1.5 * a) + 2.0**-22 + (n / 16 + 64) * 2.0**-24
        err[r] = rel * (p[:, None] @ vv.abs())[:, 0].amax(1)[:, None]
    return o, err


def check(o, q, ks, vs, heads, scale=None):
    scale = q.shape[3]**-0.5 if scale is None else scale
    want, err = ref_decode(q, ks, vs, heads, scale)
    top = torch.stack([v.abs().amax() if v.numel() else torch.zeros((), dtype=torch.float64) for v in vs])
    parts = 2.0**-16 if q.dtype == BF16 else 2.0**-24
    bound = err + parts * top[:, None, None] + (2.0**-8 if q.dtype == BF16 else 2.0**-24) * want.abs()
    off = (o.cpu().double()[:, :, 0] - want).abs()
    assert (off <= bound).all(), (off / bound).max()  # NaN fails


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,heads,group,page,layout", [
    (32, 2, 1, 16, "heads"), (32, 1, 5, 64, "joint"), (64, 3, 1, 16, "slots"), (64, 2, 4, 32, "heads"),
    (64, 1, 17, 16, "heads"), (128, 1, 1, 128, "heads"), (128, 2, 8, 16, "joint"), (128, 1, 16, 32, "slots"),
    (128, 1, 40, 64, "heads")])
def test_decode(ia, D, heads, group, page, layout, dtype):
    gen = torch.Generator().manual_seed(D + group)
    lens = [0, 1, 15, 16, 17, 255, 256, 257, 300, 511, 512, 513, 1100, 2, 0]
    cache, ks, vs, _ = make_cache(ia, gen, lens, heads, D, page, layout=layout)
    q = torch.randn((len(lens), heads * group, 1, D), generator=gen).to(dtype)
    o = ia.attn_decode_kv4(q.cuda(), cache)
    check(o, q, ks, vs, heads)
    assert torch.equal(o, ia.attn_decode_kv4(q.cuda(), cache))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 16, 100, 600, 5000, 20011])
def test_decode_one_row(ia, n, D, dtype):
    gen = torch.Generator().manual_seed(n + D)
    cache, ks, vs, _ = make_cache(ia, gen, [n], 2, D, 16)
    q = (torch.randn((1, 6, 1, D), generator=gen) * 2).to(dtype)
    check(ia.attn_decode_kv4(q.cuda(), cache), q, ks, vs, 2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_many_rows(ia, dtype):
    """More rows than are shared out together, whole rows to the workgroups and in shares."""
    gen = torch.Generator().manual_seed(3)
    for rows, heads, longest in ((300, 8, 500), (150, 1, 900), (150, 1, 1400), (600, 4, 1300)):
        lens = torch.randint(0, longest + 1, (rows,), generator=gen).tolist()
        cache, ks, vs, _ = make_cache(ia, gen, lens, heads, 32, 32)
        q = torch.randn((rows, heads, 1, 32), generator=gen).to(dtype)
        check(ia.attn_decode_kv4(q.cuda(), cache), q, ks, vs, heads)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_many_heads(ia, dtype):
    """More heads than workgroups at once: a block of rows in one share."""
    gen = torch.Generator().manual_seed(10)
    few, ks, vs, _ = make_cache(ia, gen, [1030, 0, 513], 8, 32, 16)
    pools = (t.repeat(1, 100, 1, 1) for t in (few.k, few.v, few.k_scale, few.v_scale))
    cache = ia.PagedKV4(*pools, few.table, few.lens)
    q = torch.randn((3, 800, 1, 32), generator=gen).to(dtype)
    o = ia.attn_decode_kv4(q.cuda(), cache)
    check(o, q, [k.repeat(100, 1, 1) for k in ks], [v.repeat(100, 1, 1) for v in vs], 800)


def test_rows_of_the_same_pages(ia):
    """A common beginning held once, and one row twice."""
    gen = torch.Generator().manual_seed(11)
    cache, ks, vs, _ = make_cache(ia, gen, [900, 700, 0, 0], 2, 64, 16)
    cache.table[2] = cache.table[0]
    cache.table[3] = cache.table[0]
    cache.lens[2], cache.lens[3] = 900, 333
    q = torch.randn((4, 6, 1, 64), generator=gen)
    q[2] = q[0]
    ks, vs = ([x[0], x[1], x[0], x[0][:, :333]] for x in (ks, vs))
    o = ia.attn_decode_kv4(q.cuda(), cache)
    check(o, q, ks, vs, 2)
    k, v = ia.kv4_read(cache, 900)
    assert torch.equal(k[2], k[0]) and torch.equal(v[3, :, :333], v[0, :, :333]) and not v[3, :, 333:].any()


def test_captured_twice(ia):
    """Two captured calls of one cache, workspace and result, replayed in turn with eager calls between."""
    gen = torch.Generator().manual_seed(12)
    cache, ks, vs, _ = make_cache(ia, gen, [2000, 31, 0, 700], 2, 64, 16)
    ws = ia.attn_decode_kv4_workspace(cache, 4)
    qs = [torch.randn((4, 4, 1, 64), generator=gen) for _ in range(2)]
    dev = [q.cuda() for q in qs]
    out = torch.empty_like(dev[0])
    want = [ia.attn_decode_kv4(q, cache) for q in dev]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, q in zip(graphs, dev):
        with torch.cuda.graph(graph):
            ia.attn_decode_kv4(q, cache, out=out, workspace=ws)
    for i in range(6):
        graphs[i % 2].replay()
        assert torch.equal(out, want[i % 2])
        assert torch.equal(ia.attn_decode_kv4(dev[1 - i % 2], cache, workspace=ws), want[1 - i % 2])
    check(want[0], qs[0], ks, vs, 2)


def test_decode_strided_and_in_place(ia):
    gen = torch.Generator().manual_seed(4)
    cache, ks, vs, _ = make_cache(ia, gen, [40, 700], 2, 64, 16)
    qkv = torch.randn((2, 1, 8, 64), generator=gen)
    q = qkv[:, :, :4].transpose(1, 2)
    dev = qkv.cuda()
    view = dev[:, :, :4].transpose(1, 2)
    ia.attn_decode_kv4(view, cache, scale=0.3, out=view)
    check(view, q, ks, vs, 2, scale=0.3)
    assert torch.equal(dev[:, :, 4:].cpu(), qkv[:, :, 4:])


def test_decode_bad_rows(ia):
    """Rows longer than max_len and with pages outside the pool are NaN, the others as without them; blocks of
    NaN reach what they are part of."""
    gen = torch.Generator().manual_seed(5)
    for longest in (100, 1500):
        lens = [longest, 60, longest - 1, 30, 90]
        cache, ks, vs, _ = make_cache(ia, gen, lens, 2, 64, 16)
        q = torch.randn((5, 4, 1, 64), generator=gen)
        o = ia.attn_decode_kv4(q.cuda(), cache, max_len=longest - 1)
        assert o[0].isnan().all()
        check(o[1:], q[1:], ks[1:], vs[1:], 2)
        for bad in (-1, cache.k.shape[0], 2**31 - 1):
            keep = int(cache.table[2, 5])
            cache.table[2, 5] = bad
            o = ia.attn_decode_kv4(q.cuda(), cache)
            assert o[2].isnan().all()
            others = [0, 1, 3, 4]
            check(o[others], q[others], [ks[i] for i in others], [vs[i] for i in others], 2)
            cache.table[2, 5] = keep
        page = int(cache.table[4, 1])
        cache.v_scale[page, 1, 1, 3] = 255  # head 1, channels 32 to 63 of position 19
        cache.k_scale[int(cache.table[3, 0]), 0, 0, 2] = 255  # head 0 of row 3
        o = ia.attn_decode_kv4(q.cuda(), cache).cpu()
        nan = torch.zeros((5, 4, 1, 64), dtype=torch.bool)
        nan[4, 2:, :, 32:] = True
        nan[3, :2] = True
        assert torch.equal(o.isnan(), nan)


def test_decode_far_pages(ia):
    """Pages past 2^31 bytes of a pool."""
    pages = (1 << 31) // (128 * 64) + 40
    gen = torch.Generator().manual_seed(6)
    small, ks, vs, _ = make_cache(ia, gen, [300], 1, 128, 128)
    far = ia.PagedKV4.empty(pages, 1, 128, 128, (pages - 1 - torch.arange(3, dtype=torch.int32)).cuda()[None],
                            small.lens)
    for a, b in ((far.k, small.k), (far.v, small.v), (far.k_scale, small.k_scale), (far.v_scale, small.v_scale)):
        a[far.table[0].long()] = b[small.table[0].long()]
    q = torch.randn((1, 4, 1, 128), generator=gen)
    check(ia.attn_decode_kv4(q.cuda(), far), q, ks, vs, 1)
    k, _ = ia.kv4_read(far, 300)
    assert torch.equal(k[0].cpu().double(), ks[0])
    new = torch.randn((1, 1, 300, 128), generator=gen)
    ia.kv4_append(far, new.cuda(), new.cuda())
    assert torch.equal(ia.kv4_read(far, 300)[1].cpu().double(), held(new))


def test_decode_scores_far_apart(ia):
    """One key that outweighs all, and keys so far below that nothing is left of them."""
    gen = torch.Generator().manual_seed(7)
    cache, ks, vs, _ = make_cache(ia, gen, [900], 1, 64, 16)
    q = torch.randn((1, 3, 1, 64), generator=gen) * 40
    check(ia.attn_decode_kv4(q.cuda(), cache), q, ks, vs, 1)
    o = ia.attn_decode_kv4((q * 1e30).cuda(), cache)  # scores past the largest float: +inf makes the row NaN
    s = (q[0, :, 0].double() * 1e30) @ ks[0][0].t() / 8
    assert torch.equal(o[0, :, 0].isnan().all(1).cpu(), (s.abs() > 3.5e38).any(1))


# ---- together ----------------------------------------------------------------------------------------------


def test_generation(ia):
    """Tokens of a layer: projection in 8 bits, append, attention, output projection; then the next chunk of a prompt
    over the cache read back; all captured, too."""
    gen = torch.Generator().manual_seed(8)
    rows, heads, group, D, page = 3, 2, 2, 64, 16
    C, hq = 256, heads * group
    lens = [5, 31, 64]
    for dtype in (F32, BF16):
        cache, ks, vs, free = make_cache(ia, gen, lens, heads, D, page, max_pages=8, spare=12)
        for r, n in enumerate(lens):  # pages for what comes
            k = -(-n // page)
            cache.table[r, k:k + 4] = free[4 * r:4 * r + 4].cuda()
        wq, sq = ia.quantize_i8((torch.randn((C, (hq + 2 * heads) * D), generator=gen) / 16).cuda(), transpose=True)
        wo, so = ia.quantize_i8((torch.randn((hq * D, C), generator=gen) / 16).cuda(), transpose=True)
        x, out = torch.zeros((rows, C), dtype=dtype, device="cuda"), torch.zeros((rows, C), dtype=dtype, device="cuda")
        bufs = {}

        def step():
            cache.lens.add_(1)
            qkv = ia.linear_i8(x, wq, sq).view(rows, hq + 2 * heads, 1, D)
            bufs["q"], bufs["k"], bufs["v"] = qkv[:, :hq], qkv[:, hq:hq + heads], qkv[:, hq + heads:]
            ia.kv4_append(cache, bufs["k"], bufs["v"])
            bufs["o"] = ia.attn_decode_kv4(bufs["q"], cache)
            ia.linear_i8(bufs["o"].view(rows, -1), wo, so, out=out)

        def after(i):
            nonlocal ks, vs
            k, v = held(bufs["k"].cpu()), held(bufs["v"].cpu())
            ks = [torch.cat((a, b), 1) for a, b in zip(ks, k)]
            vs = [torch.cat((a, b), 1) for a, b in zip(vs, v)]
            check(bufs["o"], bufs["q"].cpu(), ks, vs, heads)
            assert torch.equal(out, ia.linear_i8(bufs["o"].view(rows, -1), wo, so))

        for i in range(3):
            x.copy_(torch.randn((rows, C), generator=gen).to(dtype))
            step()
            after(i)
        graph, lens_now = torch.cuda.CUDAGraph(), cache.lens.clone()
        with torch.cuda.graph(graph):
            step()
        assert torch.equal(cache.lens, lens_now)
        for i in range(20):  # over the ends of pages
            x.copy_(torch.randn((rows, C), generator=gen).to(dtype))
            graph.replay()
            torch.cuda.synchronize()
            after(i)
        # the next four tokens of the first row's prompt attend to all of it, and to each other
        n = ks[0].shape[1]
        k, v = ia.kv4_read(cache, n + 4, dtype=dtype)
        assert torch.equal(k[0, :, :n].cpu().double(), ks[0]) and not k[0, :, n:].any()
        new = torch.randn((3, 1, heads, 4, D), generator=gen).to(dtype)
        k[0, :, n:], v[0, :, n:] = new[1, 0].cuda(), new[2, 0].cuda()
        o, _ = ia.attn_fwd(new[0].cuda(), k[:1], v[:1])
        kk, vv = (torch.cat((a[0], b[0].double()), 1) for a, b in ((ks, new[1]), (vs, new[2])))
        s = new[0, 0].double() @ kk.transpose(1, 2) / 8
        s = s.masked_fill(torch.arange(n + 4) > n + torch.arange(4)[:, None], -math.inf)
        want = torch.softmax(s, -1) @ vv
        tol = 1e-4 if dtype == F32 else 2e-2
        assert ((o[0].cpu().double() - want).abs().max() <= tol * want.abs().max())


def test_two_streams(ia):
    """Calls on two streams at once, each with a workspace of its own."""
    gen = torch.Generator().manual_seed(9)
    caches = [make_cache(ia, gen, [3000, 10, 700], 2, 64, 16) for _ in range(2)]
    q = torch.randn((3, 4, 1, 64), generator=gen)
    dev = q.cuda()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        outs = [ia.attn_decode_kv4(dev, c[0], stream=s) for c, s in zip(caches, streams)]
    torch.cuda.synchronize()
    for o, (_, ks, vs, _) in zip(outs, caches):
        check(o, q, ks, vs, 2)
