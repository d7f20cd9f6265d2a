"""Eviction on the GPU: positions that lie in pages outside the pool, and the widths and sizes that the moves
have variants for, against the plain selection of test_gpu_paged.py.  What is kept has to be equal."""
import math

import pytest

torch = pytest.importorskip("torch")

import test_gpu_paged as base  # noqa: E402
from test_gpu_paged import BF16, F32, ia  # noqa: E402,F401

pytestmark = pytest.mark.gpu


def same(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("in_place", [True, False])
def test_kept_position_in_a_page_outside_the_pool(ia, in_place, D, dtype):  # noqa: F811
    """A hole whose key and value have no page reads as NaN, not as what was evicted from it."""
    print(f"[case] evict from a bad page D{D} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(D)
    lens, heads, page, keep = [100, 90, 64], 2, 16, 40
    c, _, _, _ = base.make_cache(ia, gen, lens, heads, D, page, dtype)
    t = c.table.clone()
    t[0, 5], t[1, 3], t[2, 3] = c.k.shape[0], -1, 1 << 30  # positions 80 to 95, 48 to 63, 48 to 63
    c.table = t
    w = torch.rand(3, heads, c.capacity, generator=gen)
    w[0, :, 83] = w[0, :, 95] = w[1, 1, 50] = 9.0  # kept, in those pages; row 2 loses all of its page
    w[0, :, 80:83] = w[0, :, 84:95] = 0.0
    w[1, :, 48:64] *= 0.0
    w[1, 1, 50] = 9.0
    w[2, :, 48:64] = 0.0
    pos = torch.arange(c.capacity, dtype=torch.int32).expand(3, heads, c.capacity).contiguous()
    k0, v0 = c.k.cpu().clone(), c.v.cpu().clone()
    table = t.cpu()
    wd, pd = w.cuda(), pos.cuda()
    out = {} if in_place else dict(weights_out=torch.zeros_like(wd), positions_out=torch.zeros_like(pd))
    new = ia.kv_evict(c, wd, pd, keep, 0, **out)
    wo, po = out.get("weights_out", wd).cpu(), out.get("positions_out", pd).cpu()
    assert new.tolist() == [keep] * 3
    holes_of = {}
    for r, n in enumerate(lens):
        for h in range(heads):
            holes, src = base.ref_evict(w[r, h].numpy(), pos[r, h].numpy(), n, keep, 0)
            for a, b in zip(holes, src):
                pa, pb = int(table[r, a // page]), int(table[r, b // page])
                inside = 0 <= pb < k0.shape[0]
                holes_of.setdefault((r, h), []).append(inside)
                k0[pa, h, a % page] = k0[pb, h, b % page] if inside else math.nan
                v0[pa, h, a % page] = v0[pb, h, b % page] if inside else math.nan
                assert wo[r, h, a] == w[r, h, b] and po[r, h, a] == b
    assert same(c.k.cpu(), k0) and same(c.v.cpu(), v0)
    assert [sum(not x for x in holes_of[r, h]) for r in range(3) for h in range(heads)] == [2, 2, 0, 1, 0, 0]
    c.lens = new
    got = ia.attn_decode_paged(base.rnd(gen, (3, heads, 1, D), dtype).cuda(), c, max_len=keep)
    nan = got.isnan().all(dim=3)[:, :, 0]
    assert nan.tolist() == [[True, True], [False, True], [False, False]]
    assert got[~nan[:, :, None].expand(-1, -1, 1)].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,D,page,longest,keep,recent", [
    (8, 12, 128, 16, 1500, 700, 32),   # more than 4096 groups of moves: four a thread
    (40, 9, 128, 32, 1111, 600, 0),
    (2, 3, 128, 16, 6000, 5000, 100),
    (3, 2, 64, 1, 300, 299, 7),
])
def test_ragged_rows(ia, rows, heads, D, page, longest, keep, recent, dtype):  # noqa: F811
    """Rows of random lengths, in place and out of place."""
    print(f"[case] evict ragged {rows}x{heads} D{D} keep {keep} of {longest} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(rows + heads)
    lens = torch.randint(keep - 3, longest + 1, (rows,), generator=gen).tolist()
    lens[0], lens[-1] = longest, 1
    c, _, _, _ = base.make_cache(ia, gen, lens, heads, D, page, dtype)
    w = torch.rand(rows, heads, c.capacity, generator=gen)
    pos = torch.rand(w.shape, generator=gen).argsort(2).to(torch.int32)
    k0, v0 = c.k.clone(), c.v.clone()
    kw, vw, ww, pw = k0.clone(), v0.clone(), w.clone(), pos.clone()
    table = c.table.cpu()
    for r, n in enumerate(lens):
        for h in range(heads):
            holes, src = (torch.tensor(x, dtype=torch.long)
                          for x in base.ref_evict(w[r, h].numpy(), pos[r, h].numpy(), n, keep, recent))
            pa, pb = table[r, holes // page].long().cuda(), table[r, src // page].long().cuda()
            a, b = (holes % page).cuda(), (src % page).cuda()
            kw[pa, h, a], vw[pa, h, a] = k0[pb, h, b], v0[pb, h, b]
            ww[r, h, holes], pw[r, h, holes] = w[r, h, src], pos[r, h, src]
    want = [min(n, keep) for n in lens]
    for in_place in (False, True):
        c.k.copy_(k0)
        c.v.copy_(v0)
        wd, pd = w.cuda(), pos.cuda()
        wo, po = (wd, pd) if in_place else (torch.full_like(wd, -3.0), torch.full_like(pd, -4))
        new = ia.kv_evict(c, wd, pd, keep, recent, weights_out=wo, positions_out=po)
        assert new.tolist() == want
        assert same(c.k, kw) and same(c.v, vw)
        for r, m in enumerate(want):
            assert torch.equal(wo[r, :, :m].cpu(), ww[r, :, :m]) and torch.equal(po[r, :, :m].cpu(), pw[r, :, :m])
            assert in_place or ((wo[r, :, m:] == -3.0).all() and (po[r, :, m:] == -4).all())
            assert not in_place or (torch.equal(wo[r, :, m:].cpu(), w[r, :, m:]) and
                                    torch.equal(po[r, :, m:].cpu(), pos[r, :, m:]))
