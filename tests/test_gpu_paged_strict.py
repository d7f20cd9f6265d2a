"""Attention over a paged cache, its outputs compared so that NaN and a bound that is no number fail too.

Every unused slot, page and table entry of the caches is NaN or no page, so a read past a row's end or from a
wrong page shows as NaN in the output.  The cases, references and tolerances are those of test_gpu_paged.py.
"""
import math

import pytest

torch = pytest.importorskip("torch")

import test_gpu_paged as base  # noqa: E402
from test_gpu_paged import BF16, F32, ia  # noqa: E402,F401


def check_decode(q, out, ks, vs, heads, scale, dtype, skip=()):
    o, ps, err = base.ref_decode(q, ks, vs, heads, scale)
    got = out[:, :, 0].double().cpu()
    if dtype == BF16:
        err = err * (1 + 2.0**-16 / (64 * 2.0**-24)) + o.abs() * 2.0**-8
    good = (got - o).abs() <= err + 1e-30
    for r in range(q.shape[0]):
        if r not in skip:
            assert err[r].isfinite().all(), (r, ks[r].shape)
            assert good[r].all(), (r, ks[r].shape, float((got[r] - o[r]).abs().max()), float(err[r].max()))
    return ps


@pytest.fixture
def strict(monkeypatch):
    monkeypatch.setattr(base, "check_decode", check_decode)


def test_the_comparison_sees_nan():
    """On the CPU: the right output passes; NaN everywhere, in one element, or infinity fail."""
    gen = torch.Generator().manual_seed(0)
    ks, vs = ([torch.randn(2, n, 32, generator=gen).double() for n in (40, 0, 7)] for _ in range(2))
    q = torch.randn(3, 4, 1, 32, generator=gen)
    scale = 32**-0.5
    right = base.ref_decode(q, ks, vs, 2, scale)[0].float()[:, :, None]
    check_decode(q, right, ks, vs, 2, scale, F32)
    for where in (slice(None), (0, 1, 0, 31), (1, 0, 0, 0), (2, 3)):
        for value in (math.nan, math.inf):
            wrong = right.clone()
            wrong[where] = value
            with pytest.raises(AssertionError):
                check_decode(q, wrong, ks, vs, 2, scale, F32)


@pytest.mark.gpu
def test_decode(ia, strict, heads, group, page, max_pages, lens, D, dtype):  # noqa: F811
    base.test_decode(ia, heads, group, page, max_pages, lens, D, dtype)


@pytest.mark.gpu
def test_decode_many_rows(ia, strict, rows, heads, group, D, page, longest, weigh, dtype):  # noqa: F811
    base.test_decode_many_rows(ia, rows, heads, group, D, page, longest, weigh, dtype)


@pytest.mark.gpu
def test_decode_layouts(ia, strict, layout, dtype):  # noqa: F811
    base.test_decode_layouts(ia, layout, dtype)


@pytest.mark.gpu
def test_decode_bad_rows_are_nan(ia, strict, dtype):  # noqa: F811
    base.test_decode_bad_rows_are_nan(ia, dtype)


@pytest.mark.gpu
def test_decode_infinite_scores(ia, strict, dtype):  # noqa: F811
    base.test_decode_infinite_scores(ia, dtype)


@pytest.mark.gpu
def test_decode_far_offsets(ia, strict):  # noqa: F811
    base.test_decode_far_offsets(ia)


@pytest.mark.gpu
def test_decode_long(ia, strict, dtype):  # noqa: F811
    base.test_decode_long(ia, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,heads,group,longest", [(1, 2, 1, 1000), (70, 2, 18, 300), (600, 4, 1, 200)])
def test_output_over_the_queries(ia, rows, heads, group, longest, dtype):  # noqa: F811
    """o may be q itself: whole rows to a workgroup, and shares with a join."""
    print(f"[case] paged decode in place {rows} rows {heads}x{group} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, longest + 1, (rows,), generator=gen).tolist()
    lens[0] = longest
    c, ks, vs, _ = base.make_cache(ia, gen, lens, heads, 64, 16, dtype)
    q = base.rnd(gen, (rows, heads * group, 1, 64), dtype, 1.5)
    for weigh in (False, True):
        w = torch.zeros(c.meta_shape, device="cuda") if weigh else None
        x = q.cuda()
        assert ia.attn_decode_paged(x, c, max_len=longest, weights_out=w, out=x) is x
        check_decode(q, x, ks, vs, heads, ia.default_scale(64), dtype)


for _name in ("test_decode", "test_decode_many_rows", "test_decode_layouts", "test_decode_bad_rows_are_nan",
              "test_decode_infinite_scores", "test_decode_long"):  # the parameters of the same tests there
    _test = globals()[_name]
    _test.pytestmark = [*_test.pytestmark, *getattr(base, _name).pytestmark]
