"""The order of beam selection where scores are equal or close, at every row alignment and in every
width of a workgroup, on the GPU against 64 bits on the CPU.

Tolerances.  A term exp(d), d <= 0 its logit's distance from the part's largest, has the subtraction
rounded (2^-24 |d|), the product with log2 e (2^-24 |d|) and that constant (less than 2^-26 |d|), v_exp_f32
(2^-23) and two sums of a group of four (2^-23); all else is in 64 bits.  So the lse is off by
(2.25 E + 4) 2^-24 with E the mean of |d| under the terms' shares, which the test takes from its row.
"""
import math

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


def rows_at(logits, pad, shift):
    """The rows on the GPU, vocab + pad elements apart and shift elements behind an aligned address; around them
    lies what must not be read into a result."""
    rows, vocab = logits.shape
    wide = torch.full((rows * (vocab + pad) + shift + 16,), math.inf, dtype=logits.dtype, device="cuda")
    view = torch.as_strided(wide, (rows, vocab), (vocab + pad, 1), shift)
    view.copy_(logits)
    return view


# groups * beams and vocab choose the columns of a workgroup: 2048, 4096 and 8192 all occur
EQUAL = [(1, 8, 1001), (1, 8, 3001), (2, 8, 8193), (1, 8, 50257), (16, 16, 1001), (3, 32, 8193), (4, 8, 20011),
         (3, 8, 50257), (8, 8, 50257), (32, 8, 9001), (1, 4, 7), (2, 3, 2049)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("pad,shift", [(0, 0), (0, 3), (2, 1), (7, 5)])
@pytest.mark.parametrize("groups,beams,vocab", EQUAL)
def test_equal_beams_lower_first(ia, groups, beams, vocab, pad, shift, dtype):
    """Beams of the same logits and scores: all scores of a token are equal, so every token's beams come in order."""
    print(f"[case] equal beams {groups}x{beams} V{vocab} pad {pad} shift {shift} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab + pad)
    one = (torch.randn(groups, 1, vocab, generator=gen) * 2).to(dtype)
    logits = one.expand(groups, beams, vocab).reshape(groups * beams, vocab)
    tokens, parents, scores, _ = ia.beam_select(rows_at(logits, pad, shift), torch.full((groups, beams), -7.25).cuda())
    for g in range(groups):
        # distinct values from the top, each by every beam, then by its lowest token
        order = torch.sort(one[g, 0].float(), descending=True, stable=True)
        want, i = [], 0
        while len(want) < beams:
            same = [int(t) for t, v in zip(order.indices[i:i + beams], order.values[i:i + beams]) if v == order.values[i]]
            want += [(b, t) for b in range(beams) for t in same]
            i += len(same)
        assert list(zip(parents[g].tolist(), tokens[g].tolist())) == want[:beams]
        assert (scores[g, :1] == scores[g][tokens[g] == tokens[g, 0]]).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,pad", [
    (1, 8, 50257, 0), (4, 16, 50257, 0), (5, 16, 30011, 3), (64, 4, 16385, 0), (3, 32, 8193, 1), (2, 4, 4099, 0),
    (1, 4, 100003, 0), (2, 8, 300007, 1),  # more parts than lanes join at a time
])
def test_ordinary_logits(ia, groups, beams, vocab, pad, dtype):
    """Ordinary logits of odd vocabularies in every width: the candidates of all beams in 64 bits, and each score."""
    print(f"[case] ordinary logits {groups}x{beams} V{vocab} pad {pad} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab + beams)
    logits = (torch.randn(groups * beams, vocab, generator=gen) * 2.5).to(dtype)
    logits[:, -1] = logits[:, 0] = 9.0  # the edge columns among the best
    base = torch.randn(groups, beams, generator=gen) - 20.0
    tokens, parents, scores, _ = (x if x is None else x.cpu() for x in ia.beam_select(rows_at(logits, pad, 0), base.cuda()))
    x = logits.double().view(groups, beams, vocab)
    every = base.double()[:, :, None] + (x - torch.logsumexp(x, 2, keepdim=True))
    best = torch.sort(every.view(groups, -1), dim=1, descending=True, stable=True)
    assert torch.equal(parents.long() * vocab + tokens, best.indices[:, :beams])
    p = torch.softmax(x, 2)
    mean = (p * (x.amax(2, keepdim=True) - x)).sum(2).amax(1)  # E of the docstring, the largest of a group
    bound = (2.25 * mean[:, None] + 4) * 2.0**-24 + 2.0**-24 * best.values[:, :beams].abs()
    assert ((scores.double() - best.values[:, :beams]).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab,peak", [(50257, 7.75), (50257, 0.375), (1001, 5.5), (40000, 20.0)])
def test_lse_of_flat_rows(ia, vocab, peak, dtype):
    """Nearly flat rows with one peak, whose terms all round alike: scores near 0, which show the lse's error."""
    print(f"[case] flat rows V{vocab} peak {peak} {dtype}", flush=True)
    logits = torch.full((2, vocab), -0.34375, dtype=dtype)
    logits[:, vocab // 3] += peak
    x = logits.double()
    lse = torch.logsumexp(x, 1)
    base = (lse - x.amax(1)).float()[:, None]
    tokens, _, scores, _ = ia.beam_select(rows_at(logits, 1, 0), base.cuda())
    want = base.double() + (x.amax(1) - lse)[:, None]
    p = torch.softmax(x, 1)
    mean = (p * (x.amax(1, keepdim=True) - x)).sum(1)[:, None]
    assert (tokens == vocab // 3).all()
    assert ((scores.double().cpu() - want).abs() <= (2.25 * mean + 4) * 2.0**-24 + 2.0**-24 * want.abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("groups,beams,vocab,rest", [(1, 3, 200, -1.0), (2, 8, 9001, -2.0), (3, 4, 50257, -8.0),
                                                     (2, 32, 9001, None)])
def test_logits_decide_within_a_beam(ia, groups, beams, vocab, rest, dtype):
    """Logits that differ by less than their score's last bit in 64 bits: within a beam the larger one is first all
    the same.  rest None: all logits are such, more candidates of one score than are ranked at a time."""
    print(f"[case] tiny logits {groups}x{beams} V{vocab} rest {rest} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    n = vocab if rest is None else 2 * beams
    tiny = (torch.arange(1, 65) * 2.0**-90).to(dtype)  # few enough for bf16 to tell them apart
    one = torch.full((vocab,), 0.0 if rest is None else rest, dtype=dtype)
    where = torch.randperm(vocab, generator=gen)[:n]
    one[where] = tiny[torch.arange(n) % 64] if rest is None else tiny[:n]
    logits = one.expand(groups * beams, vocab).contiguous()
    tokens, parents, scores, _ = ia.beam_select(rows_at(logits, 1, 0), torch.full((groups, beams), -3.5).cuda())
    want = torch.sort(one.float(), descending=True, stable=True).indices[:beams]
    for g in range(groups):  # all scores are equal, so beam 0's best are taken
        assert parents[g].tolist() == [0] * beams and tokens[g].tolist() == want.tolist()
        assert (scores[g] == scores[g, 0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("value", ["lowest", "largest", 2.0**40, -(2.0**100), 2.0**20])
@pytest.mark.parametrize("vocab", [40, 9001])
def test_logits_far_from_zero(ia, vocab, value, dtype):
    """A beam whose logits are all at the type's lowest value (all tokens masked), or far from 0: its score counts as much
    as any other's, by (score + (logit - maximum)) - log(sum)."""
    print(f"[case] logits at {value} V{vocab} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    groups, beams = 2, 4
    far = {"lowest": torch.finfo(dtype).min, "largest": torch.finfo(dtype).max}.get(value, value)
    logits = (torch.randn(groups, beams, vocab, generator=gen) * 2).to(dtype)
    logits[0, 1:3] = far
    logits[1] = far
    logits[1, :, vocab // 2:] = torch.tensor(far * (0.5 if far > 0 else 1.0), dtype=dtype)  # half of them, or all, at the top
    logits = logits.view(groups * beams, vocab)
    scores = torch.randn(groups, beams, generator=gen) - torch.tensor([[9.0, 2.0, 1.0, 9.0], [5.0, 5.0, 5.0, 5.0]])
    scores[1, 2] = scores[1, 1]
    tokens, parents, out, _ = (x if x is None else x.cpu() for x in ia.beam_select(rows_at(logits, 1, 0), scores.cuda()))
    x = logits.double().view(groups, beams, vocab)
    d = x - x.amax(2, keepdim=True)
    p = torch.exp(d)
    every = scores.double()[:, :, None] + (d - p.sum(2, keepdim=True).log())
    best = torch.sort(every.view(groups, -1), dim=1, descending=True, stable=True)
    assert (parents.long() * vocab + tokens).tolist() == best.indices[:, :beams].tolist()
    mean = (p / p.sum(2, keepdim=True) * -d).sum(2).amax(1)
    bound = (2.25 * mean[:, None] + 4) * 2.0**-24 + 2.0**-24 * best.values[:, :beams].abs()
    assert ((out.double() - best.values[:, :beams]).abs() <= bound).all()
