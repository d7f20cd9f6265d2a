"""Calls of weights in 8 bits and a cache in 4 as programs make them: one workspace for rows that grow."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv4 import check, ia, make_cache  # noqa: E402,F401

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("rows,heads,group,D,dtype", [(1, 8, 4, 128, BF16), (3, 2, 1, 64, F32), (70, 1, 5, 32, BF16)])
def test_decode_with_one_workspace(ia, rows, heads, group, D, dtype):
    """A workspace for the capacity, the lengths of now as the bound."""
    gen = torch.Generator().manual_seed(rows + D)
    longest = 9000 if rows < 4 else 1500
    cache, ks, vs, _ = make_cache(ia, gen, [longest - 7 * i for i in range(rows)], heads, D, 32)
    ws = ia.attn_decode_kv4_workspace(cache, heads * group)
    q = torch.randn((rows, heads * group, 1, D), generator=gen).to(dtype)
    lens = cache.lens.clone()
    for bound in sorted({1, 1000, 1025, 1281, 1500, *range(2000, longest, 1511), longest} & set(range(longest + 1))):
        ws.fill_(0xFF)
        cache.lens.copy_(lens.clamp(max=bound))
        o = ia.attn_decode_kv4(q.cuda(), cache, max_len=bound, workspace=ws)
        check(o, q, [k[:, :bound] for k in ks], [v[:, :bound] for v in vs], heads)
