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


@pytest.mark.parametrize("N,K", [(1024, 8192), (130, 9000), (8200, 8200)])
def test_linear_with_one_workspace(ia, N, K):
    """A workspace for the most rows, and calls of fewer: the bits that they have with one of their own."""
    gen = torch.Generator(device="cuda").manual_seed(N)
    w, sw = ia.quantize_i8(torch.randn((K, N), generator=gen, device="cuda"), transpose=True)
    most = 2100
    ws = ia.linear_i8_workspace(most, N, K)
    product_ws = ia.gemm_i8_workspace(most, N, K)
    x = torch.randn((most, K), generator=gen, device="cuda").bfloat16()
    for M in (most, 1030, 256, 190, 129, 128, 100, 64, 9, 1):
        ws.fill_(0xFF)
        product_ws.fill_(0xFF)
        want = ia.linear_i8(x[:M], w, sw)
        assert torch.equal(ia.linear_i8(x[:M], w, sw, workspace=ws), want)
        q, s = ia.quantize_i8(x[:M])
        assert torch.equal(ia.gemm_i8(q, s, w, sw, dtype=BF16, workspace=product_ws), want)
