"""Workspaces of weights in 8 bits and a cache in 4, without a GPU: one that was sized for the longest rows, or for the
most of them, is enough for every shorter or smaller call.  (Every call here carries a workspace at an odd address, so
that it returns before any HIP call: 6 where the workspace is too small, 7 where its size is enough.)"""
import ctypes

import pytest

import inferno_amd as ia
from inferno_amd import Strides
from test_quant_args import FAKE, cache, decode, linear

ODD = FAKE + 16


def decode_bytes(c, hq, max_len):
    n = ctypes.c_size_t()
    assert ia.lib().inf_attn_decode_kv4_workspace(ctypes.byref(c), hq, max_len, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("rows,heads,hq,D,longest", [
    (1, 8, 32, 128, 32768), (1, 12, 12, 64, 8192), (4, 2, 16, 128, 131072), (32, 12, 12, 64, 4096), (3, 1, 40, 32, 65536),
    (100, 2, 2, 32, 20000), (64, 8, 32, 128, 8192), (150, 3, 6, 64, 9000)])
def test_decode_workspace_of_the_longest(rows, heads, hq, D, longest):
    pages = -(-longest // 16)
    c = cache(rows=rows, heads=heads, D=D, max_pages=pages, table_stride=pages, n_pages=rows * pages)
    q = Strides(hq * D, D, D, 1)
    whole = decode_bytes(c, hq, longest)
    assert whole
    before = 0
    for max_len in sorted({1, 1024, 1025, *range(1, longest, max(1, longest // 500)), longest}):
        n = decode_bytes(c, hq, max_len)
        assert before <= n <= whole
        before = n
        if n:
            assert decode(c, sq=q, so=q, hq=hq, max_len=max_len, ws=ODD, n=whole) == 7
            assert decode(c, sq=q, so=q, hq=hq, max_len=max_len, ws=ODD, n=n) == 7
            assert decode(c, sq=q, so=q, hq=hq, max_len=max_len, ws=ODD, n=255) == 6


def product_bytes(call, M, N, K):
    n = ctypes.c_size_t()
    assert getattr(ia.lib(), f"inf_{call}_i8_workspace")(M, N, K, ctypes.byref(n)) == 0
    return n.value


# one short K range, several, none; few outputs and many; the few-row kernel's border and past it
@pytest.mark.parametrize("N,K", [(4096, 16384), (1024, 8192), (130, 9000), (2048, 4096), (33, 100000), (64, 131071),
                                 (768, 768), (16384, 4096), (50257, 768), (1, 1), (300, 8192), (8193, 8193)])
def test_product_workspace_of_the_most_rows(N, K):
    ld = -(-K // 16) * 16
    rows = (*range(1, 300), *range(300, 1400, 37), 2047, 2048, 2049, 4096, 8192)
    for call in ("gemm", "linear"):
        before = 0
        for M in rows:
            n = product_bytes(call, M, N, K)
            assert n >= before  # one's is enough for all before it
            before = n
    for M in rows[8:]:  # from nine rows on the linear layer needs some
        args = dict(M=M, N=N, K=K, ldx=ld, ldw=ld, ldy=N, y=1 << 50, ws=ODD)
        assert linear(**args, n=product_bytes("linear", M, N, K)) == 7
        assert linear(**args, n=M * K - 1) == 6


def test_sizes_kept_are_bounded():
    """A server that asks for every length and number of rows keeps some sizes, not all that it ever asked for."""
    torch = pytest.importorskip("torch")
    quant, paged = ia.quant, ia.paged
    for M in range(1, 6000):
        assert quant._product_bytes("inf_linear_i8_workspace", M, 64, 64) == product_bytes("linear", M, 64, 64)
    assert quant._product_bytes.cache_info().currsize <= 4096
    table, lens = torch.zeros((2, 512), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros((4, 1, 16, 64))
    for c, call, more in ((ia.PagedKV4.empty(4, 1, 16, 64, table, lens), "inf_attn_decode_kv4_workspace", ()),
                          (ia.PagedKV(pool, pool, table, lens), "inf_attn_decode_paged_workspace", (0,))):
        for n in range(1, 6000):
            size = paged._bytes(c, call, 1, n, *more)
            assert size == paged._bytes(c, call, 1, n, *more)
        assert len(c.sizes) <= 4096
