"""Workspaces of weights in 8 bits and a cache in 4, without a GPU: one that was sized for the longest rows, or for the
most of them, is enough for every shorter or smaller call.  (Every call here carries a workspace at an odd address, so
that it returns before any HIP call: 6 where the workspace is too small, 7 where its size is enough.)"""
import ctypes

import pytest

import inferno_amd as ia
from inferno_amd import Strides
from test_quant_args import FAKE, cache, decode

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
