"""Sizes whose launch would need 2^32 threads or more, which no grid has: refused as shapes, on the host (no call here
gets past its checks)."""
import ctypes

import pytest

import inferno_amd as ia
from inferno_amd import Strides
from test_paged_args import FAKE, cache, decode, evict, select

SHAPE = 2
ROOM = 1 << 60


def test_decode():
    flat = Strides(0, 0, 64, 1)  # a cache that is only read may repeat itself
    wide = cache(rows=1, heads=1 << 24, sk=flat, sv=flat)
    rows = Strides((1 << 24) * 64, 64, 64, 1)
    assert decode(wide, hq=1 << 24, sq=rows, so=rows, ws=FAKE << 8, n=ROOM) == SHAPE
    tiles = cache(rows=1, heads=(1 << 24) // 17, sk=flat, sv=flat)
    assert decode(tiles, hq=(1 << 24) // 17 * 17, sq=rows, so=rows, ws=FAKE << 8, n=16) != SHAPE  # fits: the next check's
    long = cache(rows=32, page_size=1024, max_pages=1 << 20, table_stride=1 << 20)
    four = Strides(256, 64, 64, 1)
    assert decode(long, hq=2, sq=four, so=four, max_len=1 << 30, w_out=FAKE, ws=FAKE << 8, n=ROOM) == SHAPE
    assert decode(long, hq=2, sq=four, so=four, max_len=1 << 30, ws=None, n=0) == 6  # without weights it fits


def test_evict():
    def heads(n, **kw):
        s = Strides(n * 16 * 64, 16 * 64, 64, 1)
        return cache(rows=1, heads=n, sk=s, sv=s, max_pages=512, table_stride=512, **kw)

    assert evict(heads(1 << 22), max_len=4097, n=ROOM) == SHAPE       # 1024 threads a row and head
    assert evict(heads(1 << 22), max_len=4096, n=0) == 6              # 256
    assert evict(heads(1 << 24), max_len=64, n=ROOM) == SHAPE
    s = Strides(2 * 1024 * 128, 1024 * 128, 128, 1)
    long = cache(D=128, page_size=1024, max_pages=1 << 20, table_stride=1 << 20, sk=s, sv=s)
    assert evict(long, keep=1 << 28, max_len=1 << 29, n=ROOM) == SHAPE  # 2^26 workgroups of moves
    assert evict(long, keep=1 << 25, max_len=1 << 29, n=0) == 6         # 2^23


@pytest.mark.parametrize("groups,beams,vocab,status", [
    (1 << 22, 1, 1, SHAPE), (1 << 20, 16, 1, SHAPE), (1 << 12, 32, 8192 * 129, SHAPE),
    ((1 << 22) - 1, 1, 1, 0), ((1 << 20) - 1, 16, 1, 0), (1 << 12, 32, 8192 * 127, 0),
])
def test_select(groups, beams, vocab, status):
    n = ctypes.c_size_t(7)
    assert ia.lib().inf_beam_select_workspace(groups, beams, vocab, ctypes.byref(n)) == status
    assert (n.value > 0) == (status == 0)
    assert select(groups=groups, beams=beams, vocab=vocab, ld=vocab, eos=-1, n=0) == (status or 6)
