"""Results of weights in 8 bits and a cache in 4 that lie over what other workgroups still read or write: refused on the
host, without a GPU (every call here is refused, so it returns before any HIP call)."""
import ctypes

import pytest

import inferno_amd as ia
from inferno_amd import Strides
from test_quant_args import cache

OVERLAP = 3
BIG = 1 << 34
# a cache of 4 rows, 2 heads of 64, 32 pages of 16 slots: what lies where, and its bytes
POOL = dict(k=32 * 1024, v=32 * 1024, k_scale=32 * 64, v_scale=32 * 64, table=4 * 4 * 4, lens=16)
AT = {name: (i + 1) * BIG for i, name in enumerate(POOL)}


def far_cache(**kw):
    return cache(**{**AT, **kw})


def places(of, n, m, align):
    """Addresses of n bytes that meet the m bytes from `of` on, at either end and inside."""
    return sorted({of, of + (m - 1) // align * align, of - (n - 1) // align * align, of + m // 2 // align * align})


NEW = Strides(8 * 2 * 64, 64, 2 * 64, 1)  # [rows, heads, T, D] out of [rows, T, heads, D]
NEW_BYTES = 4 * 8 * 2 * 64 * 4


def read(c, k, v, first=None, s=NEW, sv=None, T=8, dt=0):
    return ia.lib().inf_kv4_read(ctypes.byref(c), first, T, k, s, v, sv or s, dt, None)


@pytest.mark.parametrize("what", POOL)
def test_read_over_the_cache(what):
    for at in places(AT[what], NEW_BYTES, POOL[what], 16):
        assert read(far_cache(), at, 20 * BIG) == OVERLAP
        assert read(far_cache(), 20 * BIG, at) == OVERLAP


def test_read_over_its_arguments():
    for at in places(20 * BIG, NEW_BYTES, NEW_BYTES, 16):
        assert read(far_cache(), 20 * BIG, at) == OVERLAP  # keys over values
        assert read(far_cache(), 20 * BIG, at, sv=Strides(8 * 2 * 64, 8 * 64, 64, 1)) == OVERLAP
    for at in places(21 * BIG, NEW_BYTES, 16, 16):
        assert read(far_cache(), at, 20 * BIG, first=21 * BIG) == OVERLAP
        assert read(far_cache(), 20 * BIG, at, first=21 * BIG) == OVERLAP


def test_read_side_by_side_but_one():
    """Keys and values out of [rows, T, 3, heads, D], where the values begin a head early."""
    s = Strides(8 * 3 * 128, 64, 3 * 128, 1)
    assert read(far_cache(), 20 * BIG, 20 * BIG + 4 * 64, s=s) == OVERLAP
    assert read(far_cache(), 20 * BIG, 20 * BIG + 4 * 5 * 64, s=s) == OVERLAP  # the next token's


ROW = Strides(4 * 64, 64, 64, 1)  # q and o [rows, q_heads, 1, D], dense
ROW_BYTES = 4 * 4 * 64 * 4


def decode(c, q, o, sq=ROW, so=ROW, ws=None, n=0, max_len=64, dt=0):
    return ia.lib().inf_attn_decode_kv4(ctypes.byref(c), q, sq, o, so, 4, max_len, 0.125, dt, ws, n, None)


@pytest.mark.parametrize("what", POOL)
def test_attention_over_the_cache(what):
    for at in places(AT[what], ROW_BYTES, POOL[what], 16):
        assert decode(far_cache(), 20 * BIG, at) == OVERLAP


def test_attention_over_its_queries():
    """The result may be the queries themselves, but not other heads' or rows' of them."""
    for at in places(20 * BIG, ROW_BYTES, ROW_BYTES, 16):
        if at != 20 * BIG:
            assert decode(far_cache(), 20 * BIG, at) == OVERLAP
    assert decode(far_cache(), 20 * BIG, 20 * BIG, so=Strides(64, 4 * 64, 64, 1)) == OVERLAP  # [heads, rows]
    wide = Strides(8 * 64, 64, 64, 1)  # out of [rows, 8 heads]
    assert decode(far_cache(), 20 * BIG, 20 * BIG + 4 * 3 * 64, sq=wide, so=wide) == OVERLAP
    assert decode(far_cache(), 20 * BIG, 20 * BIG + 4 * 5 * 64, sq=wide, so=wide) == OVERLAP  # the next row's


def test_attention_over_its_workspace():
    rows, longest = 3, 16000
    c = far_cache(rows=rows, max_pages=1000, table_stride=1000, n_pages=3000)
    n = ctypes.c_size_t()
    assert ia.lib().inf_attn_decode_kv4_workspace(ctypes.byref(c), 4, longest, ctypes.byref(n)) == 0 and n.value
    size = dict(k=3000 * 1024, v=3000 * 1024, k_scale=3000 * 64, v_scale=3000 * 64, table=3000 * 4, lens=12)
    q, o, mine = 20 * BIG, 21 * BIG, rows * 4 * 64 * 4
    for of, m in [(AT[name], size[name]) for name in POOL] + [(q, mine), (o, mine)]:
        for at in (of, of + (m - 1) // 256 * 256, of - (n.value - 1) // 256 * 256):
            assert decode(c, q, o, ws=at, n=n.value, max_len=longest) == OVERLAP


def append(c, k, v, counts=None, s=NEW, T=8, dt=0):
    return ia.lib().inf_kv4_append(ctypes.byref(c), k, s, v, s, counts, T, dt, None)


@pytest.mark.parametrize("what", ["k", "v", "k_scale", "v_scale"])
def test_append_over_what_it_reads(what):
    for at in places(AT[what], NEW_BYTES, POOL[what], 16):
        assert append(far_cache(), at, 20 * BIG) == OVERLAP
        assert append(far_cache(), 20 * BIG, at) == OVERLAP
    for at in places(AT[what], 16, POOL[what], 4):
        assert append(far_cache(), 20 * BIG, 21 * BIG, counts=at) == OVERLAP
        assert append(far_cache(lens=at), 20 * BIG, 21 * BIG) == OVERLAP
        assert append(far_cache(table=at), 20 * BIG, 21 * BIG) == OVERLAP


@pytest.mark.parametrize("a", ["k", "v", "k_scale", "v_scale"])
@pytest.mark.parametrize("b", ["k", "v", "k_scale", "v_scale"])
def test_append_to_pools_over_each_other(a, b):
    if a != b:
        for at in places(AT[a], POOL[b], POOL[a], 16):
            assert append(far_cache(**{b: at}), 20 * BIG, 21 * BIG) == OVERLAP


# ---- matrices in 8 bits


def product_bytes(call, M, N, K):
    n = ctypes.c_size_t()
    assert getattr(ia.lib(), f"inf_{call}_i8_workspace")(M, N, K, ctypes.byref(n)) == 0 and n.value
    return n.value


def test_workspace_over_what_is_read():
    M, N, K = 64, 130, 9000  # in K ranges
    x, w, sw, b, y, sx = (i * BIG for i in range(20, 26))
    ld = 9008
    for dt, es in ((0, 4), (1, 2)):
        n = product_bytes("linear", M, N, K)
        for of, m in ((x, M * K * es), (w, (N - 1) * ld + K), (sw, 4 * N), (b, es * N), (y, M * N * es)):
            for at in (of, of + (m - 1) // 256 * 256, of - (n - 1) // 256 * 256):
                assert ia.lib().inf_linear_i8(M, N, K, x, K, w, ld, sw, b, y, N, dt, at, n, None) == OVERLAP
        n = product_bytes("gemm", M, N, K)
        for of, m in ((x, (M - 1) * ld + K), (w, (N - 1) * ld + K), (sx, 4 * M), (sw, 4 * N), (b, es * N),
                      (y, M * N * es)):
            for at in (of, of + (m - 1) // 256 * 256, of - (n - 1) // 256 * 256):
                assert ia.lib().inf_gemm_i8(M, N, K, x, ld, sx, w, ld, sw, b, y, N, dt, at, n, None) == OVERLAP


def test_quantized_rows_over_their_scales():
    q = 20 * BIG
    for s in (q, q + 7 * 64 + 60, q - 28):
        assert ia.lib().inf_quantize_i8(21 * BIG, 64, 8, 64, 0, q, 64, s, 0, None) == OVERLAP


def test_results_beside_what_is_read():
    """Between y's rows there is room: not refused (6: the next check's, the workspace's)."""
    M, N, K, y = 100, 32, 64, 20 * BIG
    for dt, es in ((0, 4), (1, 2)):
        for place in ("w", "sw", "b"):
            for off in (es * N, es * N + 16):
                a = dict(w=21 * BIG, sw=22 * BIG, b=23 * BIG)
                a[place] = y + off
                kw = dict(w=K) if place == "w" else {}
                pitch = 4096
                n = 1 if place == "w" else N
                assert ia.lib().inf_linear_i8(M, n, K, 24 * BIG, K, a["w"], K, a["sw"], a["b"], y, pitch // es, dt, None,
                                              0, None) == 6
                a[place] = y + pitch - 64 if place == "w" else y + 3 * pitch - 4
                assert ia.lib().inf_linear_i8(M, N, K, 24 * BIG, K, a["w"], K, a["sw"], a["b"], y, pitch // es, dt,
                                              None, 0, None) == OVERLAP
