"""Weights in 8 bits and a cache in 4 without a GPU: workspace sizes and host-side argument checks of the C-ABI
(every call here carries an invalid argument, so it returns before any HIP call), and the torch helpers' checks of
dtypes, devices and layouts."""
import ctypes

import pytest

import inferno_amd as ia
from inferno_amd import PagedKV4Struct, Strides

FAKE = 0x10000  # never dereferenced: each call below fails validation first


def cache(**kw):
    heads, page, D = kw.get("heads", 2), kw.get("page_size", 16), kw.get("D", 64)
    s = Strides(heads * page * D // 2, page * D // 2, D // 2, 1)
    ss = Strides(heads * page * D // 32, page * D // 32, page, 1)
    a = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, sk=s, sv=s, sks=ss, svs=ss, table=FAKE, lens=FAKE,
             table_stride=4, rows=4, heads=heads, D=D, page_size=page, max_pages=4, n_pages=32)
    a.update(kw)
    return PagedKV4Struct(*(a[n] for n, _ in PagedKV4Struct._fields_))


NEW = Strides(8 * 2 * 64, 64, 2 * 64, 1)  # [rows, heads, T, D] out of [rows, T, heads, D]


def append(c, **kw):
    a = dict(k=FAKE, sk=NEW, v=FAKE, sv=NEW, T=8, dt=0)
    a.update(kw)
    return ia.lib().inf_kv4_append(ctypes.byref(c), a["k"], a["sk"], a["v"], a["sv"], None, a["T"], a["dt"], None)


def read(c, **kw):
    a = dict(k=FAKE, sk=NEW, v=FAKE, sv=NEW, T=8, dt=0)
    a.update(kw)
    return ia.lib().inf_kv4_read(ctypes.byref(c), None, a["T"], a["k"], a["sk"], a["v"], a["sv"], a["dt"], None)


def decode(c, **kw):
    a = dict(q=FAKE, sq=Strides(4 * 64, 64, 64, 1), o=FAKE, so=Strides(4 * 64, 64, 64, 1), hq=4, max_len=64,
             scale=0.125, dt=0, ws=None, n=0)
    a.update(kw)
    return ia.lib().inf_attn_decode_kv4(ctypes.byref(c), a["q"], a["sq"], a["o"], a["so"], a["hq"], a["max_len"],
                                        a["scale"], a["dt"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), 1), (dict(v=None), 1), (dict(k_scale=None), 1), (dict(v_scale=None), 1), (dict(table=None), 1),
    (dict(lens=None), 1),
    (dict(rows=0), 2), (dict(heads=0), 2), (dict(max_pages=0), 2), (dict(n_pages=0), 2), (dict(page_size=0), 2),
    (dict(rows=65536), 2), (dict(rows=60000, heads=300), 2),
    (dict(max_pages=1 << 20, page_size=2048, table_stride=1 << 20), 2),
    (dict(D=48), 5), (dict(D=256), 5), (dict(page_size=24), 5), (dict(page_size=8), 5),
    (dict(table_stride=3), 3),
    (dict(sk=Strides(1024, 512, 32, 2)), 3), (dict(svs=Strides(64, 32, -16, 1)), 3),
    (dict(sv=Strides(1024, 512, (1 << 22) + 16, 1)), 3), (dict(sks=Strides(64, 32, (1 << 22) + 4, 1)), 3),
    (dict(sk=Strides(1024, 512, 40, 1)), 7), (dict(svs=Strides(64, 34, 16, 1)), 7),
    (dict(k=FAKE + 8), 7), (dict(v_scale=FAKE + 2), 7), (dict(table=FAKE + 2), 7), (dict(lens=FAKE + 1), 7),
])
def test_bad_caches(kw, status):
    c = cache(**kw)
    assert append(c) == status
    assert read(c) == status
    assert decode(c, hq=2 * c.heads) == status


def test_null_arguments():
    n = ctypes.c_size_t(7)
    L = ia.lib()
    assert L.inf_kv4_append(None, FAKE, NEW, FAKE, NEW, None, 1, 0, None) == 1
    assert L.inf_kv4_read(None, None, 1, FAKE, NEW, FAKE, NEW, 0, None) == 1
    assert L.inf_attn_decode_kv4_workspace(None, 4, 64, ctypes.byref(n)) == 1 and n.value == 0
    assert L.inf_attn_decode_kv4_workspace(ctypes.byref(cache()), 4, 64, None) == 1
    assert L.inf_linear_i8_workspace(1, 1, 1, None) == 1 and L.inf_gemm_i8_workspace(1, 1, 1, None) == 1


@pytest.mark.parametrize("kw", [
    dict(sk=Strides(0, 512, 32, 1)), dict(sv=Strides(1024, 0, 32, 1)), dict(sk=Strides(1024, 512, 0, 1)),
    dict(sv=Strides(1024, 512, 16, 1)), dict(sks=Strides(0, 32, 16, 1)), dict(svs=Strides(64, 32, 8, 1)),
    dict(sks=Strides(64, 16, 16, 1))])
def test_written_pools_do_not_overlap_themselves(kw):
    assert append(cache(**kw)) == 3
    assert decode(cache(**kw), scale=0.0) == 8  # a cache that is only read may repeat itself


@pytest.mark.parametrize("call", [append, read])
@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), 2), (dict(k=None), 1), (dict(v=None), 1), (dict(T=0), 0), (dict(dt=2), 4), (dict(dt=9), 4),
    (dict(sk=Strides(1024, 64, 128, 2)), 3), (dict(sv=Strides(1024, 64, -128, 1)), 3),
    (dict(k=FAKE + 4), 7), (dict(sv=Strides(1024, 64, 130, 1)), 7), (dict(T=1 << 24), 2)])
def test_append_and_read_arguments(call, kw, status):
    if kw.get("T") == 1 << 24:  # views that do not overlap themselves
        s = Strides(1 << 40, 1 << 36, 64, 1)
        kw = dict(kw, sk=s, sv=s)
    assert call(cache(), **kw) == status


@pytest.mark.parametrize("s", [Strides(1024, 64, 64, 1), Strides(1024, 0, 128, 1), Strides(0, 64, 128, 1)])
def test_read_results_do_not_overlap_themselves(s):
    assert read(cache(), sk=s) == 3 and read(cache(), sv=s) == 3


@pytest.mark.parametrize("kw,status", [
    (dict(hq=0), 2), (dict(hq=3), 2), (dict(max_len=0), 2), (dict(max_len=65), 2), (dict(dt=3), 4),
    (dict(scale=0.0), 8), (dict(scale=-1.0), 8), (dict(scale=float("nan")), 8), (dict(scale=float("inf")), 8),
    (dict(q=None), 1), (dict(o=None), 1), (dict(q=FAKE + 4), 7), (dict(sq=Strides(256, 66, 64, 1)), 7),
    (dict(so=Strides(256, 0, 64, 1)), 3), (dict(so=Strides(0, 64, 64, 1)), 3)])
def test_decode_arguments(kw, status):
    assert decode(cache(), **kw) == status


def test_decode_workspace():
    n = ctypes.c_size_t()
    c = cache(rows=3, max_pages=1000, table_stride=1000, n_pages=3000)
    assert ia.lib().inf_attn_decode_kv4_workspace(ctypes.byref(c), 4, 16000, ctypes.byref(n)) == 0
    assert n.value > 0 and n.value % 256 == 0
    assert decode(c, max_len=16000, ws=None, n=n.value) == 6
    assert decode(c, max_len=16000, ws=FAKE, n=n.value - 1) == 6
    assert decode(c, max_len=16000, ws=FAKE + 16, n=n.value) == 7
    assert ia.lib().inf_attn_decode_kv4_workspace(ctypes.byref(cache()), 4, 64, ctypes.byref(n)) == 0 and n.value == 0


def test_decode_grids():
    """Sizes that no grid holds."""
    c = cache(rows=65535, heads=256, max_pages=64, table_stride=64, n_pages=1 << 20)
    assert decode(c, hq=512, max_len=64, ws=FAKE, n=1 << 62) == 2
    c = cache(rows=4096, heads=1, max_pages=4096, table_stride=4096, n_pages=1 << 20)
    assert decode(c, hq=8192, max_len=65536, ws=FAKE, n=1 << 62) == 2


def test_read_grids():
    s = Strides(32 << 24, 32, 32, 1)
    c = cache(rows=1, heads=1 << 24, D=32)
    assert read(c, T=1, sk=s, sv=s) == 2


def quantize(**kw):
    a = dict(x=FAKE, ldx=64, rows=8, cols=64, t=0, q=1 << 40, ldq=64, s=1 << 41, dt=0)
    a.update(kw)
    return ia.lib().inf_quantize_i8(a["x"], a["ldx"], a["rows"], a["cols"], a["t"], a["q"], a["ldq"], a["s"], a["dt"],
                                    None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 1), (dict(q=None), 1), (dict(s=None), 1), (dict(rows=-1), 2), (dict(cols=0), 2), (dict(rows=0), 0),
    (dict(rows=0, t=1), 2), (dict(rows=1 << 31), 2), (dict(cols=1 << 31, ldx=1 << 31), 2), (dict(rows=1 << 27), 2),
    (dict(rows=1 << 24, cols=1025, ldx=1025), 2), (dict(cols=1 << 28, ldx=1 << 28, t=1), 2),
    (dict(dt=2), 4), (dict(dt=-1), 4), (dict(ldx=63), 3), (dict(ldq=48), 3), (dict(t=1, rows=65, ldq=64), 3),
    (dict(ldq=(1 << 22) + 16), 3), (dict(ldq=72), 7), (dict(q=FAKE + 8), 7), (dict(x=FAKE + 2), 7),
    (dict(x=FAKE + 1, dt=1), 7), (dict(s=FAKE + 2), 7)])
def test_quantize_arguments(kw, status):
    assert quantize(**kw) == status


def gemm(**kw):
    a = dict(M=8, N=32, K=64, x=FAKE, ldx=64, sx=FAKE, w=FAKE, ldw=64, sw=FAKE, b=FAKE, y=1 << 40, ldy=32, dt=0, ws=None,
             n=0)
    a.update(kw)
    return ia.lib().inf_gemm_i8(a["M"], a["N"], a["K"], a["x"], a["ldx"], a["sx"], a["w"], a["ldw"], a["sw"], a["b"],
                                a["y"], a["ldy"], a["dt"], a["ws"], a["n"], None)


def linear(**kw):
    a = dict(M=8, N=32, K=64, x=FAKE, ldx=64, w=FAKE, ldw=64, sw=FAKE, b=FAKE, y=1 << 40, ldy=32, dt=0, ws=FAKE, n=1 << 40)
    a.update(kw)
    return ia.lib().inf_linear_i8(a["M"], a["N"], a["K"], a["x"], a["ldx"], a["w"], a["ldw"], a["sw"], a["b"], a["y"],
                                  a["ldy"], a["dt"], a["ws"], a["n"], None)


@pytest.mark.parametrize("call", [gemm, linear])
@pytest.mark.parametrize("kw,status", [
    (dict(M=0), 2), (dict(N=0), 2), (dict(K=0), 2), (dict(M=1 << 31), 2), (dict(N=1 << 31), 2),
    (dict(M=1 << 20, N=1 << 20), 2), (dict(M=1 << 27, N=1, K=1), 2), (dict(K=1 << 17, ldx=1 << 17, ldw=1 << 17), 5), (dict(dt=2), 4),
    (dict(x=None), 1), (dict(w=None), 1), (dict(sw=None), 1), (dict(y=None), 1),
    (dict(ldx=63), 3), (dict(ldw=48), 3), (dict(ldw=(1 << 22) + 16), 3), (dict(ldy=31), 3),
    (dict(ldw=72), 7), (dict(w=FAKE + 4), 7), (dict(sw=FAKE + 1), 7), (dict(y=FAKE + 2), 7), (dict(b=FAKE + 2), 7)])
def test_product_arguments(call, kw, status):
    assert call(**kw) == status


def test_results_over_what_is_read():
    far = 0x10000000
    for kw in (dict(w=far), dict(w=far - 31 * 64 - 48), dict(sw=far + 900), dict(b=far - 64)):
        assert gemm(y=far, **kw) == 3 and linear(y=far, **kw) == 3
    assert gemm(y=far, x=far + 1008) == 3 and gemm(y=far, sx=far - 28) == 3
    assert linear(y=far, x=far + 992) == 3 and linear(M=100, y=far, ws=far + 512) == 3
    assert quantize(q=FAKE + 2032) == 3 and quantize(s=FAKE - 28) == 3 and quantize(s=FAKE + 2044, t=1) == 3


def test_rows_that_no_grid_holds():
    assert linear(M=1 << 24, N=1, K=1040, ldx=1040, ldw=1040) == 2


def test_product_arguments_of_one_form():
    assert gemm(sx=None) == 1 and gemm(sx=FAKE + 2) == 7
    assert gemm(x=FAKE + 4) == 7 and gemm(ldx=72) == 7  # 8-bit rows
    assert linear(x=FAKE + 2) == 7
    n = ctypes.c_size_t()
    for M, N, K in ((1, 2304, 768), (300, 500, 4096), (5000, 5000, 100)):
        args = dict(M=M, N=N, K=K, ldx=K + 12, ldw=-(-K // 16) * 16, ldy=N)
        assert ia.lib().inf_linear_i8_workspace(M, N, K, ctypes.byref(n)) == 0 and n.value % 256 == 0
        assert n.value >= M * K + 4 * M or (M == 1 and n.value == 0)  # one row needs none
        if not n.value:
            continue
        assert linear(**args, ws=None, n=n.value) == 6
        assert linear(**args, ws=FAKE, n=n.value - 1) == 6
        assert linear(**args, ws=FAKE + 16, n=n.value) == 7
    assert ia.lib().inf_gemm_i8_workspace(300, 500, 4096, ctypes.byref(n)) == 0
    if n.value:
        args = dict(M=300, N=500, K=4096, ldx=4096, ldw=4096, ldy=500)
        assert gemm(**args, ws=FAKE, n=n.value - 1) == 6 and gemm(**args, ws=FAKE + 16, n=n.value) == 7
    assert ia.lib().inf_linear_i8_workspace(0, 1, 1, ctypes.byref(n)) == 2 and n.value == 0


# ---- the torch helpers: what the C-ABI cannot see


torch = pytest.importorskip("torch")


def test_helpers_refuse_the_cpu():
    x, w = torch.zeros(4, 64), torch.zeros(8, 64, dtype=torch.int8)
    with pytest.raises(ValueError):
        ia.quantize_i8(x)
    with pytest.raises(ValueError):
        ia.linear_i8(x, w, torch.ones(8))
    with pytest.raises(ValueError):
        ia.gemm_i8(w, torch.ones(8), w, torch.ones(8))
    c = pool()
    with pytest.raises(ValueError):
        ia.kv4_append(c, torch.zeros(2, 1, 1, 64), torch.zeros(2, 1, 1, 64))
    with pytest.raises(ValueError):
        ia.kv4_read(c, 4)
    with pytest.raises(ValueError):
        ia.attn_decode_kv4(torch.zeros(2, 1, 1, 64), c)


def pool(**kw):
    a = dict(k=torch.zeros((4, 1, 16, 32), dtype=torch.uint8), v=torch.zeros((4, 1, 16, 32), dtype=torch.uint8),
             k_scale=torch.zeros((4, 1, 2, 16), dtype=torch.uint8), v_scale=torch.zeros((4, 1, 2, 16), dtype=torch.uint8),
             table=torch.zeros((2, 2), dtype=torch.int32), lens=torch.zeros(2, dtype=torch.int32))
    a.update(kw)
    return ia.PagedKV4(**a)


@pytest.mark.parametrize("kw,error", [
    (dict(k=torch.zeros((4, 1, 16, 64), dtype=torch.uint8)), ValueError),
    (dict(k_scale=torch.zeros((4, 1, 16, 2), dtype=torch.uint8)), ValueError),
    (dict(v=torch.zeros((4, 1, 16, 32), dtype=torch.int8)), TypeError),
    (dict(v_scale=torch.zeros((4, 1, 2, 16))), TypeError),
    (dict(table=torch.zeros((3, 2), dtype=torch.int32)), ValueError),
    (dict(table=torch.zeros((2, 2))), TypeError), (dict(lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(table=torch.zeros((2, 4), dtype=torch.int32)[:, ::2]), ValueError),
    (dict(lens=torch.zeros(4, dtype=torch.int32)[::2]), ValueError)])
def test_cache_handles(kw, error):
    with pytest.raises(error):
        pool(**kw)
    c = pool()
    with pytest.raises(ValueError):
        c.table = torch.zeros((2, 3), dtype=torch.int32)
    with pytest.raises(TypeError):
        c.lens = torch.zeros(2)
    with pytest.raises(ValueError):
        ia.PagedKV4.empty(4, 1, 16, 48, c.table, c.lens)


def test_helpers_refuse():
    c, x = pool(), torch.zeros(2, 1, 3, 64)
    for k, v in ((x, x.bfloat16()), (x[:1], x[:1]), (x, x[:, :, :2]), (x[..., :32], x[..., :32])):
        with pytest.raises(ValueError):
            ia.kv4_append(c, k, v)
    with pytest.raises(TypeError):
        ia.kv4_append(c, x.half(), x.half())
    with pytest.raises(TypeError):
        ia.kv4_append(c, x, x, counts=torch.zeros(2))
    with pytest.raises(TypeError):
        ia.kv4_read(c, 3, dtype=torch.float16)
    with pytest.raises(ValueError):
        ia.kv4_read(c, 3, k_out=x)
    with pytest.raises(ValueError):
        ia.kv4_read(c, 4, k_out=x, v_out=x)
    with pytest.raises(TypeError):
        ia.attn_decode_kv4(torch.zeros(2, 1, 1, 64, dtype=torch.float16), c)
    with pytest.raises(ValueError):
        ia.attn_decode_kv4(torch.zeros(2, 1, 2, 64), c)
    a, w, s = torch.zeros(4, 64), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)
    with pytest.raises(TypeError):
        ia.quantize_i8(a.half())
    with pytest.raises(ValueError):
        ia.quantize_i8(a[:, ::2])
    with pytest.raises(TypeError):
        ia.linear_i8(a, w.float(), s)
    with pytest.raises(ValueError):
        ia.linear_i8(a[:, :32], w, s)
    with pytest.raises(ValueError):
        ia.linear_i8(a, w, s[:4])
    with pytest.raises(TypeError):
        ia.linear_i8(a.bfloat16(), w, s, bias=s)
    with pytest.raises(ValueError):
        ia.linear_i8(a, w, s, out=torch.zeros(4, 9))
    with pytest.raises(TypeError):
        ia.gemm_i8(w, s, w, s, dtype=torch.float16)
    with pytest.raises(ValueError):
        ia.gemm_i8(w, s[:4], w, s)
