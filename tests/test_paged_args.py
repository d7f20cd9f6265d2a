"""Generation from a paged cache without a GPU: workspace sizes and host-side argument checks of
the C-ABI (every call here carries an invalid argument, so it returns before any HIP call), and
the torch helpers' checks of dtypes, devices and layouts."""
import ctypes

import pytest

import inferno_amd as ia
from inferno_amd import PagedKVStruct, Strides

FAKE = 0x10000  # never dereferenced: each call below fails validation first


def cache(**kw):
    heads, page, D = kw.get("heads", 2), kw.get("page_size", 16), kw.get("D", 64)
    s = Strides(heads * page * D, page * D, D, 1)
    a = dict(k=FAKE, v=FAKE, sk=s, sv=s, table=FAKE, lens=FAKE, table_stride=4, rows=4, heads=heads, D=D,
             page_size=page, max_pages=4, n_pages=32, dt=ia.INF_F32)
    a.update(kw)
    return PagedKVStruct(*(a[n] for n, _ in PagedKVStruct._fields_))


BAD_CACHE = [
    (dict(k=None), 1), (dict(v=None), 1), (dict(table=None), 1), (dict(lens=None), 1),
    (dict(rows=0), 2), (dict(heads=0), 2), (dict(max_pages=0), 2), (dict(n_pages=0), 2), (dict(page_size=0), 2),
    (dict(rows=65536), 2), (dict(rows=60000, heads=300), 2),
    (dict(max_pages=1 << 20, page_size=2048, table_stride=1 << 20), 2),  # more than 2^30 positions
    (dict(D=48), 5), (dict(D=256), 5), (dict(page_size=24), 5),
    (dict(dt=ia.INF_F64), 4), (dict(dt=7), 4),
    (dict(table_stride=3), 3),
    (dict(sk=Strides(2048, 1024, 64, 2)), 3), (dict(sv=Strides(-2048, 1024, 64, 1)), 3),
    (dict(sk=Strides(2048, 1024, (1 << 22) + 4, 1)), 3),
    (dict(sk=Strides(2048, 1024, 66, 1)), 7),
    (dict(k=FAKE + 8), 7),
    (dict(dt=ia.INF_BF16, sk=Strides(2048, 1024, 68, 1)), 7),   # 8-byte rows: the cache needs 16
    (dict(table=FAKE + 2), 7), (dict(lens=FAKE + 1), 7),
]
NEW = Strides(8 * 2 * 64, 64, 2 * 64, 1)


def append(c, **kw):
    a = dict(k=FAKE, sk=NEW, v=FAKE, sv=NEW, T=8)
    a.update(kw)
    return ia.lib().inf_kv_append(ctypes.byref(c), a["k"], a["sk"], a["v"], a["sv"], None, a["T"], None, None, None,
                                  None)


def decode(c, **kw):
    a = dict(q=FAKE, sq=Strides(4 * 64, 64, 64, 1), o=FAKE, so=Strides(4 * 64, 64, 64, 1), hq=4, max_len=64,
             scale=0.125, w_in=None, w_out=None, ws=None, n=0)
    a.update(kw)
    return ia.lib().inf_attn_decode_paged(ctypes.byref(c), a["q"], a["sq"], a["o"], a["so"], a["hq"], a["max_len"],
                                          a["scale"], a["w_in"], a["w_out"], a["ws"], a["n"], None)


def evict(c, **kw):
    a = dict(w=FAKE, wo=FAKE, p=FAKE, po=FAKE, lo=FAKE, keep=16, recent=4, max_len=64, ws=FAKE, n=1 << 20)
    a.update(kw)
    return ia.lib().inf_kv_evict(ctypes.byref(c), a["w"], a["wo"], a["p"], a["po"], a["lo"], a["keep"], a["recent"],
                                 a["max_len"], a["ws"], a["n"], None)


def reorder(c, **kw):
    a = dict(layers=1, kl=0, vl=0, parents=FAKE, beams=2, out=FAKE + 4096, stride=4, spare=FAKE, spare_out=FAKE + 256)
    a.update(kw)
    return ia.lib().inf_beam_reorder(ctypes.byref(c), a["layers"], a["kl"], a["vl"], a["parents"], a["beams"], a["out"],
                                     a["stride"], a["spare"], a["spare_out"], None)


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_bad_caches(kw, status):
    c = cache(**kw)
    assert append(c) == status
    assert decode(c, hq=2 * c.heads) == status
    assert evict(c) == status
    assert reorder(c) == status


def test_null_cache():
    n = ctypes.c_size_t(7)
    L = ia.lib()
    assert L.inf_kv_append(None, FAKE, NEW, FAKE, NEW, None, 1, None, None, None, None) == 1
    assert L.inf_attn_decode_paged_workspace(None, 4, 64, 0, ctypes.byref(n)) == 1 and n.value == 0
    assert L.inf_attn_decode_paged_workspace(ctypes.byref(cache()), 4, 64, 0, None) == 1
    assert L.inf_kv_evict_workspace(None, 4, 64, ctypes.byref(n)) == 1


@pytest.mark.parametrize("view", ["sk", "sv"])
@pytest.mark.parametrize("s", [Strides(0, 1024, 64, 1), Strides(2048, 0, 64, 1), Strides(2048, 1024, 0, 1),
                               Strides(2048, 1024, 32, 1), Strides(1024, 1024, 64, 1)])
def test_written_pools_do_not_overlap_themselves(view, s):
    c = cache(**{view: s})
    assert append(c) == 3 and evict(c) == 3 and reorder(c) == 3
    assert decode(c, scale=0.0) == 8  # a cache that is only read may repeat itself


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), 2), (dict(k=None), 1), (dict(v=None), 1), (dict(T=0), 0),
    (dict(sk=Strides(1024, 64, 128, 2)), 3), (dict(sv=Strides(1024, 64, -128, 1)), 3),
    (dict(k=FAKE + 4), 7), (dict(sv=Strides(1024, 64, 130, 1)), 7), (dict(T=1 << 24), 2),
])
def test_append_arguments(kw, status):
    assert append(cache(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(hq=0), 2), (dict(hq=3), 2), (dict(max_len=0), 2), (dict(max_len=65), 2),
    (dict(scale=0.0), 8), (dict(scale=-1.0), 8), (dict(scale=float("nan")), 8), (dict(scale=float("inf")), 8),
    (dict(q=None), 1), (dict(o=None), 1), (dict(q=FAKE + 4), 7), (dict(sq=Strides(256, 66, 64, 1)), 7),
    (dict(so=Strides(256, 0, 64, 1)), 3), (dict(so=Strides(0, 64, 64, 1)), 3),
    (dict(w_in=FAKE), 1),                                   # nowhere to write the sums
    (dict(w_out=FAKE), 6), (dict(w_out=FAKE, ws=FAKE, n=256), 6), (dict(w_out=FAKE, ws=FAKE + 128, n=1 << 20), 7),
])
def test_decode_arguments(kw, status):
    assert decode(cache(), **kw) == status


def test_outputs_that_overlap_the_inputs_in_part():
    c = cache()
    whole = 4 * 2 * 64 * 4  # rows, heads, capacity, bytes
    for off in (4, 64, whole - 4, -whole + 4):
        assert evict(c, wo=FAKE + off) == 3 and evict(c, po=FAKE + off) == 3
        assert decode(c, w_in=FAKE, w_out=FAKE + off, ws=FAKE, n=1 << 30) == 3
    assert evict(c, wo=FAKE + whole, n=0) == 6  # behind them: the next check's


def test_decode_workspace():
    L, n = ia.lib(), ctypes.c_size_t(0)

    def need(c, hq, max_len, w):
        assert L.inf_attn_decode_paged_workspace(ctypes.byref(c), hq, max_len, w, ctypes.byref(n)) == 0
        return n.value

    assert need(cache(), 4, 64, 0) == 0                     # one split
    with_scores = need(cache(), 4, 64, 1)
    assert with_scores >= 4 * 4 * (66 + 64) * 4 and with_scores % 256 == 0
    long = cache(max_pages=8192, table_stride=8192, rows=1)
    split = need(long, 2, 131072, 0)
    assert split >= 2 * 2 * 66 * 4 and split % 256 == 0
    assert decode(long, hq=2, max_len=131072) == 6
    assert decode(long, hq=2, max_len=131072, ws=FAKE, n=split - 256) == 6
    assert decode(long, hq=2, max_len=131072, ws=FAKE + 16, n=split) == 7
    for bad in (dict(hq=3), dict(max_len=0), dict(max_len=131073)):
        a = dict(dict(hq=2, max_len=64), **bad)
        assert L.inf_attn_decode_paged_workspace(ctypes.byref(long), a["hq"], a["max_len"], 0, ctypes.byref(n)) == 2


@pytest.mark.parametrize("kw,status", [
    (dict(keep=0), 2), (dict(recent=-1), 2), (dict(recent=17), 2), (dict(max_len=0), 2), (dict(max_len=65), 2),
    (dict(w=None), 1), (dict(wo=None), 1), (dict(p=None), 1), (dict(po=None), 1), (dict(lo=None), 1),
    (dict(ws=None), 6), (dict(n=64), 6), (dict(ws=FAKE + 2), 7),
])
def test_evict_arguments(kw, status):
    assert evict(cache(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(layers=0), 2), (dict(beams=0), 2), (dict(beams=3), 2),       # 4 rows
    (dict(parents=None), 1), (dict(out=None), 1), (dict(spare=None), 1), (dict(spare_out=None), 1),
    (dict(spare_out=FAKE), 3), (dict(spare_out=FAKE + 12), 3), (dict(spare_out=FAKE - 12), 3),  # over the spare pages
    (dict(stride=3), 3), (dict(out=FAKE), 3), (dict(out=FAKE + 60), 3), (dict(out=FAKE - 60), 3),  # over the table
    (dict(layers=2, kl=2048 * 32, vl=-4), 3), (dict(layers=2, kl=2048 * 32 + 2, vl=2048 * 32), 7),
    (dict(layers=2, kl=2048, vl=2048 * 32), 3),                        # layers on one another
])
def test_reorder_arguments(kw, status):
    assert reorder(cache(), **kw) == status


def select(**kw):
    a = dict(logits=FAKE, ld=100, scores=FAKE, fin=None, groups=2, beams=4, vocab=100, eos=-1, tok=FAKE, par=FAKE,
             out=FAKE, fo=None, dt=ia.INF_F32, ws=FAKE, n=1 << 20)
    a.update(kw)
    return ia.lib().inf_beam_select(a["logits"], a["ld"], a["scores"], a["fin"], a["groups"], a["beams"], a["vocab"],
                                    a["eos"], a["tok"], a["par"], a["out"], a["fo"], a["dt"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(dt=ia.INF_F64), 4), (dict(groups=0), 2), (dict(beams=0), 2), (dict(vocab=0), 2), (dict(beams=33), 5),
    (dict(vocab=1 << 31), 2), (dict(groups=1 << 25), 2), (dict(logits=None), 1), (dict(scores=None), 1),
    (dict(tok=None), 1), (dict(par=None), 1), (dict(out=None), 1), (dict(eos=100), 2),
    (dict(fin=FAKE), 2),                                   # finished beams need the token that ends them
    (dict(ld=99), 3), (dict(logits=FAKE + 2), 7), (dict(ws=None), 6), (dict(n=64), 6), (dict(ws=FAKE + 8), 7),
])
def test_select_arguments(kw, status):
    assert select(**kw) == status


# ---- the torch helpers -----------------------------------------------------------------------------
torch = pytest.importorskip("torch")


def pools(pages=8, heads=2, page=16, D=64, dtype=torch.float32):
    return (torch.zeros(pages, heads, page, D, dtype=dtype), torch.zeros(pages, heads, page, D, dtype=dtype),
            torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_handle_checks():
    k, v, table, lens = pools()
    c = ia.PagedKV(k, v, table, lens)
    assert (c.rows, c.heads, c.D, c.page_size, c.capacity, c.layers) == (3, 2, 64, 16, 32, 1)
    with pytest.raises(ValueError):
        ia.PagedKV(k, v[:4], table, lens)
    with pytest.raises(TypeError):
        ia.PagedKV(k, v.bfloat16(), table, lens)
    with pytest.raises(TypeError):
        ia.PagedKV(k, v, table.long(), lens)
    with pytest.raises(TypeError):
        ia.PagedKV(k, v, table, lens.float())
    with pytest.raises(ValueError):
        ia.PagedKV(k, v, table, lens[:2])
    with pytest.raises(ValueError):
        ia.PagedKV(k, v, table.t().contiguous().t(), lens)
    with pytest.raises(ValueError):
        c.table = table[:2]
    with pytest.raises(TypeError):
        c.lens = lens.long()
    with pytest.raises(ValueError):
        c.layer(0)
    wide = torch.zeros(3, 5, dtype=torch.int32)[:, 1:3]
    c.table = wide
    assert c.struct.table == wide.data_ptr() and c.struct.table_stride == 5


def test_helpers_refuse_what_the_abi_cannot_see():
    k, v, table, lens = pools()
    c = ia.PagedKV(k, v, table, lens)
    new = torch.zeros(3, 2, 1, 64)
    with pytest.raises(ValueError):
        ia.kv_append(c, new[:, :1], new[:, :1])
    with pytest.raises(TypeError):
        ia.kv_append(c, new.bfloat16(), new.bfloat16())
    with pytest.raises(ValueError):
        ia.attn_decode_paged(torch.zeros(3, 4, 2, 64), c)
    with pytest.raises(ValueError):
        ia.attn_decode_paged(torch.zeros(3, 4, 1, 64, dtype=torch.bfloat16), c)
    with pytest.raises(ValueError):
        ia.attn_decode_paged(torch.zeros(3, 4, 1, 64), c, weights=torch.zeros(3, 2, 32))
    with pytest.raises(ValueError):
        ia.attn_decode_paged(torch.zeros(3, 4, 1, 64), c, weights_out=torch.zeros(3, 2, 31))
    with pytest.raises(ValueError):
        ia.beam_select(torch.zeros(6, 10), torch.zeros(2, 2))
    with pytest.raises(TypeError):
        ia.beam_select(torch.zeros(4, 10, dtype=torch.float16), torch.zeros(2, 2))
    with pytest.raises(ValueError):
        ia.beam_select(torch.zeros(4, 10), torch.zeros(2, 2), finished=torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(TypeError):
        ia.beam_select(torch.zeros(4, 10), torch.zeros(2, 2, dtype=torch.float64))
    with pytest.raises(ValueError):
        ia.beam_reorder(c, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def test_helpers_refuse_host_tensors():
    k, v, table, lens = pools()
    c = ia.PagedKV(k, v, table, lens)
    new, meta, pos = torch.zeros(3, 2, 1, 64), torch.zeros(3, 2, 32), torch.zeros(3, 2, 32, dtype=torch.int32)
    for call in (lambda: ia.kv_append(c, new, new), lambda: ia.attn_decode_paged(new, c),
                 lambda: ia.kv_evict(c, meta, pos, 4), lambda: ia.beam_select(torch.zeros(4, 10), torch.zeros(2, 2)),
                 lambda: ia.beam_reorder(c, torch.zeros(1, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError, match="GPU"):
            call()
