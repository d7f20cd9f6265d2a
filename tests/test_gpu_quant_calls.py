"""Calls of weights in 8 bits and a cache in 4 as programs make them: one workspace for rows that grow, results beside
what is read, two query heads a kv head, few rows of a vocabulary's width."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv4 import check, ia, make_cache  # noqa: E402,F401
from test_gpu_quant import check_product, rand_i8, ref_quantize  # noqa: E402

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


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M", [1, 4, 40, 200])
def test_linear_within_one_matrix(ia, M, dtype):
    """Input and result are columns of one matrix, bias and scales lie behind a row's end."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    K, N = 96, 100
    buf = torch.full((M, K + N + 60), 7.0, dtype=dtype, device="cuda")
    x = torch.randn((M, K), generator=gen, device="cuda").to(dtype)
    w, sw = ia.quantize_i8(torch.randn((K, N), generator=gen, device="cuda"), transpose=True)
    bias = torch.randn(N, generator=gen, device="cuda").to(dtype)
    want = ia.linear_i8(x, w, sw, bias=bias)
    for first in (True, False):  # the input before the result, and behind it
        buf.fill_(7.0)
        a, b = (buf[:, :K], buf[:, K:K + N]) if first else (buf[:, N:N + K], buf[:, :N])
        a.copy_(x)
        ia.linear_i8(a, w, sw, bias=bias, out=b)
        assert torch.equal(b, want) and torch.equal(a, x) and (buf[:, K + N:] == 7).all()
        if M > 1:
            with pytest.raises(ia.InfernoError):
                ia.linear_i8(a, w, sw, bias=bias, out=buf[:, 1:N + 1])
    q, s = ia.quantize_i8(x)
    rows = torch.full((M, 96 + 4 * N + 16), 9, dtype=torch.uint8, device="cuda")  # rows in 8 bits, the result's behind
    q2, y = rows[:, :K].view(torch.int8), rows[:, 96:96 + 4 * N].view(F32)
    q2.copy_(q)
    ia.gemm_i8(q2, s, w, sw, out=y)
    assert torch.equal(y, ia.gemm_i8(q, s, w, sw)) and torch.equal(q2, q) and (rows[:, 96 + 4 * N:] == 9).all()


class Arena:
    """Tensors one behind the other in one piece of memory."""

    def __init__(self, nbytes):
        self.data, self.at = torch.zeros(nbytes, dtype=torch.uint8, device="cuda"), 0

    def take(self, shape, dtype):
        n = torch.empty(shape, dtype=dtype, device="meta").nbytes
        t = self.data[self.at:self.at + n].view(dtype).view(shape)
        self.at += -(-n // 16) * 16
        return t


def in_one_arena(ia, cache, arena):
    """The same cache with a page's keys, their scales, values and theirs side by side, then its table and lengths."""
    pages, heads, P, half = cache.k.shape
    parts = [cache.k, cache.k_scale, cache.v, cache.v_scale]
    page = arena.take((pages, sum(t[0].numel() for t in parts)), torch.uint8)
    mine, at = [], 0
    for t in parts:
        n = t[0].numel()
        mine.append(page[:, at:at + n].unflatten(1, t.shape[1:]))
        mine[-1].copy_(t)
        at += n
    table, lens = arena.take(cache.table.shape, torch.int32), arena.take(cache.lens.shape, torch.int32)
    table.copy_(cache.table)
    lens.copy_(cache.lens)
    return ia.PagedKV4(mine[0], mine[2], mine[1], mine[3], table, lens)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_read_beside_the_cache(ia, D):
    """Cache and results in one piece of memory, keys and values beside each other."""
    gen = torch.Generator().manual_seed(D)
    cache, ks, vs, _ = make_cache(ia, gen, [9, 30], 2, D, 16)
    for dtype in (F32, BF16):
        arena = Arena(1 << 20)
        both = arena.take((2, 30, 2, 2, D), dtype)
        here = in_one_arena(ia, cache, arena)
        other = arena.take((2, 2, 30, 2, D), dtype)
        first = arena.take((2,), torch.int32)
        for k, v in ((both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)), (other[:, :, :, 0], other[:, :, :, 1])):
            ia.kv4_read(here, 30, first=first, k_out=k, v_out=v)
            assert torch.equal(k[1].cpu().double(), ks[1]) and torch.equal(v[1].cpu().double(), vs[1])
            assert torch.equal(v[0, :, :9].cpu().double(), vs[0]) and not k[0, :, 9:].any()
        with pytest.raises(ia.InfernoError):
            ia.kv4_read(here, 30, k_out=k, v_out=k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[40, 700], [0, 3001]])
def test_attention_beside_the_cache(ia, lens, dtype):
    """Queries, cache, workspace and results in one piece of memory; results in the queries' place, whole rows to the
    workgroups and in shares."""
    gen = torch.Generator().manual_seed(lens[1])
    cache, ks, vs, _ = make_cache(ia, gen, lens, 2, 64, 16)
    n = ia.attn_decode_kv4_workspace(cache, 6).nbytes
    assert bool(n) == (lens[1] > 1024)
    arena = Arena(n + (2 << 20))
    ws = arena.take((n,), torch.uint8)  # at the start: on 256 bytes
    both = arena.take((2, 12, 1, 64), dtype)
    here = in_one_arena(ia, cache, arena)
    q = torch.randn((2, 6, 1, 64), generator=gen).to(dtype)
    both[:, :6].copy_(q)
    ia.attn_decode_kv4(both[:, :6], here, out=both[:, 6:], workspace=ws)
    check(both[:, 6:], q, ks, vs, 2)
    want = both[:, 6:].clone()
    ia.attn_decode_kv4(both[:, :6], here, out=both[:, :6], workspace=ws)
    assert torch.equal(both[:, :6], want) and torch.equal(both[:, 6:], want)
    with pytest.raises(ia.InfernoError):
        ia.attn_decode_kv4(both[:, :6], here, out=both[:, 5:11], workspace=ws)


@pytest.mark.parametrize("D,layout", [(32, "heads"), (64, "slots"), (128, "joint")])
def test_append_beside_the_cache(ia, D, layout):
    """New keys and values, counts and cache in one piece of memory: what a cache of separate tensors holds."""
    gen = torch.Generator().manual_seed(D + 1)
    cache, _, _, _ = make_cache(ia, gen, [9, 30, 16], 2, D, 16, layout=layout)
    arena = Arena(1 << 20)
    qkv = arena.take((3, 7, 3, 2, D), F32)
    here = in_one_arena(ia, cache, arena)
    counts = arena.take((3,), torch.int32)
    qkv.copy_(torch.randn(qkv.shape, generator=gen))
    counts.copy_(torch.tensor([7, 0, 5], dtype=torch.int32))
    for c in (cache, here):
        ia.kv4_append(c, qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2), counts=counts)
    for a, b in ((cache.k, here.k), (cache.v, here.v), (cache.k_scale, here.k_scale), (cache.v_scale, here.v_scale)):
        assert torch.equal(a, b)
    with pytest.raises(ia.InfernoError):  # keys and values in one pool
        ia.kv4_append(ia.PagedKV4(here.k, here.k, here.k_scale, here.v_scale, here.table, here.lens),
                      qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_two_query_heads(ia, D, dtype):
    """Two query heads a kv head, whole rows to the workgroups and in shares."""
    gen = torch.Generator().manual_seed(D + 2)
    for lens in ([0, 1, 15, 16, 17, 255, 256, 257, 513, 1000], [3000, 0, 700, 1]):
        cache, ks, vs, _ = make_cache(ia, gen, lens, 3, D, 16)
        q = torch.randn((len(lens), 6, 1, D), generator=gen).to(dtype)
        check(ia.attn_decode_kv4(q.cuda(), cache), q, ks, vs, 3)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_read_on_8_bytes(ia, D):
    """bf16 results whose rows lie on 8 bytes only; what lies beside them stays."""
    gen = torch.Generator().manual_seed(D + 3)
    cache, ks, vs, _ = make_cache(ia, gen, [9, 0, 77], 2, D, 16)
    first = torch.tensor([2, 0, 1], dtype=torch.int32).cuda()
    store = torch.full((2, 3, 2, 80, D + 4), 5.0, dtype=BF16, device="cuda")
    k, v = store[0, ..., 4:], store[1, ..., :D]
    ia.kv4_read(cache, 80, first=first, k_out=k, v_out=v)
    for got, want in ((k, ks), (v, vs)):
        for r, n in enumerate([9, 0, 77]):
            f = int(first[r])
            m = max(n - f, 0)
            assert torch.equal(got[r, :, :m].cpu().double(), want[r][:, f:]) and not got[r, :, m:].any()
    assert (store[0, ..., :4] == 5).all() and (store[1, ..., D:] == 5).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 50257, 768), (2, 50257, 130), (17, 50257, 768), (33, 50257, 768), (64, 32000, 300),
                                   (1, 8200, 9000), (1, 700, 14336), (5, 300, 11008), (1, 28672, 1000)])
def test_few_rows_of_wide_layers(ia, M, N, K, dtype):
    """A vocabulary's projection and long inner layers at few tokens, past the few-row kernel's sizes."""
    gen = torch.Generator().manual_seed(M + N + K)
    x = torch.randn((M, K), generator=gen).to(dtype)
    w, dw = rand_i8(gen, N, K)
    sw = torch.rand(N, generator=gen) + 0.1
    bias = (torch.randn(N, generator=gen) * 1000).to(dtype)
    qx, sx = ref_quantize(x)
    y = ia.linear_i8(x.cuda(), dw, sw.cuda(), bias=bias.cuda())
    check_product(y, qx @ w.double().t(), sx, sw, bias, dtype)
    q, s = ia.quantize_i8(x.cuda())
    assert torch.equal(ia.gemm_i8(q, s, dw, sw.cuda(), bias=bias.cuda(), dtype=dtype), y)
