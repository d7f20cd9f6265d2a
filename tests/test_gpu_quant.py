"""Matrices in 8 bits on the GPU against plain implementations in 64 bits on the CPU: rows and columns
quantised, products of every plan, the linear layer made of both.

What is quantised has to be equal: scales are one fp32 product, the quotient is rounded as if it were exact.
A product's sum is exact; it is rounded to fp32 (2^-24), multiplied by two scales (2^-24 each, the second
with the bias added in one rounding) and rounded to its type: 3 2^-24 of the product without the bias, and 2^-24 or 2^-8 of
the result.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INV127 = torch.tensor(np.float32(1.0) / np.float32(127.0))
TINY = 2.0**-126


@pytest.fixture(scope="module")
def ia():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import inferno_amd

    inferno_amd.lib()
    return inferno_amd


def ref_quantize(x):
    """(q in 64 bits, scale) of the rows of a CPU matrix."""
    x = x.float()
    top = x.abs().amax(1)
    scale = top * INV127
    bad = ~torch.isfinite(x).all(1)
    none = bad | (scale < TINY)
    s = torch.where(none, torch.ones(()), scale).double()
    q = torch.round(x.double() / s[:, None]).clamp(-127, 127)  # 53 bits: on the right side of every middle
    q[none] = 0
    scale = torch.where(scale < TINY, torch.zeros(()), scale)
    return q, torch.where(bad, torch.full((), float("nan")), scale)


def check_quantized(q, scale, x):
    rq, rs = ref_quantize(x)
    assert torch.equal(scale.cpu(), rs) or torch.equal(scale.cpu().nan_to_num(nan=-1.0), rs.nan_to_num(nan=-1.0))
    assert torch.equal(q.cpu().double(), rq)


SHAPES = [(1, 1), (3, 15), (5, 16), (7, 17), (2, 511), (9, 512), (3, 513), (4, 1024), (5, 1025), (2, 2048), (3, 2049),
          (2, 4104), (1, 8192), (3, 9001), (2, 20000), (1025, 5), (1026, 500), (1027, 1024), (1024, 1025), (1100, 2048),
          (1023, 700)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rows(ia, rows, cols, dtype):
    gen = torch.Generator().manual_seed(rows * 10007 + cols)
    x = (torch.randn((rows, cols), generator=gen) * torch.exp(2 * torch.randn((rows, 1), generator=gen))).to(dtype)
    q, s = ia.quantize_i8(x.cuda())
    assert q.shape == (rows, cols) and q.stride(0) % 16 == 0
    check_quantized(q, s, x)
    # what lies between a row's end and whole 16 bytes is zeros
    padded = torch.as_strided(q, (rows, q.stride(0)), (q.stride(0), 1))
    assert not padded[:, cols:].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (15, 31), (16, 32), (17, 33), (511, 64), (513, 65), (1030, 100)])
def test_columns(ia, rows, cols, dtype):
    gen = torch.Generator().manual_seed(rows * 10007 + cols)
    x = torch.randn((rows, cols), generator=gen).to(dtype)
    q, s = ia.quantize_i8(x.cuda(), transpose=True)
    assert q.shape == (cols, rows)
    check_quantized(q, s, x.t().contiguous())
    padded = torch.as_strided(q, (cols, q.stride(0)), (q.stride(0), 1))
    assert not padded[:, rows:].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ld,off", [(100, 0), (101, 0), (100, 1), (104, 4)])
def test_strided_rows(ia, ld, off, dtype):
    gen = torch.Generator().manual_seed(ld + off)
    store = torch.randn(20 * ld + off, generator=gen).to(dtype)
    x = torch.as_strided(store, (20, 97), (ld, 1), off)
    dev = torch.as_strided(store.cuda(), (20, 97), (ld, 1), off)
    check_quantized(*ia.quantize_i8(dev), x)
    check_quantized(*ia.quantize_i8(dev, transpose=True), x.t().contiguous())


def special_rows(dtype):
    """Middles between whole numbers, zeros, non-finite rows, the ends of the range."""
    k = torch.arange(-126, 127, dtype=torch.float64)
    rows = [torch.cat((k + 0.5, torch.tensor([127.0])))]
    # multiples of half a scale that is a power of two (bf16 holds them), and next to them
    scale = (torch.tensor(4.0) * INV127).double()  # of rows whose largest is 4
    mid = ((k + 0.5) * scale).float()
    rows += [torch.cat((mid, torch.tensor([4.0]))).double(),
             torch.cat((torch.nextafter(mid, torch.tensor(9.0)), torch.tensor([4.0]))).double(),
             torch.cat((torch.nextafter(mid, torch.tensor(-9.0)), torch.tensor([4.0]))).double()]
    n = rows[0].numel()
    rows.append(torch.zeros(n, dtype=torch.float64))
    for special in (float("inf"), -float("inf"), float("nan")):
        r = torch.linspace(-3, 3, n, dtype=torch.float64)
        r[n // 2] = special
        rows.append(r)
    ramp = torch.linspace(-1, 1, n, dtype=torch.float64)
    # 127 2^-126 / 2 and 2 times it; the largest; subnormals alone
    rows += [ramp * 63 * TINY, ramp * 255 * TINY, ramp * 3.3e38, ramp * 1e-40]
    return torch.stack(rows).float().to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("wide", [1, 9, 40])
def test_special_rows(ia, wide, dtype):
    x = special_rows(dtype).repeat(1, wide)
    check_quantized(*ia.quantize_i8(x.cuda()), x)
    check_quantized(*ia.quantize_i8(x.t().contiguous().cuda(), transpose=True), x)


def rand_i8(gen, rows, cols, junk=True):
    """int8 [rows, cols] on the GPU, rows on 16 bytes, anything behind their ends."""
    ld = -(-cols // 16) * 16
    store = torch.randint(-128, 128, (rows, ld), generator=gen, dtype=torch.int8)
    return store[:, :cols], store.cuda()[:, :cols]


def check_product(y, acc, sx, sw, bias, dtype):
    p = acc.double() * sx.double()[:, None] * sw.double()
    want = p if bias is None else p + bias.double()
    half = 2.0**-24 if dtype == F32 else 2.0**-8
    bound = 3.01 * 2.0**-24 * p.abs() + 1.01 * half * want.abs() + 2.0**-140
    err = (y.cpu().double() - want).abs()
    assert (err <= bound).all(), (err / bound).max()  # NaN fails


# few rows and few outputs: K ranges per wave; else tiles of 64, 128 or 256, those of 64 in K ranges where there are few
PRODUCTS = [(40, 50, 8192), (8, 64, 8200), (64, 40, 5000), (50, 8300, 130), (20, 9000, 2100), (100, 100, 3000),
            (700, 1100, 2050), (2100, 2200, 70), (1, 1, 1), (1, 16, 16), (2, 17, 33), (15, 100, 63), (16, 64, 64), (17, 48, 65), (31, 200, 129),
            (33, 130, 257), (48, 96, 1000), (64, 33, 500), (65, 127, 127), (100, 129, 1), (128, 128, 128),
            (129, 257, 300), (200, 130, 2000), (300, 515, 4090), (130, 100, 9000), (513, 70, 200), (70, 1030, 384)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_products(ia, M, N, K, dtype):
    gen = torch.Generator().manual_seed(M * 7 + N * 3 + K)
    x, dx = rand_i8(gen, M, K)
    w, dw = rand_i8(gen, N, K)
    sx, sw = torch.rand(M, generator=gen) + 0.1, torch.rand(N, generator=gen) + 0.1
    bias = (torch.randn(N, generator=gen) * 1000).to(dtype) if (M + N) % 2 else None
    y = ia.gemm_i8(dx, sx.cuda(), dw, sw.cuda(), bias=None if bias is None else bias.cuda(), dtype=dtype)
    check_product(y, x.double() @ w.double().t(), sx, sw, bias, dtype)


@pytest.mark.parametrize("M,N,K", [(3500, 3600, 333), (4096, 3328, 256), (257, 52000, 130)])
def test_large_products(ia, M, N, K):
    gen = torch.Generator().manual_seed(M)
    x, dx = rand_i8(gen, M, K)
    w, dw = rand_i8(gen, N, K)
    sx, sw = torch.rand(M, generator=gen) + 0.1, torch.rand(N, generator=gen) + 0.1
    y = ia.gemm_i8(dx, sx.cuda(), dw, sw.cuda(), dtype=BF16)
    check_product(y, (x.float() @ w.float().t()).double(), sx, sw, None, BF16)  # sums below 2^24: exact


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(3600, 3500, 2050), (3841, 4000, 530), (3842, 4094, 2300), (1660, 2040, 400),
                                   (1500, 2000, 3110), (2000, 2040, 3240)])
def test_large_tiles(ia, M, N, K, dtype):
    """Tiles of 256 with K long and short, and few of 128; sums below 2^24: exact in fp32."""
    gen = torch.Generator().manual_seed(M)
    (x, dx), (w, dw) = ((t[:, :K], t.cuda()[:, :K]) for t in (
        torch.randint(-70, 71, (n, -(-K // 16) * 16), generator=gen, dtype=torch.int8) for n in (M, N)))
    sx, sw = torch.rand(M, generator=gen) + 0.1, torch.rand(N, generator=gen) + 0.1
    bias = (torch.randn(N, generator=gen) * 1000).to(dtype)
    y = ia.gemm_i8(dx, sx.cuda(), dw, sw.cuda(), bias=bias.cuda(), dtype=dtype)
    check_product(y, (x.float() @ w.float().t()).double(), sx, sw, bias, dtype)


def test_largest_sums(ia):
    """-128 squared, 2^17 - 1 times."""
    K = (1 << 17) - 1
    for M in (1, 70):
        x = torch.full((M, K + 1), -128, dtype=torch.int8, device="cuda")
        w = torch.full((5, K + 1), -128, dtype=torch.int8, device="cuda")
        one = torch.ones(M, device="cuda")
        y = ia.gemm_i8(x[:, :K], one, w[:, :K], one[:1].expand(5).contiguous())
        assert (y.cpu().double() == float(np.float32(16384.0 * K))).all()


def test_strided_products(ia):
    """Rows of y further apart, at odd places, scales and bias on 4 bytes only: what lies beside stays."""
    gen = torch.Generator().manual_seed(5)
    for M, N, K in ((9, 50, 100), (90, 150, 700), (1, 64, 64)):
        x, dx = rand_i8(gen, M, K)
        w, dw = rand_i8(gen, N, K)
        sx, sw = torch.rand(M, generator=gen) + 0.1, torch.rand(N + 1, generator=gen) + 0.1
        bias = torch.randn(N + 1, generator=gen)
        for ld, off in ((N, 0), (N + 3, 1), (N + 6, 2)):
            store = torch.full((M * ld + off + 9,), 77.0, device="cuda")
            out = torch.as_strided(store, (M, N), (ld, 1), off)
            ia.gemm_i8(dx, sx.cuda(), dw, sw.cuda()[1:], bias=bias.cuda()[1:], out=out)
            check_product(out, x.double() @ w.double().t(), sx, sw[1:], bias[1:], F32)
            rest = store.clone()
            torch.as_strided(rest, (M, N), (ld, 1), off).fill_(77.0)
            assert (rest == 77.0).all()


# one kernel takes x as it is for one row, and for few short ones
LINEARS = [(1, 2304, 768), (1, 100, 65), (1, 50, 16384), (1, 33, 16385), (31, 70, 528), (32, 100, 512), (3, 40, 2001),
           (4, 4096, 4100), (7, 96, 1000), (16, 300, 4096), (33, 64, 128), (80, 200, 513), (260, 300, 96),
           (1, 100, 8192), (2, 70, 1024), (4, 70, 1025), (5, 70, 130), (8, 70, 512), (8, 70, 513), (9, 70, 300)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", LINEARS)
def test_linear(ia, M, N, K, dtype):
    gen = torch.Generator().manual_seed(M + N + K)
    x = torch.randn((M, K), generator=gen).to(dtype)
    weight = torch.randn((K, N), generator=gen) * K**-0.5
    bias = torch.randn(N, generator=gen).to(dtype)
    w, sw = ia.quantize_i8(weight.cuda(), transpose=True)
    y = ia.linear_i8(x.cuda(), w, sw, bias=bias.cuda())
    qx, sx = ref_quantize(x)
    qw, rsw = ref_quantize(weight.t().contiguous())
    check_product(y, qx @ qw.t(), sx, rsw, bias, dtype)
    # and what it approximates: half a step a factor on either side
    full = x.double() @ weight.double() + bias.double()
    half = 0.5 * (sx.double()[:, None] * weight.abs().double().sum(0) + x.abs().double().sum(1)[:, None] * rsw.double())
    half += 0.25 * K * sx.double()[:, None] * rsw.double()
    assert ((y.cpu().double() - full).abs() <= 1.01 * half + 2.0**-7 * full.abs()).all()
    # the same bits in two calls, by way of the parts it is made of, and with the caller's workspace
    q, s = ia.quantize_i8(x.cuda())
    ws = ia.linear_i8_workspace(M, N, K)
    ws.fill_(0xFF)
    assert torch.equal(ia.gemm_i8(q, s, w, sw, bias=bias.cuda(), dtype=dtype), y)
    assert torch.equal(ia.linear_i8(x.cuda(), w, sw, bias=bias.cuda(), workspace=ws), y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 70, 301), (5, 70, 301), (40, 70, 301), (200, 70, 301), (1, 70, 512), (6, 70, 512)])
def test_linear_strided_rows(ia, M, N, K, dtype):
    """Rows of x further apart and at odd places: the bits that dense rows give."""
    gen = torch.Generator().manual_seed(M + K)
    x = torch.randn((M, K), generator=gen).to(dtype).cuda()
    w, sw = ia.quantize_i8(torch.randn((K, N), generator=gen).cuda(), transpose=True)
    want = ia.linear_i8(x, w, sw)
    for ld, off in ((K + 1, 0), (K + 1, 1), (K + 8, 4), (K + 19, 3)):
        store = torch.full((M * ld + off,), float("nan"), dtype=dtype, device="cuda")
        view = torch.as_strided(store, (M, K), (ld, 1), off)
        view.copy_(x)
        assert torch.equal(ia.linear_i8(view, w, sw), want)


@pytest.mark.parametrize("M", [1, 5, 40, 200])
def test_linear_special_rows(ia, M):
    """A non-finite row is NaN and leaves the others alone; a row of zeros is the bias."""
    gen = torch.Generator().manual_seed(M)
    x = torch.randn((M, 200), generator=gen)
    weight = torch.randn((200, 70), generator=gen)
    bias = torch.randn(70, generator=gen)
    w, sw = ia.quantize_i8(weight.cuda(), transpose=True)
    plain = ia.linear_i8(x.cuda(), w, sw, bias=bias.cuda())
    for special in (float("nan"), float("inf")):
        y = x.clone()
        y[M // 2, 77] = special
        if M > 3:
            y[0] = 0
        out = ia.linear_i8(y.cuda(), w, sw, bias=bias.cuda())
        assert out[M // 2].isnan().all()
        if M > 3:
            assert torch.equal(out[0].cpu(), bias)
            keep = [i for i in range(1, M) if i != M // 2]
            assert torch.equal(out[keep], plain[keep])


def test_linear_of_no_rows(ia):
    w, sw = ia.quantize_i8(torch.randn(64, 32).cuda(), transpose=True)
    assert ia.linear_i8(torch.empty((0, 64), device="cuda"), w, sw).shape == (0, 32)
    q, s = ia.quantize_i8(torch.empty((0, 64), device="cuda"))
    assert q.shape == (0, 64) and s.shape == (0,)
    assert ia.gemm_i8(q, s, w, sw).shape == (0, 32)


@pytest.mark.parametrize("M", [3, 200])
def test_linear_streams_and_graphs(ia, M):
    """On a stream of the caller's, and captured: every replay is that of the inputs of then."""
    gen = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn((M, 2000), generator=gen, device="cuda")
    w, sw = ia.quantize_i8(torch.randn((2000, 300), generator=gen, device="cuda"), transpose=True)
    want = ia.linear_i8(x, w, sw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ia.linear_i8(x, w, sw, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    ws, out = ia.linear_i8_workspace(M, 300, 2000), torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ia.linear_i8(x, w, sw, out=out, workspace=ws)
    for i in range(4):
        x.normal_(generator=gen)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ia.linear_i8(x, w, sw))
