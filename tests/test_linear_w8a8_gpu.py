"""The linear layer of int8 weights: against exact integer sums, at every way that a call is cut."""
import pytest
import torch

import superl8_amd as sl8
from superl8_amd import _C
from superl8_amd.format import QTensor

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DEV = "cuda"


def inputs(M, N, K, dtype, bias=None, full=False):
    x = torch.randn(M, K, device=DEV).to(dtype)
    w = torch.randint(-128, 128, (N, K), device=DEV, dtype=torch.int8)
    ws = (torch.rand(N, device=DEV) + 0.5) * 1e-3
    b = None if bias is None else (torch.randn(N, device=DEV) * 3).to(bias)
    return x, w, ws, b


def check(x, w, ws, bias, out):
    """The codes are those of quantize_i8_rowwise, bit for bit, and the integer sums exact. Roundings: the sum and
    two products (3 * 2^-24 of the product), the addition of the bias, the output's."""
    y = sl8.linear_w8a8(x, w, ws, bias=bias, out_dtype=out)
    c, xs = sl8.quantize_i8_rowwise(x.reshape(-1, x.shape[-1]).contiguous())
    p = torch.cat([c.double() @ part.double().T for part in w.split(4096)], 1) * xs.double()[:, None] * ws.double()
    want = p if bias is None else p + bias.double()
    lim = 3.01 * 2.0 ** -24 * p.abs() + (2.0 ** -24 + torch.finfo(out).eps / 2) * 1.0001 * want.abs() + \
        (2.0 ** -25 if out == F16 else 0)
    assert y.dtype == out and y.shape == (*x.shape[:-1], w.shape[0])
    err = (y.reshape(want.shape).double() - want).abs()
    assert bool((err <= lim).all()), (float((err - lim).max()), float(err.max()))
    return y


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 129, 257])
@pytest.mark.parametrize("N,K", [(1, 16), (16, 64), (33, 20), (100, 128), (127, 132), (256, 1040), (130, 2052),
                                 (515, 5120), (64, 5124)])
def test_sizes(M, N, K):
    dt = (F16, BF16, F32)[(M + N) % 3]
    check(*inputs(M, N, K, dt, (None, F16, BF16, F32)[(M + K // 4) % 4]), (F16, BF16, F32)[M % 3])


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (16, 17408, 512), (5, 5000, 4100), (24, 17408, 1024),
                                   (64, 4096, 4096), (128, 1024, 8192), (200, 4096, 4096), (700, 5003, 1028),
                                   (1000, 8192, 1024), (2100, 4100, 260), (2049, 4099, 2052), (4096, 4352, 1024),
                                   (3, 64, 20000), (40, 40, 131068), (300, 700, 33000), (5, 300000, 64)])
@pytest.mark.parametrize("out", [F16, F32])
def test_large(M, N, K, out):
    check(*inputs(M, N, K, F16, BF16), out)


@pytest.mark.parametrize("M", [1, 40, 300])
def test_extremes(M):
    """The largest sums, rows of zeros, an outlier in a row, subnormal rows."""
    K = 131068
    w = torch.full((40, K), -128, device=DEV, dtype=torch.int8)
    check(torch.full((M, K), 3.0, device=DEV, dtype=F16), w, torch.ones(40, device=DEV) * 1e-9, None, F32)
    x, w, ws, _ = inputs(M, 64, 512, F16)
    x[0] = 0
    x[-1, 7] = 60000.0
    check(x, w, ws, None, F32)
    assert bool((sl8.linear_w8a8(torch.zeros_like(x), w, ws) == 0).all())
    x, w, ws, _ = inputs(M, 64, 512, BF16)
    check(x * 1e-30, w, ws * 1e30, None, F32)
    check((x.float() * 2.0 ** -18).to(F16), w, ws, None, F32)


def test_tails_are_not_read():
    """K that is no multiple of 16 or 128: weights and activations end where the buffers end."""
    for K in (20, 36, 124, 132, 1036):
        pool = torch.zeros(50 * K, device=DEV, dtype=torch.int8)
        w = pool[-7 * K:].view(7, K)
        w.copy_(torch.randint(-127, 128, (7, K), device=DEV, dtype=torch.int8))
        for M in (1, 20, 70):
            check(torch.randn(M, K, device=DEV).half(), w, torch.ones(7, device=DEV), None, F32)


def test_views_and_leading_dimensions():
    x, w, ws, b = inputs(12, 96, 256, F16, F16)
    want = check(x, w, ws, b, F16)
    assert torch.equal(sl8.linear_w8a8(x.view(3, 4, 256), w, ws, bias=b), want.view(3, 4, 96))
    assert torch.equal(sl8.linear_w8a8(x.t().contiguous().t(), w.t().contiguous().t(), ws, bias=b), want)
    y = torch.empty(12 * 256 + 1, device=DEV, dtype=F16)[1:].view(12, 256)
    v = torch.empty(96 * 256 + 4, device=DEV, dtype=torch.int8)[4:].view(96, 256)
    y.copy_(x)
    v.copy_(w)
    assert torch.equal(sl8.linear_w8a8(y, v, ws, bias=torch.stack([b, b], 1)[:, 0]), want)
    assert sl8.linear_w8a8(x[:0], w, ws).shape == (0, 96) and sl8.linear_w8a8(x, w[:0], ws[:0]).shape == (12, 0)
    assert torch.equal(sl8.linear_w8a8(x[0], w, ws, bias=b), sl8.linear_w8a8(x[:1], w, ws, bias=b)[0])


def test_rows_do_not_depend_on_the_batch():
    """A row's result is the same bits alone and in batches that are cut in other ways."""
    x, w, ws, b = inputs(600, 1000, 2048, BF16, F32)
    all_rows = sl8.linear_w8a8(x, w, ws, bias=b, out_dtype=F32)
    for n in (1, 7, 16, 30, 64, 100, 300):
        assert torch.equal(sl8.linear_w8a8(x[:n], w, ws, bias=b, out_dtype=F32), all_rows[:n])


def test_qtensor():
    x, w, ws, b = inputs(20, 96, 256, F16, F16)
    assert torch.equal(sl8.linear(x, QTensor(w, ws, "per_row_i8"), bias=b), sl8.linear_w8a8(x, w, ws, bias=b))
    with pytest.raises(ValueError, match="rotated"):
        sl8.linear(x, QTensor(w, ws, "per_row_i8", rotated=True))


@pytest.mark.parametrize("M,N,K", [(1, 512, 512), (200, 4096, 4096)])
def test_streams_and_graphs(M, N, K):
    x, w, ws, b = inputs(M, N, K, F16, F16)
    want = sl8.linear_w8a8(x, w, ws, bias=b)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)] * 3:
        with torch.cuda.stream(s):
            got.append(sl8.linear_w8a8(x, w, ws, bias=b))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sl8.linear_w8a8(x, w, ws, bias=b)
    for _ in range(4):
        x.copy_(torch.randn(x.shape, device=DEV))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sl8.linear_w8a8(x, w, ws, bias=b))


def test_refusals():
    x, w, ws, b = inputs(4, 32, 64, F16, F16)
    base = dict(x=x, w=w, w_scale=ws, bias=b)
    for change in [dict(x=x.double()), dict(x=x[None]), dict(x=x[:, :60]), dict(x=x[:, :12], w=w[:, :12].contiguous()),
                   dict(x=x[:, :18].contiguous(), w=w[:, :18].contiguous()), dict(w=w.float()), dict(w=w[0]),
                   dict(w_scale=ws.half()), dict(w_scale=ws[:5]), dict(bias=b[:5]), dict(bias=b[:, None]),
                   dict(bias=b.int()), dict(out_dtype=torch.int8), dict(w=w.cpu()), dict(bias=b.cpu()),
                   dict(x=x.t().contiguous().t()),
                   dict(x=torch.zeros(1, 131072, device=DEV, dtype=F16), w=torch.zeros(32, 131072, device=DEV, dtype=torch.int8))]:
        with pytest.raises(RuntimeError, match="fni8"):
            _C.linear_w8a8(**base | change)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", [(3, 40, 512), (16, 40, 5120), (33, 257, 1028), (700, 300, 20000)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_not_finite(M, N, K, dtype, bad):
    """A row with NaN or infinity has no finite output; the others do not change."""
    x, w, ws, b = inputs(M, N, K, dtype, F32)
    rows = [1, M - 1]
    x[rows[0], K - 1] = bad
    x[rows[1], K // 3] = bad
    y = sl8.linear_w8a8(x, w, ws, bias=b)
    assert not bool(y[rows].isfinite().any())
    x[rows] = 0
    rest = [i for i in range(M) if i not in rows]
    assert torch.equal(y[rest], sl8.linear_w8a8(x, w, ws, bias=b)[rest])


@pytest.mark.parametrize("N,K", [(300, 1024), (4099, 2052), (1000, 20000)])
def test_bits_of_a_row_in_any_batch(N, K):
    """Streamed, in tiles, in parts of K: a row's outputs are the same bits."""
    x, w, ws, b = inputs(1500, N, K, BF16, F16)
    y = sl8.linear_w8a8(x, w, ws, bias=b, out_dtype=F32)
    for M in (1, 3, 7, 16, 40, 100, 400):
        assert torch.equal(sl8.linear_w8a8(x[:M], w, ws, bias=b, out_dtype=F32), y[:M])


@pytest.mark.parametrize("out", [F16, BF16])
@pytest.mark.parametrize("N,K,most", [(60000, 512, 300), (30000, 4096, 40), (4099, 2052, 1500), (20000, 5120, 100)])
@pytest.mark.parametrize("bias", [None, F16])
def test_roundings_do_not_go_by_the_batch(N, K, most, out, bias):
    """16-bit outputs too are the same bits streamed, in tiles and in parts of K: some of so many lie next to the
    middle of two neighbours, where one rounding and two give different ones."""
    x, w, ws, b = inputs(most, N, K, out, bias)
    y = sl8.linear_w8a8(x, w, ws, bias=b, out_dtype=out)
    exact = sl8.linear_w8a8(x, w, ws, bias=b, out_dtype=F32)
    assert torch.equal(y, exact.to(out))
    for M in (1, 4, 7, 16, 33, 100, 300, 700):
        if M < most:
            assert torch.equal(sl8.linear_w8a8(x[:M], w, ws, bias=b, out_dtype=out), y[:M]), M


@pytest.mark.parametrize("M,N,K", [(1, 128256, 4096), (16, 128256, 4096), (33, 128256, 4096), (64, 128256, 4096),
                                   (100, 128256, 4096), (1, 151936, 5120), (4, 57344, 8192), (3, 58591, 5148), (9, 48000, 10212),
                                   (120, 65381, 2048)])
def test_few_rows_of_many_channels(M, N, K):
    """Where every tile comes to the time of the weights' bytes."""
    check(*inputs(M, N, K, F16, BF16), F16)


@pytest.mark.parametrize("M,N,K", [(1, 14336, 4096), (1, 17408, 5120), (4, 30000, 4096), (16, 12288, 4096), (2, 20011, 2052),
                                   (16, 9001, 4100), (7, 40000, 1024)])
@pytest.mark.parametrize("out", [F16, F32])
def test_many_turns_of_the_streaming_kernel(M, N, K, out):
    """3 to 8 groups of channels a workgroup: the places of the waves' sums are written again, other waves put them out."""
    check(*inputs(M, N, K, BF16, F16), out)
