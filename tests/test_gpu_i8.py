"""8-bit rows and matrix products on the GPU against plain 64-bit forms (tests/serve_ref.py):
codes exactly, scales and products within their fp32 roundings."""
from __future__ import annotations

import pytest

from tests import serve_ref as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2048), (3, 31), (7, 155), (300, 128), (2, 9001), (1, 131072), (129, 768), (2100, 400),
                                       (2050, 4100), (2048, 33)])
@pytest.mark.parametrize("norm", [False, True])
def test_rows(rows, cols, dtype, norm):
    from tinygiant_b200.int8 import quantize_rows
    x = randn(cols, rows, cols).to(dtype)
    w = 1 + 0.2 * randn(1, cols) if norm else None
    codes, scales = quantize_rows(x, w, 1e-5)
    want, ws = R.i8_rows(x, w, 1e-5)
    assert codes.shape == (rows, (cols + 15) // 16 * 16)
    assert torch.equal(codes[:, :cols].double(), want) and not codes[:, cols:].any()
    # the maximum, a quotient; with the norm a sum of cols squares, its quotient, root, quotient and product
    tol = (2 + (cols / 2 + 6 if norm else 0)) * 2.0 ** -24
    assert ((scales.double()[:, None] - ws).abs() <= tol * ws).all()


def test_rows_ties_zeros_tiny_and_not_finite():
    from tinygiant_b200.int8 import quantize_rows
    x = randn(2, 12, 64)
    x[0] = 0
    x[1] = torch.arange(64, device="cuda") - 31.5
    x[1, 0] = 127                    # quotients k + 1/2: to even
    x[2, 0] = 254                    # 127 x / 254 = x / 2
    x[2, 1:] = torch.arange(63, device="cuda").float()
    x[3] *= 1e-38
    x[4] *= 1e-44
    x[5, 7] = float("inf")
    x[6, 8] = float("nan")
    x[7, 3] = 3.4e38
    x[8] = 1e-45
    codes, scales = quantize_rows(x)
    fine = [i for i in range(12) if i not in (5, 6)]
    want, ws = R.i8_rows(x[fine])
    assert torch.equal(codes[fine].double(), want)
    # half a step of the smallest number where the scale is subnormal
    assert ((scales[fine].double()[:, None] - ws).abs() <= 2 * 2.0 ** -24 * ws + 2.0 ** -150).all()
    assert torch.isnan(scales[5:7]).all() and not codes[5:7].any()
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(3, 5, 64))
    out = lin(x)
    assert torch.isnan(out[5:7]).all() and not out[0].any()
    # row 7's products reach 3.4e38 times a weight above 1: what is beyond fp32 there is an infinity
    ref = (want @ lin.codes.double().T) * ws * lin.scales.double()
    assert torch.equal(torch.isfinite(out[fine]), ref.abs() < 3.4028235677973366e38)


def product_ref(x, lin, norm, eps, residual):
    codes, s = R.i8_rows(x, norm, eps)
    k = x.shape[1]
    out = (codes @ lin.codes[:, :k].double().T) * s * lin.scales.double()
    return (out if residual is None else out + residual.double()), out


def check(x, lin, norm=None, residual=None, eps=1e-5, **kw):
    got = lin(x, norm=norm, eps=eps, residual=residual, **kw)
    ref, prod = product_ref(x, lin, norm, eps, residual)
    # the integer sum to fp32, sa, sa * sw and its product (sa: see the rows), the residual's sum,
    # the type's rounding
    k = x.shape[1]
    tol = (6 + (k / 2 + 6 if norm is not None else 0)) * 2.0 ** -24 * prod.abs() + 2.0 ** -24 * ref.abs()
    tol = tol + 1.001 * R.EPS[x.dtype] * (ref.abs() + tol) + (2.0 ** -25 if x.dtype == F16 else 1e-44)
    assert got.dtype == x.dtype
    d = (got.double() - ref).abs()
    assert (d <= tol).all(), (d / tol).max().item()
    return got


SHAPES = [(1, 1, 1), (1, 5120, 2048), (2, 37, 155), (3, 129, 48), (8, 512, 4096), (9, 1000, 1000), (16, 257, 2049),
          (17, 64, 16), (31, 2048, 768), (64, 300, 4096), (65, 1025, 333), (128, 128, 128), (129, 255, 640),
          (200, 777, 1999), (513, 513, 513), (1, 33, 131072), (300, 40, 7168), (96, 2048, 4096),
          (90, 500, 8000), (250, 1000, 2048), (700, 2000, 300)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, dtype):
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(1, n, k) * 0.05)
    x = (randn(2, m, k) * 2).to(dtype)
    check(x, lin)
    check(x, lin, norm=1 + 0.2 * randn(3, k), residual=randn(4, m, n).to(dtype))


def test_every_row_count():
    """Each m through the boundaries between variants, against one large product's rows."""
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(5, 301, 500) * 0.05)
    x = randn(6, 280, 500)
    whole = check(x, lin)
    for m in list(range(1, 70)) + [127, 128, 129, 255, 256, 257]:
        assert torch.equal(lin(x[:m]), whole[:m]), m


def test_largest_sums():
    """All codes +-127 over the longest rows: the integer sum's extremes."""
    from tinygiant_b200.int8 import Int8Linear
    k = 131072
    w = torch.ones(40, k, device="cuda")
    w[1::2] = -1
    lin = Int8Linear.quantize(w)
    for m in (1, 20, 150):
        check(torch.full((m, k), 3.0, device="cuda"), lin)


def test_strides_alignment_in_place_and_empty():
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(7, 150, 150) * 0.1)
    for m in (3, 40, 300):
        for dtype in (F32, BF16):
            wide = randn(8, m, 500).to(dtype)
            x = wide[:, 101:251]                          # rows that start on no vector boundary
            want = check(x.contiguous(), lin)
            out = torch.full((m, 333), 4.0, dtype=dtype, device="cuda")
            lin(x, out=out[:, 17:167])
            assert torch.equal(out[:, 17:167], want)
            assert (out[:, :17] == 4).all() and (out[:, 167:] == 4).all()
            h = x.contiguous()
            res = check(x.contiguous(), lin, residual=x)
            lin(h, residual=h, out=h)                     # out over residual and x
            assert torch.equal(h, res)
    assert lin(torch.empty(0, 150, device="cuda")).shape == (0, 150)


@pytest.mark.parametrize("m", [1, 24, 200])
def test_streams_and_graphs(m):
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(9, 600, 1024) * 0.05)
    x, norm = randn(10, m, 1024), 1 + 0.1 * randn(11, 1024)
    want = lin(x, norm=norm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = lin(x, norm=norm, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lin(x, norm=norm))
        graphs.append(g)
    x.copy_(randn(12, m, 1024))
    ref = lin(x, norm=norm)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k", [(2100, 8449, 2048), (2177, 8500, 100), (4097, 4700, 31), (2305, 8193, 16), (76000, 100, 130),
                                   (300, 38000, 500)])
def test_product_of_many_tiles(m, n, k, dtype):
    """Tokens and channels for several rounds of the largest tiles, whose last ones are nearly empty."""
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(1, n, k) * 0.05)
    x = (randn(2, m, k) * 2).to(dtype)
    got = check(x, lin)
    if dtype == BF16:
        check(x, lin, norm=1 + 0.2 * randn(3, k), residual=randn(4, m, n).to(dtype))
        wide = torch.full((m, n + 3), 7.0, dtype=dtype, device="cuda")   # rows on no vector boundary
        lin(x, out=wide[:, 1:n + 1])
        assert torch.equal(wide[:, 1:n + 1], got) and (wide[:, 0] == 7).all() and (wide[:, n + 1:] == 7).all()
        graph, y = torch.cuda.CUDAGraph(), torch.empty_like(got)
        with torch.cuda.graph(graph):
            lin(x, out=y)
        x.mul_(0.5)   # the codes stay, the scales halve
        for _ in range(3):
            y.fill_(1)
            graph.replay()
            assert torch.equal(y, lin(x))


def test_host_threads():
    """Products of other tile widths from host threads, each on its own stream: no call disturbs
    another's launch."""
    import threading
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(1, 640, 512) * 0.05)
    xs = [randn(2, 3, 512), randn(3, 200, 512)] * 2
    want, wrong = [lin(x) for x in xs], []
    torch.cuda.synchronize()

    def work(x, y):
        try:
            stream = torch.cuda.Stream()
            for _ in range(2000):
                got = lin(x, stream=stream)
            stream.synchronize()
            assert torch.equal(got, y)
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(xs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[0]


def test_rows_of_zeros_under_weights_far_above_the_maximum():
    """A weight times 127 / max |y| beyond fp32 meets values that are 0 or next to it."""
    from tinygiant_b200.int8 import quantize_rows
    for cols in (64, 50):
        x = torch.zeros(3, cols, device="cuda")
        w = torch.ones(cols, device="cuda")
        w[5:9] = 1e10
        x[0, 0], x[1, 0], x[2, 0] = 1e-28, 1e-28, -2e-29
        x[1, 6], x[2, 7] = 3e-39, -1e-39     # products of 3e-29 and -1e-29
        codes, _ = quantize_rows(x, w, 1e-5)
        assert torch.equal(codes[:, :cols].double(), R.i8_rows(x, w, 1e-5)[0])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(1, 300, 2048), (3, 129, 47), (70, 257, 333), (2100, 64, 400)])
def test_fp32_rows_as_a_16_bit_type(m, n, k, dtype):
    """The same bits as from x.to(dtype), strided rows included; finite values beyond the type's
    range, which would become infinities there, count as they are."""
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(1, n, k) * 0.05)
    wide = randn(2, m, k + 9) * 10.0 ** torch.randint(-6, 3, (m, 1), generator=torch.Generator().manual_seed(k)).cuda()
    norm, res = 1 + 0.2 * randn(3, k), randn(4, m, n).to(dtype)
    for x in (wide[:, 5:5 + k], wide[:, 5:5 + k].contiguous()):
        y = x.to(dtype)
        assert torch.equal(lin(x, dtype=dtype), lin(y))
        assert torch.equal(lin(x, norm=norm, residual=res, dtype=dtype), lin(y, norm=norm, residual=res))
    big = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).cuda()
    big[:, ::7] *= 1e6 if dtype == F16 else 1e20
    if dtype == BF16:
        big[:, 0] = 3.4e38                        # rounds to an infinity in bfloat16
    rounded = torch.where(torch.isfinite(big.to(dtype)), big.to(dtype).float(), big)
    assert torch.equal(lin(big, dtype=dtype), lin(rounded).to(dtype))
    if dtype == F16:   # squares of 3e38 are beyond fp32's sums
        got, want = lin(big, norm=norm, dtype=dtype).double(), lin(rounded, norm=norm).double()
        # sums of squares in another order, and the type's rounding
        assert ((got - want).abs() <= (k * 2.0 ** -24 + 1.001 * 2.0 ** -11) * want.abs() + 2.0 ** -25).all()



def test_refuses_other_types_of_rows():
    from tinygiant_b200.int8 import Int8Linear
    lin = Int8Linear.quantize(randn(1, 8, 32))
    x = randn(2, 3, 32)
    for bad in (dict(x=x.half(), dtype=BF16), dict(x=x.half(), dtype=F32), dict(x=x, dtype=torch.float64), dict(x=x.double())):
        with pytest.raises(TypeError):
            lin(**bad)
    for bad in (dict(out=torch.empty(3, 8, device="cuda")), dict(residual=torch.zeros(3, 8, device="cuda"))):
        with pytest.raises(ValueError):
            lin(x, dtype=BF16, **bad)
