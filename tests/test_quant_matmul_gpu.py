"""The 8-bit matrix product on the GPU: 64-bit results, odd sizes, alignment, refusals."""
import pytest
import torch

import dense_layer_ref as ref

pytestmark = pytest.mark.gpu


def _rows(g, n, k):
    return torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8), torch.rand(n, generator=g) * 0.02 + 1e-4


def _check(out, x, w, xs, ws, bias, dtype):
    want, tol = ref.quant_matmul(x, w, xs, ws, bias)
    u = ref.half_step(dtype)
    assert out.dtype == dtype
    ref.assert_within(out, want, tol + u * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * u)


SIZES = [
    (1, 1, 1), (1, 16, 64), (2, 33, 65), (7, 129, 127), (16, 256, 512), (17, 130, 1000), (33, 513, 4096),
    (64, 576, 7168), (65, 200, 2112), (100, 512, 16), (128, 128, 128), (129, 127, 63), (255, 257, 192),
    (256, 256, 256), (300, 1000, 1024), (513, 640, 130), (1021, 2113, 515), (24, 300, 4112), (48, 1000, 2064),
    (200, 136, 4096), (2900, 3000, 200), (2817, 3001, 77),
]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_64_bits(dsa, dev, M, N, K, dtype):
    g = torch.Generator().manual_seed(M * 7 + N * 3 + K)
    (x, xs), (w, ws) = _rows(g, M, K), _rows(g, N, K)
    bias = torch.randn(N, generator=g) if (M + N) % 2 else None
    out = dsa.quant_matmul(x.to(dev), w.to(dev), xs.to(dev).view(-1, 1), ws.to(dev).view(-1, 1),
                           None if bias is None else bias.to(dev), dtype=dtype)
    assert tuple(out.shape) == (M, N)
    _check(out, x, w, xs, ws, bias, dtype)


@pytest.mark.parametrize("M,N,K", [(1100, 1981, 4160), (1030, 2012, 4113), (700, 2689, 4099)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_three_shares_of_a_long_k(dsa, dev, M, N, K, dtype):
    """Tiles for more than half and at most two thirds of the CUs."""
    g = torch.Generator().manual_seed(M + N + K)
    (x, xs), (w, ws) = _rows(g, M, K), _rows(g, N, K)
    out = dsa.quant_matmul(x.to(dev), w.to(dev), xs.to(dev), ws.to(dev), dtype=dtype)
    _check(out, x, w, xs, ws, None, dtype)


@pytest.mark.parametrize("M", [1, 5, 40, 130, 600])
def test_fp16_and_leading_dimensions(dsa, dev, M):
    g = torch.Generator().manual_seed(M)
    (x, xs), (w, ws) = _rows(g, 2 * M, 320), _rows(g, 96, 320)
    out = dsa.quant_matmul(x.view(2, M, 320).to(dev), w.to(dev), xs.view(2, M, 1).to(dev), ws.to(dev),
                           dtype=torch.float16)
    assert tuple(out.shape) == (2, M, 96)
    _check(out.view(2 * M, 96), x, w, xs, ws, None, torch.float16)


@pytest.mark.parametrize("off", [1, 3, 4, 8])
@pytest.mark.parametrize("M,N,K", [(3, 70, 160), (70, 300, 256), (300, 300, 192)])
def test_rows_off_16_bytes(dsa, dev, off, M, N, K):
    """Operands that start anywhere (views into a larger buffer) give the aligned call's bits."""
    g = torch.Generator().manual_seed(off)
    (x, xs), (w, ws) = _rows(g, M, K), _rows(g, N, K)
    want = dsa.quant_matmul(x.to(dev), w.to(dev), xs.to(dev), ws.to(dev), dtype=torch.float32)
    xb, wb = torch.zeros(M * K + 64, dtype=torch.int8, device=dev), torch.zeros(N * K + 64, dtype=torch.int8, device=dev)
    xv, wv = xb[off:off + M * K].view(M, K), wb[off:off + N * K].view(N, K)
    xv.copy_(x)
    wv.copy_(w)
    got = dsa.quant_matmul(xv, wv, xs.to(dev), ws.to(dev), dtype=torch.float32)
    assert torch.equal(got, want)


@pytest.mark.parametrize("M,N", [(1, 64), (200, 300)])
def test_extreme_sums(dsa, dev, M, N):
    """The longest rows at the largest products: -128 * -128 * 131071 < 2^31."""
    K = 131071
    x = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((N, K), -128, dtype=torch.int8, device=dev)
    w[1::2] = 127
    one = torch.ones(max(M, N), device=dev)
    out = dsa.quant_matmul(x, w, one[:M], one[:N], dtype=torch.float32)
    want = torch.where(torch.arange(N) % 2 == 0, 16384 * K, -128 * 127 * K).double().expand(M, N)
    ref.assert_within(out, want, ref.F32 * want.abs())


def test_behind_the_quantiser(dsa, dev):
    """act_quant's rows and scales go in as they come; the product is within the quantisation of the fp32 one."""
    g = torch.Generator().manual_seed(5)
    x, w = torch.randn(2, 37, 512, generator=g), torch.randn(130, 512, generator=g) / 512 ** 0.5
    xq, xs = dsa.act_quant(x.to(dev))
    wq, ws = dsa.act_quant(w.to(dev))
    out = dsa.quant_matmul(xq, wq, xs, ws, dtype=torch.float32).cpu().double()
    want = x.double() @ w.double().t()
    # Half a step of each operand, s / 2 apiece: sum_k (|x| sw / 2 + |w| sx / 2 + sx sw / 4).
    sx, sw = xs.cpu().double(), ws.cpu().double().view(1, 1, -1)
    tol = (x.double().abs().sum(-1, keepdim=True) * sw / 2 + w.double().abs().sum(-1).view(1, 1, -1) * sx / 2
           + 512 * sx * sw / 4) * (1 + 1e-5)
    assert ((out - want).abs() <= tol).all()


def test_empty(dsa, dev):
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device=dev)
    f = lambda n: torch.ones(n, device=dev)
    assert dsa.quant_matmul(z(0, 64), z(8, 64), f(0), f(8)).shape == (0, 8)
    assert dsa.quant_matmul(z(3, 64), z(0, 64), f(3), f(0)).shape == (3, 0)


def test_a_scale_that_is_not_finite_stays_in_its_row(dsa, dev):
    g = torch.Generator().manual_seed(9)
    (x, xs), (w, ws) = _rows(g, 40, 128), _rows(g, 64, 128)
    clean = dsa.quant_matmul(x.to(dev), w.to(dev), xs.to(dev), ws.to(dev))
    xs2 = xs.clone()
    xs2[7] = float("nan")
    got = dsa.quant_matmul(x.to(dev), w.to(dev), xs2.to(dev), ws.to(dev))
    assert torch.isnan(got[7]).all()
    keep = torch.arange(40, device=dev) != 7
    assert torch.equal(got[keep], clean[keep])


def test_wrapper_route_equals_native_route(dsa, dev):
    """A 16-bit bias goes through the Python route; its fp32 copy through the native one."""
    g = torch.Generator().manual_seed(3)
    (x, xs), (w, ws) = _rows(g, 20, 96), _rows(g, 48, 96)
    bias = torch.randn(48, generator=g).to(torch.bfloat16).to(dev)
    a = [t.to(dev) for t in (x, w, xs, ws)]
    assert torch.equal(dsa.quant_matmul(*a, bias), dsa.quant_matmul(*a, bias.float()))
    ops = dsa.load_torch_ops()
    assert torch.equal(ops.quant_matmul(*a, bias), dsa.quant_matmul(*a, bias))


def test_refusals(dsa, dev):
    z = torch.zeros(4, 64, dtype=torch.int8, device=dev)
    s = torch.ones(4, device=dev)
    with pytest.raises(ValueError, match="int8"):
        dsa.quant_matmul(z.float(), z, s, s)
    with pytest.raises(ValueError, match="float32"):
        dsa.quant_matmul(z, z, s.half(), s)
    with pytest.raises(ValueError, match="contiguous"):
        dsa.quant_matmul(z.t().contiguous().t(), z, s, s)
    with pytest.raises(ValueError, match="one entry per row"):
        dsa.quant_matmul(z, z, s[:3], s)
    with pytest.raises(ValueError, match="output channel"):
        dsa.quant_matmul(z, z, s, s[:3])
    with pytest.raises(ValueError, match="bias"):
        dsa.quant_matmul(z, z, s, s, torch.ones(5, device=dev))
    with pytest.raises(ValueError, match="dtype"):
        dsa.quant_matmul(z, z, s, s, dtype=torch.float64)
    with pytest.raises(ValueError, match="one device|HIP"):
        dsa.quant_matmul(z, z.cpu(), s, s)
    with pytest.raises(ValueError, match="K must be"):
        dsa.quant_matmul(torch.zeros(1, 131072, dtype=torch.int8, device=dev),
                         torch.zeros(1, 131072, dtype=torch.int8, device=dev), s[:1], s[:1])


def test_fewer_tokens_take_no_longer(dsa, dev):
    """128 tokens of a wide product are half the work of 256: they must not be put into tiles that they half fill."""
    N, K = 32768, 4096
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randint(-127, 128, (256, K), dtype=torch.int8, device=dev, generator=g)
    w = torch.randint(-127, 128, (N, K), dtype=torch.int8, device=dev, generator=g)
    xs, ws = torch.rand(256, device=dev, generator=g), torch.rand(N, device=dev, generator=g)

    def us(M):
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(10):
                dsa.quant_matmul(x[:M], w, xs[:M], ws)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b) * 100)
        return sorted(times)[2]

    half, all_ = us(128), us(256)
    assert half < 1.1 * all_, f"128 tokens {half:.0f} us, 256 {all_:.0f}"
