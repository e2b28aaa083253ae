"""The 8-bit product on more tiles than the device holds at once: whole results against 64-bit restatements."""
import pytest
import torch

from . import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OUTPUTS = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def completed():
    yield
    from svoo_b200 import ops
    assert ops.linear_status(torch.device(DEV)) == 0


def rand(M, K, dtype, seed, scale=1.0):
    g = torch.Generator(DEV).manual_seed(seed)
    return (torch.randn(M, K, generator=g, device=DEV) * (0.3 + torch.rand(K, generator=g, device=DEV)) * scale).to(dtype)


def check_e4m3(h, y32):
    """h holds the 32-bit results y32 in blocks along their columns: scales bit for bit; a number is the nearest to a quotient that
    is off by at most 2^-23 of itself (half a unit of its rounding and 2^-22 of one)."""
    _, scale = R.quantize(y32, 1, 128)
    assert torch.equal(h.scale.t(), scale)
    v = y32.double() / scale.double().repeat_interleave(128, 1)[:, :y32.shape[1]]
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp_min(-6) - 3)
    assert ((h.q.double() - v).abs() <= step / 2 + v.abs() * 2.0 ** -23).all()


@pytest.mark.parametrize("M,N,K", [(40008, 640, 128), (32760, 384, 128), (40001, 333, 128), (20000, 872, 256)])
def test_tiles_behind_the_last_column(M, N, K):
    """The last column tile is half empty: the warps of its empty half go on to a tile that is not, and store while a box of the
    tile before may still be on its way.  One or two blocks of k, so that the next box follows at once."""
    from svoo_b200 import ops
    x, w = rand(M, K, torch.bfloat16, M + K), rand(N, K, torch.bfloat16, N + K, 0.05)
    a, b = ops.quantize_rows(x), ops.quantize_blocks(w)
    ad, bd = R.dequantize(x, 1, 128), R.dequantize(w, 128, 128)
    want = ad @ bd.t()
    for _ in range(3):
        for dtype in OUTPUTS:
            y = ops.mm_fp8(a, b, None, None, dtype)
            assert ((y.double() - want).abs() <= R.product_bound(ad, bd, dtype, want)).all()
        check_e4m3(ops.mm_fp8(a, b, None, None, ops.E4M3), y)


# more than 148 tiles of 128 x 128, so that tiles go to pairs of SMs, and more than 74 of 256 x 256, so that a pair walks several
PAIRS = [(9000, 777, 130), (5001, 1160, 260), (20000, 384, 128), (19201, 5, 300), (9473, 513, 2000), (300, 8200, 1001), (19000, 640, 16)]


def test_the_sizes_walk():
    for M, N, _ in PAIRS:
        assert -(-M // 128) * -(-N // 128) > 148 and -(-M // 256) * -(-N // 256) > (74 if M > 300 else 65)


@pytest.mark.parametrize("dtype", OUTPUTS)
@pytest.mark.parametrize("M,N,K", PAIRS)
def test_pairs_of_sms(M, N, K, dtype):
    """Bias, GELU and every output type with block scales; rows whose 16-byte pieces TMA cannot store (odd N) among them."""
    from svoo_b200 import ops
    x, w = rand(M, K, dtype, M + K), rand(N, K, dtype, N + K, 0.05)
    bias = rand(1, N, OUTPUTS[(M + N + OUTPUTS.index(dtype)) % 3], N)[0]
    a, b = ops.quantize_rows(x), ops.quantize_blocks(w)
    ad, bd = R.dequantize(x, 1, 128), R.dequantize(w, 128, 128)
    plain = ad @ bd.t()
    want = plain + bias.double()
    g = R.gelu(want)
    for out in OUTPUTS:
        y = ops.mm_fp8(a, b, None, None, out)
        assert y.dtype == out and ((y.double() - plain).abs() <= R.product_bound(ad, bd, out, plain)).all()
        y = ops.mm_fp8(a, b, bias, None, out)
        tol = R.product_bound(ad, bd, torch.float32, want) + 2.0 ** -22 * bias.double().abs()
        assert ((y.double() - want).abs() <= tol + R.half_step(out) * want.abs() + torch.finfo(out).tiny).all()
        y = ops.mm_fp8(a, b, bias, "gelu", out)
        # GELU's slope is at most 1.13; its own evaluation is off by a few 2^-21 of its argument (exponential, division)
        assert ((y.double() - g).abs() <= 1.13 * tol + 2.0 ** -19 * want.abs() + R.half_step(out) * g.abs() + torch.finfo(out).tiny).all()
    check_e4m3(ops.mm_fp8(a, b, bias, "gelu", ops.E4M3), y)
    check_e4m3(ops.mm_fp8(a, b, bias, None, ops.E4M3), ops.mm_fp8(a, b, bias, None, torch.float32))
    assert torch.equal(ops.linear_fp8(x, b, bias, "gelu", torch.float32), y)


@pytest.mark.parametrize("dtype", OUTPUTS)
@pytest.mark.parametrize("M,N,K", [(5001, 1160, 260), (2500, 2310, 129), (300, 19001, 64), (4100, 1300, 2000)])
def test_pairs_of_sms_with_scales_per_row(M, N, K, dtype):
    from svoo_b200 import ops
    x, w = rand(M, K, dtype, M + K), rand(N, K, dtype, N + K, 0.05)
    a, b = ops.quantize_rows(x), ops.quantize_columns(w.t().contiguous())
    ad, bd = R.dequantize(x, 1, 128), R.dequantize(w, 1, 128)
    want = ad @ bd.t()
    assert -(-M // 256) * -(-N // 256) > 74
    for out in OUTPUTS:
        y = ops.mm_fp8(a, b, None, None, out)
        assert y.dtype == out and ((y.double() - want).abs() <= R.product_bound(ad, bd, out, want)).all()


@pytest.mark.parametrize("dtype", OUTPUTS)
def test_training_step_on_pairs_of_sms(dtype):
    """All three products of a step walk several tiles a pair."""
    from svoo_b200 import linear
    M, N, K = 5200, 4100, 1300
    x, w, dy, b = rand(M, K, dtype, 1), rand(N, K, dtype, 2, 0.05), rand(M, N, dtype, 3, 0.01), rand(1, N, torch.float32, 4)[0]
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear.linear_fp8(x, w, b)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach() for t in (x, w, b))
    for got, u, v, add in ((y.detach(), R.dequantize(x, 1, 128), R.dequantize(w, 128, 128), b.double()),
                           (dx, R.dequantize(dy, 1, 128), R.dequantize(w, 128, 128).t(), 0),
                           (dw, R.dequantize(dy.t().contiguous(), 1, 128), R.dequantize(x.t().contiguous(), 1, 128), 0)):
        want = u @ v.t() + add
        tol = R.product_bound(u, v, dtype, want) + (2.0 ** -22 * add.abs() if got.shape == (M, N) else 0)
        assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all()
    ref = dy.double().sum(0)
    # 64 additions of 128 rows' sums and of 41 such sums
    assert ((db.double() - ref).abs() <= 110 * 2.0 ** -24 * dy.double().abs().sum(0) + 1e-30).all()
