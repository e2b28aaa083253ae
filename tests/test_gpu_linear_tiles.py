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
