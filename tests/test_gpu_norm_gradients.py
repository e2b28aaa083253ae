"""The gradient of the layer norm where its forms meet: samples with gains of their own, far means, constant rows."""
import pytest
import torch

from . import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def completed():
    yield
    from svoo_b200 import ops
    assert ops.linear_status(torch.device(DEV)) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,C", [(3, 5, 64), (2, 40, 1001), (4, 1, 1536)])
def test_gradient_of_x_alone_takes_every_samples_gain(dtype, B, S, C):
    """The call of the library without dgain, whether or not it is told that sums would be per sample: the bits of the full call."""
    from svoo_b200 import ops
    from svoo_b200._lib import LIB, check
    g = torch.Generator(DEV).manual_seed(C)
    x, dy = (torch.randn(B, S, C, generator=g, device=DEV).to(dtype) for _ in range(2))
    six = torch.randn(B, 6, C, generator=g, device=DEV)
    scale = six[:, 2:3]
    _, mean, rstd = ops.layer_norm(x, scale=scale, return_stats=True)
    want = ops.layer_norm_backward(dy, x, mean, rstd, scale=scale)[0]
    ref = R.layer_norm_grad(x, dy, 1 + scale.double(), 1e-6)[0]
    assert (want.double() - ref).norm() <= 2 * R.half_step(dtype) * ref.norm() + 1e-5 * ref.norm()      # gains are taken, not one for all
    for per_sample in (0, 1):
        dx = torch.empty_like(x)
        check(LIB.svoo_b200_layer_norm_backward(dy.data_ptr(), S * C, C, x.data_ptr(), ops.TYPES[dtype], B, S, C, S * C, C, mean.data_ptr(),
                                                rstd.data_ptr(), scale.data_ptr(), 6 * C, 2, 1, per_sample, dx.data_ptr(), None, None, None, 0,
                                                torch.cuda.current_stream().cuda_stream), "layer_norm_backward")
        assert torch.equal(dx, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [1, 40, 64, 1001, 4096, 8200])
def test_constant_rows_have_no_slope(dtype, C):
    """x - mean is zero (one column; or a value whose sums are exact), so xhat and with it dgain are, whatever rstd = 1000 makes of a
    rounding; dx = rstd (w - mean w), for one column what rounding w leaves: w = dy g is subtracted unrounded from the mean of the
    rounded w, at most 2^-24 |w| apart, and the product with rstd and the result are rounded once each."""
    from svoo_b200 import ops
    x = torch.tensor([1.0, 1000.0, 10000.0, -3.0], device=DEV).to(dtype).view(4, 1).expand(4, C).contiguous()
    dy = torch.randn(4, C, device=DEV).to(dtype)
    g = torch.randn(C, device=DEV)
    y, mean, rstd = ops.layer_norm(x, g, torch.zeros_like(g), return_stats=True)
    dx, dgain, doffset = ops.layer_norm_backward(dy, x, mean, rstd, g)
    still = mean == x[:, 0].float()                          # a reciprocal of C that is rounded may put the mean beside the value
    assert C not in (1, 64, 4096) or still.all()
    if still.all():
        assert not dgain.any() and not y.any()
    left = rstd.double()[:, None] * 2.0 ** -24 * (dy.double() * g.double()).abs()
    assert C > 1 or (dx.double().abs() <= left * (1 + 2.0 ** -23 + R.half_step(dtype)) + torch.finfo(dtype).tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,C", [(5, 64), (3, 777), (4, 1536), (2, 5121), (2, 8200), (2, 12290)])
@pytest.mark.parametrize("centre", [0.0, 30.0, 1000.0])
def test_far_means_cost_the_gradient_no_digits(dtype, B, C, centre):
    """One row a sample, so that dgain is dy xhat of it.  Against 64 bits on the statistics that the forward call gave: x - mean and the
    product with rstd round once each, dy once more, whatever the mean."""
    from svoo_b200 import ops
    gen = torch.Generator(DEV).manual_seed(C)
    x = (torch.randn(B, 1, C, generator=gen, device=DEV) + centre).to(dtype)
    dy = torch.randn(B, 1, C, generator=gen, device=DEV).to(dtype)
    scale = torch.randn(B, 1, C, generator=gen, device=DEV)
    _, mean, rstd = ops.layer_norm(x, scale=scale, return_stats=True)
    dx, dgain, _ = ops.layer_norm_backward(dy, x, mean, rstd, scale=scale)
    r = rstd.double()[..., None]
    xhat = (x.double() - mean.double()[..., None]) * r
    want = dy.double() * xhat
    assert ((dgain.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs() + torch.finfo(torch.float32).tiny).all()
    w = dy.double() * (1 + scale.double())
    want = r * (w - w.mean(-1, keepdim=True) - xhat * (w * xhat).mean(-1, keepdim=True))
    # sums of at most 46 additions a thread and tree and 14 other roundings, each of its term's magnitude
    size = w.abs() + w.abs().mean(-1, keepdim=True) + xhat.abs() * (w * xhat).abs().mean(-1, keepdim=True)
    assert ((dx.double() - want).abs() <= r * 60 * 2.0 ** -24 * size + R.half_step(dtype) * want.abs() + torch.finfo(dtype).tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_overlap_or_are_one(dtype):
    """One row seen as many, windows that overlap, samples that overlap."""
    from svoo_b200 import ops
    flat = torch.randn(6000, device=DEV).to(dtype)
    for x in (flat[:64].expand(50, 64), flat[:1000].view(1, 1000).expand(3, 7, 1000), flat.as_strided((90, 64), (3, 1)), flat.as_strided((2, 30, 129), (40, 100, 1)),
              flat.as_strided((3, 20, 200), (8, 16, 1), 8), flat[3:67].expand(1, 1, 64)):
        C = x.shape[-1]
        g, o = torch.randn(C, device=DEV), torch.randn(C, device=DEV)
        y, mean, rstd = ops.layer_norm(x, g, o, return_stats=True)
        want, _, m, r = R.layer_norm(x, g, o, 1e-6)
        # the mean is off by 80 x 2^-24 of the largest magnitude at most, everything else by less
        tol = (80 * 2.0 ** -24 * 8 * r * (1 + r)) * g.abs().double() + 2.0 ** -20 * (want.abs() + o.abs()) + R.half_step(dtype) * want.abs()
        assert x.abs().max() < 7.9 and ((y.double() - want).abs() <= tol).all()
        got = ops.layer_norm_backward(y, x, mean, rstd, g)
        ref = R.layer_norm_grad(x, y, g, 1e-6)[0]
        assert (got[0].double() - ref).norm() <= 1.01 * R.half_step(dtype) * ref.norm() + 1e-5 * (r * g.abs().max() * y.double().abs()).norm()
        if x.dim() == 2:
            assert torch.equal(ops.quantize_rows(x).q.view(torch.uint8), ops.quantize_rows(x.contiguous()).q.view(torch.uint8))
            assert torch.equal(ops.quantize_columns(x).q.view(torch.uint8), ops.quantize_columns(x.contiguous()).q.view(torch.uint8))
