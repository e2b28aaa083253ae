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
