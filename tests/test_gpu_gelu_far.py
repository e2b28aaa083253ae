"""GELU in the products' epilogues at arguments far from zero: rows of zeros make every argument a bias."""
import pytest
import torch

from . import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ARGS = [-float("inf"), -3.4e38, -1e30, -1e18, -65504.0, -100.0, -8.0, -7.0, -3.0, -1e-30, 0.0, 1e-30, 2.0, 7.0, 100.0, 1e18, 3.4e38, float("inf"),
        float("nan")]


# few rows in one launch, tiles shared out in clusters, tiles on pairs of SMs (more than 148 of 128 x 128)
@pytest.mark.parametrize("M,N", [(1, 300), (16, 300), (20, 300), (20000, 300)])
@pytest.mark.parametrize("at", range(2))
def test_far_arguments(M, N, at):
    """At every argument, next to one of either kind: two columns share a reciprocal."""
    from svoo_b200 import ops
    x = torch.zeros(M, 256, device=DEV)
    w = ops.quantize_blocks(torch.randn(N, 256, device=DEV))
    bias = torch.linspace(-4, 4, N, device=DEV)
    bias[at:at + 2 * len(ARGS):2] = torch.tensor(ARGS, device=DEV)
    y = ops.linear_fp8(x, w, bias, "gelu")
    want = R.gelu(bias.double())
    far = bias <= -8
    assert torch.equal(torch.isnan(y), (torch.isnan(want) | (bias == -float("inf"))).expand(M, N))   # -inf: 0 times infinity, as torch has it
    far &= bias > -float("inf")
    assert not y[:, far].any()
    fine = torch.isfinite(bias) & ~far
    # a few 2^-21 of the argument for the evaluation, and what the cut leaves out
    assert ((y[:, fine].double() - want[fine]).abs() <= 2.0 ** -19 * bias[fine].double().abs() + 2.0 ** -57).all()
    assert (y[:, bias == float("inf")] == float("inf")).all()


@pytest.mark.parametrize("M", [20, 20000])
def test_far_argument_leaves_its_block_alone(M):
    """With an e4m3 output a pre-activation of the type's lowest value must not set the scale of its block."""
    from svoo_b200 import ops
    a = ops.quantize_rows(torch.zeros(M, 256, device=DEV))
    w = ops.quantize_blocks(torch.randn(256, 256, device=DEV))
    bias = torch.linspace(0.5, 4, 256, device=DEV)
    bias[5], bias[200] = torch.finfo(torch.float32).min, -1e18
    h = ops.mm_fp8(a, w, bias, "gelu", ops.E4M3)
    q, s = R.quantize(ops.mm_fp8(a, w, bias, "gelu", torch.float32), 1, 128)
    assert torch.equal(h.scale.t(), s) and (s < 4.1 / 448).all()
    assert not h.float()[:, [5, 200]].any()
    # e4m3 rounds by at most 2^-4 of the value; the smallest here, 0.35, is far above the block's underflow
    g = R.gelu(bias.double()).clamp_min(0)
    assert ((h.float().double() - g).abs() <= 2.0 ** -4 * (1 + 2.0 ** -18) * g).all()
