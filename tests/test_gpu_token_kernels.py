"""The token-wise half of a DiT block on this package's kernels: modules, and whole blocks against the torch ones."""
import pytest
import torch
import torch.nn as nn

from . import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dense_dit(cls_name, **kw):
    """A small DiT whose self-attention takes the dense branch: what differs between two of them are norms and linear layers."""
    from svoo_b200 import processor, wan_dit
    cfg = wan_dit.WanDiTConfig(num_layers=2, dim=512, heads=4, ffn_dim=1024, text_dim=64, text_len=16, latent=(3, 16, 20))
    model = wan_dit.WanDiT(cfg).init_weights(1).to(device=DEV, dtype=torch.bfloat16).eval()
    cls = type(cls_name, (processor.WanAttn_SAPAttn_Processor,), {"_seen_timesteps": set()})
    wan_dit.install_processors(model, cls, cfg.grid, num_q_centroids=4, num_k_centroids=8, top_p_kmeans=0.9, min_kc_ratio=0.2,
                               kmeans_iter_init=1, kmeans_iter_step=1, first_times_fp=0.0)
    wan_dit.set_attention_step(model, 1)
    return cfg, model


@torch.no_grad()
def test_blocks_with_token_kernels():
    """Norms alone change roundings of a block's inputs to bf16, a fraction of 2^-8 of them per norm; e4m3 linear layers are a few
    per cent off each (2^-4 at most per operand, uniform over it: 2.6 % in the 2-norm), which residual and gates dampen."""
    cfg, plain = dense_dit("Plain")
    g = torch.Generator("cpu").manual_seed(0)
    lat = torch.randn(1, 16, *cfg.latent, generator=g).bfloat16().to(DEV)
    text = torch.randn(1, 16, 64, generator=g).bfloat16().to(DEV)
    t = torch.tensor([900.0], device=DEV)
    want = plain(lat, t, text).double()
    for fp8_linears, most in ((False, 2e-2), (True, 0.1)):
        _, model = dense_dit("Kernels")
        model.use_token_kernels(fp8_linears=fp8_linears)
        got = model(lat, t, text).double()
        assert (got - want).norm() <= most * want.norm()
        assert torch.equal(got, model(lat, t, text).double())


@torch.no_grad()
def test_block_norms_are_those_of_torch():
    """The three norms of a block, on what the block hands them: scale and shift are slices of one tensor of six."""
    from svoo_b200 import wan_dit
    cfg, model = dense_dit("Norms")
    block = model.blocks[0]
    x = torch.randn(1, 77, 512, device=DEV).bfloat16()
    shift, scale = (0.3 * torch.randn(1, 6, 512, device=DEV)).chunk(6, dim=1)[3:5]
    for ln, kw in ((block.norm1, dict(scale=scale, shift=shift)), (block.norm2, {})):
        block.fused_norms = False
        want = block._norm(ln, x, **kw)
        block.fused_norms = True
        got = block._norm(ln, x, **kw)
        assert got.dtype == want.dtype
        # both are within a few 2^-22 of the value before it is rounded to bf16: at most one bf16 step apart
        assert ((got.double() - want.double()).abs() <= 2 * R.half_step(torch.bfloat16) * want.double().abs() + 1e-5).all()


@torch.no_grad()
def test_modules_follow_devices_types_and_state_dicts():
    from svoo_b200 import linear, ops
    lin = nn.Linear(200, 136).to(DEV, torch.bfloat16)
    m = linear.Fp8Linear.from_linear(lin)
    x = torch.randn(3, 7, 200, device=DEV).bfloat16()
    want = linear.linear_fp8(x, ops.quantize_blocks(lin.weight), lin.bias)
    assert torch.equal(m(x), want)
    copy = linear.Fp8Linear(200, 136, dtype=torch.bfloat16)
    copy.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()})
    assert torch.equal(copy.to(DEV)(x), want)
    assert torch.equal(m.to(torch.float16)(x).float(), want.float()) or (m(x).float() - want.float()).abs().max() < 2e-2   # the bias in fp16
    back = linear.Fp8Linear.from_linear(nn.Linear(64, 40, bias=False).to(DEV), input_grad=True)
    with torch.enable_grad():
        z = torch.randn(5, 64, device=DEV, requires_grad=True)
        back(z).sum().backward()
    w = back.weight
    dz = R.dequantize(torch.ones(5, 40, device=DEV), 1, 128) @ w.float().double()
    assert ((z.grad.double() - dz).abs() <= R.product_bound(torch.ones(5, 40, device=DEV).double(), w.float().double().t(), torch.float32, dz)).all()
    ff = nn.Sequential(nn.Linear(200, 300), nn.GELU(approximate="tanh"), nn.Linear(300, 200)).to(DEV, torch.bfloat16)
    q = linear.Fp8FeedForward.from_sequential(ff)
    assert torch.equal(q(x), linear.mlp_fp8(x, ops.quantize_blocks(ff[0].weight), ff[0].bias, ops.quantize_blocks(ff[2].weight), ff[2].bias))
    with pytest.raises(ValueError):
        linear.Fp8FeedForward.from_sequential(nn.Sequential(nn.Linear(8, 8), nn.ReLU(), nn.Linear(8, 8)))
    with pytest.raises(ValueError):
        m.set_weight(ops.quantize_blocks(torch.randn(8, 200, device=DEV)))
