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


def test_first_calls_in_a_capture_and_two_graphs_at_once():
    """Calls that were never made before capture; two graphs of the same operators replayed on two streams do not share anything."""
    from svoo_b200 import ops
    x, w, dy = (torch.randn(*s, device=DEV).half() for s in ((1000, 640), (512, 640), (1000, 512)))
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        b = ops.quantize_blocks(w, transposed=True)
        y = ops.linear_fp8(x, b, None, "gelu")
        few = ops.linear_fp8(x[:5], b)
        n, mean, rstd = ops.layer_norm(x, return_stats=True)
        dx = ops.layer_norm_backward(n, x, mean, rstd)[0]
        dw = ops.mm_fp8(ops.quantize_columns(dy), ops.quantize_columns(x))
    with torch.cuda.graph(two):
        y2 = ops.linear_fp8(x, b, None, "gelu")
        n2 = ops.layer_norm(x)
    one.replay()
    torch.cuda.synchronize()
    want = [t.clone() for t in (y, few, n, dx, dw)]
    eager = (ops.linear_fp8(x, ops.quantize_blocks(w), None, "gelu"), ops.linear_fp8(x[:5], b), ops.layer_norm(x),
             ops.layer_norm_backward(n, x, mean, rstd)[0], ops.mm_fp8(ops.quantize_columns(dy), ops.quantize_columns(x)))
    assert all(torch.equal(u, v) for u, v in zip(want, eager))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(50):
        for graph, stream in zip((one, two), streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip((y, few, n, dx, dw, y2, n2), want + [want[0], want[2]]))


def test_captured_training_step():
    from svoo_b200 import linear, norm
    x, w, b = (torch.randn(*s, device=DEV).bfloat16().requires_grad_(True) for s in ((300, 256), (384, 256), (384,)))
    dy = torch.randn(300, 384, device=DEV).bfloat16()

    def step():
        return torch.autograd.grad(linear.linear_fp8(norm.layer_norm(x), w, b), (x, w, b), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, step()))


def test_many_samples_of_one_row():
    from svoo_b200 import ops
    x, s, t = (torch.randn(3000, 1, 64, device=DEV) for _ in range(3))
    y, mean, rstd = ops.layer_norm(x, scale=s, shift=t, return_stats=True)
    want, xhat, _, _ = R.layer_norm(x, 1 + s.double(), t, 1e-6)
    assert (y.double() - want).abs().max() < 1e-4            # 80 x 2^-24 x 20 at most before the gain, by far
    _, dg, do = ops.layer_norm_backward(y, x, mean, rstd, scale=s)
    assert (dg.double() - y.double() * xhat).abs().max() < 1e-3 and torch.equal(do, y)


@torch.no_grad()
def test_token_kernels_twice():
    """A second call keeps the layers that are in e4m3; norms follow the last call."""
    cfg, model = dense_dit("Twice")
    lat = torch.randn(1, 16, *cfg.latent, device=DEV).bfloat16()
    text = torch.randn(1, 16, 64, device=DEV).bfloat16()
    t = torch.tensor([900.0], device=DEV)
    want = model.use_token_kernels()(lat, t, text)
    layer = model.blocks[0].attn1.to_q
    assert torch.equal(model.use_token_kernels()(lat, t, text), want)
    assert model.blocks[0].attn1.to_q is layer
    model.use_token_kernels(norms=False)
    assert not model.blocks[0].fused_norms and model.blocks[0].attn1.to_q is layer


def check_product(y, a, b):
    want = a @ b.t()
    assert ((y.double() - want).abs() <= R.product_bound(a, b, torch.float32, want)).all()


@torch.no_grad()
def test_offsets_beyond_32_bits():
    """Every kernel on tensors of more than 2^31 elements.  The last rows of norms and quantisers are those of a call on the last
    rows alone, bit for bit; products are checked against 64 bits."""
    from svoo_b200 import ops
    M, C, tail = 140_000, 16_384, 256                       # 140,000 is a multiple of 32, not of 128
    assert M * C > 2 ** 31
    x = torch.empty(M, C, device=DEV, dtype=torch.bfloat16).normal_()
    end = x[M - tail:].clone()
    # layer norm of the widest rows, and of the same numbers as rows of 5,120 with a pitch of 16,384
    for src in (x, x[:, 7:5127]):
        gain = torch.randn(src.shape[1], device=DEV)
        part = src[M - tail:]
        y, mean, rstd = ops.layer_norm(src, gain, gain, return_stats=True)
        y1, mean1, rstd1 = ops.layer_norm(part, gain, gain, return_stats=True)
        assert torch.equal(y[M - tail:], y1) and torch.equal(mean[M - tail:], mean1) and torch.equal(rstd[M - tail:], rstd1)
        dx = ops.layer_norm_backward(y, src, mean, rstd, gain)[0]
        assert torch.equal(dx[M - tail:], ops.layer_norm_backward(y1, part, mean1, rstd1, gain)[0])
        del y, dx
    rows, columns = ops.quantize_both(x)
    alone = ops.quantize_rows(end)
    for r in (rows, ops.quantize_rows(x)):
        assert torch.equal(r.q[M - tail:].view(torch.uint8), alone.q.view(torch.uint8)) and torch.equal(r.scale[:, M - tail:], alone.scale)
    first = M // 128 * 128                                  # the last block along the columns
    last = ops.quantize_columns(x[first:].clone())
    for c in (columns, ops.quantize_columns(x)):
        assert torch.equal(c.q[:, first:].view(torch.uint8), last.q.view(torch.uint8)) and torch.equal(c.scale[-1], last.scale[0])
    del columns, c, r
    # products: a of more than 2^31 bytes, b of as many, and a result of as many numbers
    end_d = R.dequantize(end, 1, 128)
    w, w_d = ops.quantize_blocks(x[:200].clone()), R.dequantize(x[:200], 128, 128)
    check_product(ops.mm_fp8(rows, w, out_dtype=torch.float32)[M - tail:], end_d, w_d)
    del rows
    big = ops.quantize_blocks(x, transposed=True)
    end_w, w_d = ops.quantize_blocks(x[first:].clone(), transposed=True), R.dequantize(x[first:], 128, 128)
    assert torch.equal(big.q[first:].view(torch.uint8), end_w.q.view(torch.uint8))
    assert torch.equal(big.qt[:, first:].view(torch.uint8), end_w.qt.view(torch.uint8))
    check_product(ops.linear_fp8(end[:3], big, out_dtype=torch.float32)[:, first:], end_d[:3], w_d)
    check_product(ops.mm_fp8(alone, big, out_dtype=torch.float32)[:, first:], end_d, w_d)
    del x, big
    a, b = (torch.randn(n, 130, device=DEV).bfloat16() for n in (70_001, 40_008))
    out = ops.mm_fp8(ops.quantize_rows(a), ops.quantize_blocks(b), out_dtype=torch.float32)
    assert out.numel() > 2 ** 31
    check_product(out[-177:], R.dequantize(a[-177:], 1, 128), R.dequantize(b, 128, 128))
