"""Layer norm and its gradient on the GPU against 64-bit restatements."""
import pytest
import torch

from . import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(shape, dtype, seed, spread=2.0, centre=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    C = shape[-1]
    x = torch.randn(*shape, generator=g) * (0.5 + spread * torch.rand(C, generator=g)) + centre * torch.randn(C, generator=g)
    return x.to(dtype).to(DEV)


def params(mode, B, C, dtype, seed, p32=False):
    g = torch.Generator("cpu").manual_seed(seed)
    t = torch.float32 if p32 else dtype
    if mode == "affine":
        return dict(weight=(1 + 0.2 * torch.randn(C, generator=g)).to(t).to(DEV), bias=(0.3 * torch.randn(C, generator=g)).to(t).to(DEV))
    if mode == "modulate":
        six = (0.3 * torch.randn(B, 6, C, generator=g)).to(t).to(DEV)
        return dict(scale=six[:, 1:2], shift=six[:, 4:5])
    return {}


def gain_offset(p, x):
    one = torch.ones((), dtype=torch.float64, device=x.device)
    if "weight" in p:
        return p["weight"].double(), p["bias"].double()
    if "scale" in p:
        return 1 + p["scale"].double(), p["shift"].double()
    return one, 0 * one


def xhat_bound(x, mean, rstd, C):
    """|xhat - its value|: the mean is off by (a pairwise tree of at most 64 + 13 additions) x 2^-24 of the largest
    magnitude, x - mean by one rounding, rstd by half of the variance's relative error and three roundings."""
    top = x.double().abs().amax(-1, keepdim=True) + mean.abs()
    shift = 80 * 2.0 ** -24 * top * rstd
    xhat = ((x.double() - mean) * rstd).abs()
    return shift + (50 * 2.0 ** -24 + shift.square() + shift / C ** 0.5) * (xhat + 1) + shift * xhat


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mode,p32", [("none", False), ("affine", False), ("affine", True), ("modulate", True), ("modulate", False)])
@pytest.mark.parametrize("B,S,C", [(1, 1, 1), (1, 3, 7), (2, 5, 64), (1, 33, 514), (3, 4, 1001), (1, 70, 1536), (2, 9, 2049), (1, 6, 5120),
                                   (1, 2, 8193), (2, 2, 16384)])
def test_forward(dtype, mode, p32, B, S, C):
    from svoo_b200 import ops
    x = make((B, S, C), dtype, 1000 * C + S)
    p = params(mode, B, C, dtype, C, p32)
    y, mean, rstd = ops.layer_norm(x, eps=1e-5, return_stats=True, **p)
    g, o = gain_offset(p, x)
    want, xhat, m, r = R.layer_norm(x, g, o, 1e-5)
    tol = xhat_bound(x, m, r, C) * g.abs() + 2.0 ** -22 * (o.abs() + want.abs()) + R.half_step(dtype) * want.abs() + torch.finfo(dtype).tiny
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() - tol).max()
    assert mean.shape == (B, S) and (rstd.double() / r[..., 0] - 1).abs().max() < 1e-4
    assert torch.equal(y, ops.layer_norm(x, eps=1e-5, **p))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mode,p32", [("none", False), ("affine", False), ("affine", True), ("modulate", True), ("modulate", False)])
@pytest.mark.parametrize("B,S,C", [(1, 1, 1), (1, 3, 7), (2, 300, 64), (1, 33, 514), (3, 40, 1001), (1, 2000, 1536), (2, 9, 2049), (1, 60, 5120),
                                   (1, 2, 8193), (2, 3, 16384)])
def test_backward(dtype, mode, p32, B, S, C):
    from svoo_b200 import ops
    x, dy = make((B, S, C), dtype, 7 * C + S), make((B, S, C), dtype, 9 * C + S, 0.5, 0.1)
    p = params(mode, B, C, dtype, C, p32)
    _, mean, rstd = ops.layer_norm(x, eps=1e-5, return_stats=True, **p)
    dx, dgain, doffset = ops.layer_norm_backward(dy, x, mean, rstd, p.get("weight"), p.get("scale"))
    g, _ = gain_offset(p, x)
    want, dg_rows, do_rows = R.layer_norm_grad(x, dy, g, 1e-5)
    _, xhat, m, r = R.layer_norm(x, g, 0 * g, 1e-5)
    hb = xhat_bound(x, m, r, C)
    w = (dy.double() * g).abs()
    mean_w, mean_wh = w.mean(-1, keepdim=True), (w * xhat.abs()).mean(-1, keepdim=True)
    # every term with the error of its sums (at most 32 + 14 additions per thread and tree, 14 other roundings) and of xhat
    tol = r * (60 * 2.0 ** -24 * (w + mean_w + xhat.abs() * mean_wh) + hb * mean_wh + (xhat.abs() + hb) * (w * hb).mean(-1, keepdim=True)) \
        + (hb + 2.0 ** -20) * want.abs() + R.half_step(dtype) * want.abs() + torch.finfo(dtype).tiny
    assert ((dx.double() - want).abs() <= tol).all(), ((dx.double() - want).abs() - tol).max()
    if mode == "none":
        assert dgain is None and doffset is None
        return
    like = p.get("weight", p.get("scale"))
    dims = (0, 1) if mode == "affine" else (1,)
    n = 200                                                 # additions of one sum: rows of a CTA, then the parts
    for got, rows, err in ((dgain, dg_rows, dy.double().abs() * hb), (doffset, do_rows, 0 * dg_rows)):
        ref = rows.sum(dims).view(like.shape)
        bound = (n * 2.0 ** -24 * rows.abs().sum(dims) + err.sum(dims)).view(like.shape) + R.half_step(like.dtype) * ref.abs()
        assert got.dtype == like.dtype and got.shape == like.shape
        assert ((got.double() - ref).abs() <= bound + torch.finfo(like.dtype).tiny).all()
    again = ops.layer_norm_backward(dy, x, mean, rstd, p.get("weight"), p.get("scale"))
    assert torch.equal(dx, again[0]) and torch.equal(dgain, again[1]) and torch.equal(doffset, again[2])


def test_strided_rows_and_samples():
    """Column slices of wider rows, leading tokens of longer samples, unaligned starts, and a gradient that is expanded."""
    from svoo_b200 import ops
    wide = make((2, 50, 300), torch.bfloat16, 3)
    for x in (wide[:, :37, :256], wide[:, 5:, 3:260], wide[:, ::2, 44:172], wide[0, :, 1:2]):
        C = x.shape[-1]
        p = params("affine", 2, C, torch.bfloat16, 5)
        assert torch.equal(ops.layer_norm(x, **p), ops.layer_norm(x.contiguous(), **p))
        _, mean, rstd = ops.layer_norm(x, return_stats=True, **p)
        dy = torch.randn(1, 1, C, device=DEV).to(torch.bfloat16).expand(x.shape) if x.dim() == 3 else torch.randn(1, C, device=DEV).bfloat16().expand(x.shape)
        a = ops.layer_norm_backward(dy, x, mean, rstd, p["weight"])
        b = ops.layer_norm_backward(dy.contiguous(), x.contiguous(), mean, rstd, p["weight"])
        # the rows are taken by the same CTAs, but other widths of access put other columns on a thread
        assert all(torch.allclose(u.float(), v.float(), rtol=2 ** -7, atol=1e-3) for u, v in zip(a, b))


def test_far_mean_constant_rows_and_values_that_are_not_finite():
    from svoo_b200 import ops
    x = torch.randn(4, 1000, device=DEV) + 1000
    y = ops.layer_norm(x)
    want = R.layer_norm(x, torch.ones((), device=DEV), torch.zeros((), device=DEV), 1e-6)[0]
    assert (y - want).abs().max() < 5e-3                     # 80 x 2^-24 x 1000 = 4.8e-3 at most, by xhat_bound
    assert torch.equal(ops.layer_norm(torch.full((3, 40), 7.0, device=DEV)), torch.zeros(3, 40, device=DEV))
    x = torch.randn(5, 64, device=DEV)
    x[1, 3], x[2, 0], x[3, 63] = float("inf"), float("nan"), float("-inf")
    y = ops.layer_norm(x)
    assert torch.isnan(y[1:4]).all() and torch.isfinite(y[[0, 4]]).all()


def test_no_rows():
    from svoo_b200 import ops
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    for shape in ((0, 64), (2, 0, 64), (0, 3, 64)):
        x = torch.empty(shape, device=DEV)
        y, mean, rstd = ops.layer_norm(x, w, b, return_stats=True)
        assert y.shape == x.shape
        dx, dg, do = ops.layer_norm_backward(x, x, mean, rstd, w)
        assert dx.shape == x.shape and not dg.any() and not do.any()
    x = torch.empty(2, 0, 64, device=DEV)
    s = torch.ones(2, 1, 64, device=DEV)
    _, mean, rstd = ops.layer_norm(x, scale=s, shift=s, return_stats=True)
    _, dg, do = ops.layer_norm_backward(x, x, mean, rstd, scale=s)
    assert dg.shape == s.shape and not dg.any() and not do.any()


def test_autograd_shared_modulation_and_differences():
    """Gradients through norm.layer_norm: broadcast modulation is summed over the samples, parameters that need none get none,
    and central differences in 32 bits agree."""
    from svoo_b200 import norm
    g = torch.Generator("cpu").manual_seed(11)
    x = torch.randn(2, 3, 24, generator=g).to(DEV).requires_grad_(True)
    scale = (0.3 * torch.randn(1, 1, 24, generator=g)).to(DEV).requires_grad_(True)
    shift = (0.3 * torch.randn(1, 1, 24, generator=g)).to(DEV).requires_grad_(True)
    dy = torch.randn(2, 3, 24, generator=g).to(DEV)

    def loss(a, b, c):
        return (R.layer_norm(a, 1 + b.double(), c, 1e-6)[0] * dy.double()).sum()

    grads = torch.autograd.grad(norm.layer_norm(x, scale=scale, shift=shift), (x, scale, shift), dy)
    leaves = [t.detach().double() for t in (x, scale, shift)]
    for i, got in enumerate(grads):
        flat = leaves[i].view(-1)
        for j in range(0, flat.numel(), 5):
            h = 1e-5
            flat[j] += h
            up = loss(*leaves)
            flat[j] -= 2 * h
            down = loss(*leaves)
            flat[j] += h
            assert abs((up - down) / (2 * h) - got.view(-1)[j].double()) < 1e-4
    y = norm.layer_norm(x.detach(), scale=scale, shift=shift.detach())
    y.sum().backward()                                       # a gradient that is expanded
    assert scale.grad is not None and shift.grad is None


def test_captured_forward_and_backward():
    """Forward and backward in one graph, replayed on new inputs, give the eager bits."""
    from svoo_b200 import ops
    x, dy, w, b = (torch.randn(*s, device=DEV).bfloat16() for s in ((40, 1536), (40, 1536), (1536,), (1536,)))

    def step():
        y, mean, rstd = ops.layer_norm(x, w, b, return_stats=True)
        return (y,) + ops.layer_norm_backward(dy, x, mean, rstd, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(2):
        x.copy_(torch.randn(40, 1536, device=DEV))
        dy.copy_(torch.randn(40, 1536, device=DEV))
        graph.replay()
        assert all(torch.equal(u, v) for u, v in zip(got, step()))


def test_refusals():
    from svoo_b200 import ops
    x = torch.randn(2, 3, 64, device=DEV)
    w, s = torch.ones(64, device=DEV), torch.ones(2, 1, 64, device=DEV)
    bad = [dict(weight=w, scale=s), dict(bias=w), dict(shift=s), dict(weight=w[:32]), dict(weight=w, bias=w.bfloat16()), dict(weight=w.double()),
           dict(weight=w.half()), dict(scale=s[:, :, :32]), dict(scale=torch.ones(3, 1, 64, device=DEV)), dict(scale=torch.ones(2, 3, 64, device=DEV)),
           dict(scale=s, shift=s[:1]), dict(weight=torch.ones(128, device=DEV)[::2])]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.layer_norm(x, **kw)
    for t in (x.transpose(1, 2), x.double(), torch.empty(3, 0, device=DEV), torch.empty(1, 16385, device=DEV), x.cpu(),
              torch.randn(2, 3, 4, 8, device=DEV).transpose(0, 1)):
        with pytest.raises(ValueError):
            ops.layer_norm(t)
    y, mean, rstd = ops.layer_norm(x, return_stats=True)
    for args in ((y[:1], x, mean, rstd), (y.bfloat16(), x, mean, rstd), (y, x, mean[:1], rstd), (y, x, mean.double(), rstd)):
        with pytest.raises(ValueError):
            ops.layer_norm_backward(*args)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,C", [(310, 8200), (301, 10001), (300, 11500), (40, 12290), (299, 16383), (297, 16384)])
def test_rows_of_more_than_8192_columns(dtype, S, C):
    """More rows than there are CTAs: the walk, its one or two places in shared memory, and the sums joined behind it."""
    test_forward(dtype, "affine", True, 1, S, C)
    test_backward(dtype, "affine", False, 1, S, C)
    test_backward(dtype, "modulate", True, 2, S, C)
