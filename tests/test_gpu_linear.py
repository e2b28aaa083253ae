"""Quantisers and 8-bit products on the GPU against plain torch and 64-bit restatements."""
import pytest
import torch

from . import rows_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def rand(M, K, dtype, seed, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    x = torch.randn(M, K, generator=g) * (0.3 + torch.rand(K, generator=g)) * scale
    return x.to(dtype).to(DEV)


def same_values(q, want):
    return torch.equal(q.float(), want)


@pytest.fixture(autouse=True)
def completed():
    yield
    from svoo_b200 import ops
    assert ops.linear_status(torch.device(DEV)) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 8), (5, 129), (130, 1000), (257, 777), (64, 1536), (1000, 136)])
def test_quantisers_bit_for_bit(dtype, M, K):
    from svoo_b200 import ops
    x = rand(M, K, dtype, M * 1000 + K)
    x[M // 2, : K // 2] = 0                                   # a block of zeros where K > 255
    r = ops.quantize_rows(x)
    q, s = R.quantize(x, 1, 128)
    assert torch.equal(r.scale.t(), s) and same_values(r.q, q)
    assert torch.equal(r.float(), q * s.repeat_interleave(128, 1)[:, :K])
    c, sums = ops.quantize_columns(x, torch.float32)
    q, s = R.quantize(x.t().contiguous(), 1, 128)
    assert torch.equal(c.scale.t(), s) and same_values(c.q, q)
    ref = x.double().sum(0)
    assert ((sums.double() - ref).abs() <= 40 * 2.0 ** -24 * x.double().abs().sum(0) + 1e-30).all()
    b = ops.quantize_blocks(x, transposed=True)
    q, s = R.quantize(x, 128, 128)
    assert torch.equal(b.scale, s) and same_values(b.q, q) and same_values(b.qt, q.t())
    r2, c2, sums2 = ops.quantize_both(x, torch.float32)
    for one, two in ((r, r2), (c, c2)):
        assert torch.equal(one.q.view(torch.uint8), two.q.view(torch.uint8)) and torch.equal(one.scale, two.scale)
    assert ((sums2.double() - ref).abs() <= 100 * 2.0 ** -24 * x.double().abs().sum(0) + 1e-30).all()
    # what lies behind a row is zero up to the next multiple of 16
    for t in (r.q, c.q, b.q, b.qt, r2.q, c2.q):
        whole = torch.as_strided(t.view(torch.uint8), (t.shape[0], t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16),
                                 (t.stride(0), 1))
        assert not whole[:, t.shape[1]:].any()


def test_quantisers_extreme_values():
    """Zeros, the smallest and largest numbers, and blocks with values that are not finite."""
    from svoo_b200 import ops
    x = torch.zeros(6, 256, device=DEV)
    x[1, 0], x[2, :128], x[3, 5], x[4, 200], x[5, 1] = 1e-45, 3.4e38, float("inf"), float("nan"), 448.0 * 2.0 ** -126
    r = ops.quantize_rows(x)
    q, s = R.quantize(x, 1, 128)
    for got, want in ((r.scale.t(), s), (r.q.float(), q)):
        assert torch.equal(torch.nan_to_num(got, nan=7.5, posinf=9e9), torch.nan_to_num(want.to(got.dtype), nan=7.5, posinf=9e9))
    v = r.float()
    assert torch.isnan(v[3, :128]).all() and torch.isnan(v[4, 128:]).all() and not v[0].any() and torch.isfinite(v[[0, 1, 2, 5]]).all()
    y = ops.mm_fp8(r, ops.quantize_blocks(torch.randn(40, 256, device=DEV)), None, None, torch.float32)
    assert torch.isnan(y[3:5]).all() and not y[0].any() and torch.isfinite(y[[0, 1, 5]]).all()


def test_quantise_strided():
    from svoo_b200 import ops
    wide = rand(70, 400, torch.bfloat16, 5)
    for x in (wide[:, :256], wide[:, 3:260], wide[::3, 8:136], wide[7:8, 1:2]):
        for fn in (ops.quantize_rows, ops.quantize_columns, ops.quantize_blocks, lambda t: ops.quantize_both(t)[0], lambda t: ops.quantize_both(t)[1]):
            a, b = fn(x), fn(x.contiguous())
            assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)


SIZES = [(1, 1, 1), (1, 128, 128), (2, 5, 300), (17, 40, 1000), (33, 777, 1000), (128, 256, 128), (129, 257, 129), (300, 130, 16), (64, 512, 4096),
         (333, 777, 1001), (700, 1536, 512), (2500, 300, 260)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_with_blocks(dtype, M, N, K):
    from svoo_b200 import ops
    x, w = rand(M, K, dtype, M + K), rand(N, K, dtype, N + K, 0.05)
    bias = rand(1, N, [torch.float32, dtype][M % 2], N)[0]
    a, b = ops.quantize_rows(x), ops.quantize_blocks(w)
    ad, bd = R.dequantize(x, 1, 128), R.dequantize(w, 128, 128)
    want = ad @ bd.t()
    y = ops.mm_fp8(a, b, None, None, dtype)
    assert y.dtype == dtype and ((y.double() - want).abs() <= R.product_bound(ad, bd, dtype, want)).all()
    want = want + bias.double()
    y = ops.mm_fp8(a, b, bias, None, torch.float32)
    assert ((y.double() - want).abs() <= R.product_bound(ad, bd, torch.float32, want) + 2.0 ** -23 * bias.double().abs()).all()
    y = ops.mm_fp8(a, b, bias, "gelu", dtype)
    # GELU's slope is at most 1.13; its own evaluation is off by a few 2^-21 of its argument (exponential, division)
    tol = 1.13 * R.product_bound(ad, bd, torch.float32, want) + 2.0 ** -19 * want.abs() + 2.0 ** -22 * bias.double().abs()
    g = R.gelu(want)
    assert ((y.double() - g).abs() <= tol + R.half_step(dtype) * g.abs() + torch.finfo(dtype).tiny).all()
    # quantised output: the 32-bit results, at most one e4m3 step apart where a rounding border lies between
    y32 = ops.mm_fp8(a, b, bias, "gelu", torch.float32)
    h = ops.mm_fp8(a, b, bias, "gelu", ops.E4M3)
    q, s = R.quantize(y32, 1, 128)
    assert torch.equal(h.scale.t(), s) and same_values(h.q, q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 5, 16), (2, 130, 300), (3, 777, 1001), (7, 4800, 130), (8, 33, 2048), (9, 40, 257), (15, 5000, 640), (16, 5120, 1300), (9, 64, 4100), (5, 6000, 200), (12, 2400, 600),
                                   (16, 129, 1000), (17, 129, 1000)])
def test_linear_of_few_rows(dtype, M, N, K):
    """One launch up to 16 rows: quantised, multiplied, bias and GELU; weights with bytes behind their rows, rows of a wider tensor."""
    from svoo_b200 import ops
    wide = rand(M, K + 24, dtype, M + K)
    w = rand(N, K, dtype, N + K, 0.05)
    bias = rand(1, N, [torch.float32, dtype][M % 2], N)[0]
    b = ops.quantize_blocks(w)
    if K % 16:
        torch.as_strided(b.q.view(torch.uint8), (N, -K % 16), (b.q.stride(0) if N > 1 else (K + 15) // 16 * 16, 1), K).fill_(0x7f)   # NaN
    bd = R.dequantize(w, 128, 128)
    for x in (wide[:, :K].contiguous(), wide[:, 8:K + 8], wide[:, 3:K + 3]):
        ad = R.dequantize(x.contiguous(), 1, 128)
        want = ad @ bd.t() + bias.double()
        tol = R.product_bound(ad, bd, torch.float32, want) + 2.0 ** -22 * bias.double().abs()
        y = ops.linear_fp8(x, b, bias, None, torch.float32)
        assert ((y.double() - want).abs() <= tol).all()
        y = ops.linear_fp8(x, b, None, None, torch.float32)
        plain = ad @ bd.t()
        assert ((y.double() - plain).abs() <= R.product_bound(ad, bd, torch.float32, plain)).all()
        y = ops.linear_fp8(x, b, bias, "gelu")
        g = R.gelu(want)
        assert y.dtype == dtype
        assert ((y.double() - g).abs() <= 1.13 * tol + 2.0 ** -19 * want.abs() + R.half_step(dtype) * g.abs() + torch.finfo(dtype).tiny).all()
        h, q = ops.linear_fp8(x, b, bias, None, ops.E4M3), ops.mm_fp8(ops.quantize_rows(x), b, bias, None, ops.E4M3)
        assert torch.equal(h.q.view(torch.uint8), q.q.view(torch.uint8)) and torch.equal(h.scale, q.scale)
    x = wide[:, :K].contiguous()
    x[0, K // 2] = float("nan")
    y = ops.linear_fp8(x, b, bias)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_with_rows(dtype, M, N, K):
    """Both operands with 1 x 128 scales: the gradient of a weight."""
    from svoo_b200 import ops
    x, w = rand(M, K, dtype, M + K), rand(N, K, dtype, N + K, 0.05)
    a = ops.quantize_rows(x)
    b = ops.quantize_columns(w.t().contiguous())
    ad, bd = R.dequantize(x, 1, 128), R.dequantize(w, 1, 128)
    want = ad @ bd.t()
    y = ops.mm_fp8(a, b, None, None, dtype)
    assert ((y.double() - want).abs() <= R.product_bound(ad, bd, dtype, want)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,bias", [(1, 1, 1, True), (5, 130, 260, True), (200, 384, 500, False), (400, 256, 1000, True)])
def test_linear_with_gradients(dtype, M, N, K, bias):
    from svoo_b200 import linear
    x, w, dy = rand(M, K, dtype, 1), rand(N, K, dtype, 2, 0.05), rand(M, N, dtype, 3, 0.01)
    b = rand(1, N, dtype, 4)[0] if bias else None
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = linear.linear_fp8(x.view(1, M, K), w, b)
    assert y.shape == (1, M, N)
    grads = torch.autograd.grad(y, leaves, dy.view(1, M, N))
    x, w, b = (None if t is None else t.detach() for t in (x, w, b))
    for got, u, v in ((y[0], R.dequantize(x, 1, 128), R.dequantize(w, 128, 128)),
                      (grads[0], R.dequantize(dy, 1, 128), R.dequantize(w, 128, 128).t()),
                      (grads[1], R.dequantize(dy.t().contiguous(), 1, 128), R.dequantize(x.t().contiguous(), 1, 128))):
        want = u @ v.t()
        tol = R.product_bound(u, v, dtype, want)
        if got is y[0] or got.shape == (M, N) and got.data_ptr() == y.data_ptr():
            want = want + (0 if b is None else b.double())
            tol = R.product_bound(u, v, dtype, want) + (0 if b is None else 2.0 ** -23 * b.double().abs())
        assert got.dtype == dtype and ((got.double() - want).abs() <= tol).all()
    if bias:
        ref = dy.double().sum(0)
        assert ((grads[2].double() - ref).abs() <= 64 * 2.0 ** -24 * dy.double().abs().sum(0) + R.half_step(dtype) * ref.abs()
                + torch.finfo(dtype).tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (70, 130, 260), (300, 200, 129)])
def test_training_calls_are_the_separate_calls(dtype, M, N, K):
    """Bit for bit, for every subset of gradients, with rows of wider tensors."""
    from svoo_b200 import linear, ops
    x, w, g = rand(M, K + 5, dtype, 1)[:, 5:], rand(N, K + 3, dtype, 2, 0.05)[:, :K], rand(M, N + 1, dtype, 3)[:, 1:]
    b = rand(1, N, torch.float32, 4)[0]
    y, saved = ops.linear_train_forward(x, w, b)
    q = ops.quantize_blocks(w, transposed=True)
    assert torch.equal(y, ops.mm_fp8(ops.quantize_rows(x), q, b, None, dtype))
    dx, dw, db = ops.linear_train_backward(g, saved, K, w_dtype=torch.float32, bias_dtype=torch.float32)
    assert torch.equal(dx, ops.mm_fp8(ops.quantize_rows(g), q.transposed(), None, None, dtype))
    gt, sums = ops.quantize_columns(g, torch.float32)
    dw_t = ops.mm_fp8(gt, ops.quantize_columns(x), None, None, dtype)
    assert torch.equal(dw, ops.mm_fp8(gt, ops.quantize_columns(x), None, None, torch.float32)) and torch.equal(db, sums)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 0, 1), (0, 1, 1)):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
        got = torch.autograd.grad(linear.linear_fp8(*leaves), [t for t, n in zip(leaves, need) if n], g)
        for t, ref in zip(got, [r for r, n in zip((dx, dw_t, db), need) if n]):
            assert torch.equal(t, ref)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    part, = torch.autograd.grad(linear.linear_fp8(*leaves), leaves[1:2], g)              # kept for all, asked for one
    assert torch.equal(part, dw_t)
    for bad in (dict(saved=saved[:-1]), dict(K=K + 1), dict(keep_w_grad=False, w_dtype=torch.float32), dict(w_dtype=torch.float64)):
        kw = dict(dict(saved=saved, K=K), **bad)
        if kw["K"] == K + 1 and kw["saved"].shape[0] == ops._train_bytes(M, N, K + 1, True, True)[0]:
            continue
        with pytest.raises(ValueError):
            ops.linear_train_backward(g, **kw)
    with pytest.raises(ValueError):
        ops.linear_train_forward(x, w[:, 1:], b)
    with pytest.raises(ValueError):
        ops.linear_train_forward(x[:0], w, b)


def test_gradients_are_those_of_a_linear_layer():
    """Against the unquantised layer: e4m3 rounds each operand by up to 2^-4, about 2.6 % of its norm, so a product of two
    is within 5 % of the true one in the 2-norm."""
    from svoo_b200 import linear, ops
    x, w, b, dy = rand(500, 640, torch.bfloat16, 1), rand(384, 640, torch.bfloat16, 2, 0.05), rand(1, 384, torch.bfloat16, 3)[0], rand(500, 384, torch.bfloat16, 4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(linear.linear_fp8(x, w, b), leaves, dy)
    want = torch.autograd.grad(torch.nn.functional.linear(x.double(), w.double(), b.double()), leaves, dy.double())
    for u, v in zip(got, want):
        assert (u.double() - v.double()).norm() <= 0.05 * v.double().norm()
    # a stored weight is a constant: the gradient of x alone, through its transpose
    stored = ops.quantize_blocks(w.detach(), transposed=True)
    dx, = torch.autograd.grad(linear.linear_fp8(x, stored, b.detach()), (x,), dy)
    assert torch.equal(dx, got[0])
    with pytest.raises(ValueError):
        linear.linear_fp8(x, ops.quantize_blocks(w.detach()), b.detach())


@pytest.mark.parametrize("M,K,F", [(1, 64, 300), (50, 200, 1000), (300, 512, 1024)])
@pytest.mark.parametrize("dtype", TYPES)
def test_mlp(dtype, M, K, F):
    """norm -> linear -> gelu -> linear as a block runs them, against the same chain in 64 bits on what the kernels quantised."""
    from svoo_b200 import linear, ops
    x = ops.layer_norm(rand(M, K, dtype, 1))
    w1, w2 = ops.quantize_blocks(rand(F, K, dtype, 2, 0.05)), ops.quantize_blocks(rand(K, F, dtype, 3, 0.05))
    b1, b2 = rand(1, F, dtype, 4)[0], rand(1, K, dtype, 5)[0]
    y = linear.mlp_fp8(x, w1, b1, w2, b2)
    h = ops.mm_fp8(ops.quantize_rows(x), w1, b1, "gelu", ops.E4M3)
    u, v = h.float().double(), w2.float().double()
    want = u @ v.t() + b2.double()
    assert y.dtype == dtype and ((y.double() - want).abs() <= R.product_bound(u, v, dtype, want) + 2.0 ** -22 * b2.double().abs()).all()


def test_no_rows_and_leading_dimensions():
    from svoo_b200 import linear, ops
    w = torch.randn(40, 64, device=DEV, requires_grad=True)
    b = torch.zeros(40, device=DEV, requires_grad=True)
    x = torch.empty(2, 0, 64, device=DEV, requires_grad=True)
    y = linear.linear_fp8(x, w, b)
    assert y.shape == (2, 0, 40)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert dx.shape == x.shape and not dw.any() and not db.any()
    s = ops.quantize_blocks(w.detach())
    x = torch.randn(3, 5, 64, device=DEV)
    assert torch.equal(linear.linear_fp8(x, s), linear.linear_fp8(x.view(15, 64), s).view(3, 5, 40))
    assert torch.equal(linear.linear_fp8(x.transpose(0, 1), s), linear.linear_fp8(x.transpose(0, 1).contiguous(), s))
    assert linear.linear_fp8(x[0, 0], s).shape == (40,)


def test_captured_and_on_two_streams():
    """A captured training step replays to the eager bits; two streams at once do not disturb one another."""
    from svoo_b200 import linear, ops
    x, w, dy = rand(300, 512, torch.bfloat16, 1), rand(384, 512, torch.bfloat16, 2, 0.05), rand(300, 384, torch.bfloat16, 3)
    s = ops.quantize_blocks(w)

    def step():
        a = ops.quantize_rows(x)
        return linear.linear_fp8(x, s), ops.mm_fp8(ops.quantize_columns(dy), ops.quantize_columns(x), None, None, torch.float32), a.q

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(rand(300, 512, torch.bfloat16, 9))
    graph.replay()
    want = step()
    assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(got, want))
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                results[i].append(step())
    torch.cuda.synchronize()
    for r in results[0] + results[1]:
        assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(r, want))


def test_refusals():
    from svoo_b200 import linear, ops
    x, w = torch.randn(8, 64, device=DEV), torch.randn(40, 64, device=DEV)
    a, b = ops.quantize_rows(x), ops.quantize_blocks(w)
    for fn in (ops.quantize_rows, ops.quantize_columns, ops.quantize_blocks, ops.quantize_both):
        for t in (x.double(), x.t(), x[None], x.cpu(), x[:, :0]):
            with pytest.raises(ValueError):
                fn(t)
    for args in ((a, ops.quantize_blocks(w[:, :32])), (a, b, w[0]), (a, b, torch.zeros(80, device=DEV)[::2]), (a, b, None, "relu"),
                 (a, b, None, None, torch.float64), (a, ops.quantize_columns(w.t().contiguous()), None, "gelu"),
                 (a, ops.quantize_columns(w.t().contiguous()), None, None, ops.E4M3), (a, ops.Fp8Blocks(b.q, b.scale.double())),
                 (a, ops.Fp8Blocks(b.q, b.scale[:, :0])), (ops.Fp8Rows(a.q.float(), a.scale), b), (a, ops.Fp8Blocks(b.q.t(), b.scale)),
                 (ops.Fp8Rows(torch.empty(8, 72, device=DEV).to(ops.E4M3)[:, 4:68], a.scale), b), (a, b, torch.zeros(40))):
        with pytest.raises(ValueError):
            ops.mm_fp8(*args)
    with pytest.raises(ValueError):
        b.transposed()
    with pytest.raises(ValueError):
        linear.linear_fp8(x.requires_grad_(True), w, None, "gelu")
    with pytest.raises(ValueError):
        linear.mlp_fp8(x, b, None, b, None)
