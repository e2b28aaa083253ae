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


@pytest.mark.parametrize("xt,wt,bt", [(torch.bfloat16, torch.float32, torch.float16), (torch.float16, torch.bfloat16, torch.float32),
                                      (torch.float32, torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("M,N,K", [(40, 72, 200), (9000, 777, 130)])
def test_training_with_types_of_their_own(M, N, K, xt, wt, bt):
    """Input, weight and bias of three types: every gradient is of its tensor's type, and the weight's or the bias's may be asked for alone."""
    from svoo_b200 import linear
    x, w, b = rand(M, K, xt, 1), rand(N, K, wt, 2, 0.05), rand(1, N, bt, 3)[0]
    dy = rand(M, N, xt, 4, 0.01)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear.linear_fp8(x, w, b)
    grads = torch.autograd.grad(y, leaves, dy)
    assert y.dtype == xt and [g.dtype for g in grads] == [xt, wt, bt]
    x, w, b = (t.detach() for t in leaves)
    for got, u, v, add in ((y.detach(), R.dequantize(x, 1, 128), R.dequantize(w, 128, 128), b.double()),
                           (grads[0], R.dequantize(dy, 1, 128), R.dequantize(w, 128, 128).t(), torch.zeros((), device=DEV)),
                           (grads[1], R.dequantize(dy.t().contiguous(), 1, 128), R.dequantize(x.t().contiguous(), 1, 128), torch.zeros((), device=DEV))):
        want = u @ v.t() + add
        assert ((got.double() - want).abs() <= R.product_bound(u, v, got.dtype, want) + 2.0 ** -22 * add.abs()).all()
    for i in (1, 2):
        assert torch.equal(torch.autograd.grad(linear.linear_fp8(*leaves), leaves[i:i + 1], dy)[0], grads[i])


def test_one_tensor_in_two_places():
    """x as its own weight: both gradients add up; scale and shift of a norm from one leaf as well."""
    from svoo_b200 import linear, norm
    x = rand(300, 200, torch.float32, 5).requires_grad_(True)
    u = x.detach().clone().requires_grad_(True)
    dy = rand(300, 300, torch.float32, 6)
    both, = torch.autograd.grad(linear.linear_fp8(x, x), (x,), dy)
    one, two = torch.autograd.grad(linear.linear_fp8(x, u), (x, u), dy)
    assert torch.equal(both, one + two)
    s = rand(2, 64, torch.float32, 7).requires_grad_(True)
    z, dz = rand(20, 64, torch.float32, 8).view(2, 10, 64), rand(20, 64, torch.float32, 9).view(2, 10, 64)
    t = s.detach().clone().requires_grad_(True)
    both, = torch.autograd.grad(norm.layer_norm(z, scale=s, shift=s), (s,), dz)
    one, two = torch.autograd.grad(norm.layer_norm(z, scale=s, shift=t), (s, t), dz)
    assert torch.equal(both, one + two)


def test_walking_products_on_two_streams_and_in_a_graph():
    """A training step whose products walk, eagerly on two streams at once and replayed: the same bits."""
    from svoo_b200 import linear
    x, w, b = (t.requires_grad_(True) for t in (rand(5200, 1300, torch.bfloat16, 1), rand(2310, 1300, torch.bfloat16, 2, 0.05), rand(1, 2310, torch.bfloat16, 3)[0]))
    dy = rand(5200, 2310, torch.bfloat16, 4, 0.01)

    def step():
        y = linear.linear_fp8(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                results.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for r in results for u, v in zip(r, want))


@pytest.mark.parametrize("M,N", [(5, 300), (40, 300), (9600, 300)])
@pytest.mark.parametrize("K", [1, 130, 200, 250])
def test_operands_that_are_slices(M, N, K):
    """The leading columns of wider operands, whose bytes behind the row are not zeros, rows from the middle, and rows of blocks."""
    from svoo_b200 import ops
    x, w = rand(M + 8, 256, torch.float32, M), rand(N + 256, 256, torch.float32, N, 0.05)
    a, b, t = ops.quantize_rows(x), ops.quantize_blocks(w), ops.quantize_rows(w)
    kb = -(-K // 128)
    ad = R.dequantize(x, 1, 128)[5:M + 5, :K]
    a = ops.Fp8Rows(a.q[5:M + 5, :K], a.scale[:kb, 5:M + 5])
    n = slice(128, 128 + N)
    bd = R.dequantize(w, 128, 128)[n, :K]
    y = ops.mm_fp8(a, ops.Fp8Blocks(b.q[n, :K], b.scale[1:1 + -(-N // 128), :kb]), None, None, torch.float32)
    want = ad @ bd.t()
    assert ((y.double() - want).abs() <= R.product_bound(ad, bd, torch.float32, want)).all()
    y = ops.linear_fp8(x[5:M + 5, :K], ops.Fp8Blocks(b.q[n, :K], b.scale[1:1 + -(-N // 128), :kb]))
    u = R.dequantize(x[5:M + 5, :K], 1, 128)
    want = u @ bd.t()
    assert ((y.double() - want).abs() <= R.product_bound(u, bd, torch.float32, want)).all()
    bd = R.dequantize(w, 1, 128)[n, :K]
    y = ops.mm_fp8(a, ops.Fp8Rows(t.q[n, :K], t.scale[:kb, n]), None, None, torch.float32)
    want = ad @ bd.t()
    assert ((y.double() - want).abs() <= R.product_bound(ad, bd, torch.float32, want)).all()
