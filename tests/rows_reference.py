"""Plain 64-bit restatements of the token-wise operators, for their tests."""
import torch

E4M3 = torch.float8_e4m3fn


def half_step(dtype):
    """A rounding to dtype is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def layer_norm(x, gain, offset, eps):
    """y, xhat, mean, rstd in 64 bits; gain and offset broadcast against x."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xhat = (x - mean) * rstd
    return xhat * gain.double() + offset.double(), xhat, mean, rstd


def layer_norm_grad(x, dy, gain, eps):
    """dx, and dgain and doffset of every row."""
    _, xhat, _, rstd = layer_norm(x, gain, torch.zeros((), dtype=torch.float64, device=x.device), eps)
    dy = dy.double()
    w = dy * gain.double()
    return rstd * (w - w.mean(-1, keepdim=True) - xhat * (w * xhat).mean(-1, keepdim=True)), dy * xhat, dy


def quantize(x, rows, cols):
    """(e4m3 values as fp32, scales) of x [M, K] in blocks of rows x cols, by 32-bit torch operations."""
    M, K = x.shape
    p = torch.nn.functional.pad(x.float(), (0, -K % cols, 0, -M % rows))
    b = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    amax = b.abs().amax((1, 3), keepdim=True)
    scale = (amax / torch.full_like(amax, 448.0)).clamp_min(2.0 ** -126)
    q = (b / scale).to(E4M3).float().view(p.shape)[:M, :K]
    return q, scale[:, 0, :, 0]


def dequantize(x, rows, cols):
    """The values x stands for after quantisation, in 64 bits."""
    q, s = quantize(x, rows, cols)
    return q.double() * s.double().repeat_interleave(rows, 0)[:x.shape[0]].repeat_interleave(cols, 1)[:, :x.shape[1]]


def gelu(y):
    return 0.5 * y * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3)))


def product_bound(a, b, dtype, y):
    """How far a product may be off: half a step of its type, and for every sum a step of 2^-23 of the sum of magnitudes -- 32
    products and four steps inside a block, one addition per block, two roundings of the factor and one of the bias."""
    blocks = -(-a.shape[1] // 128)
    return half_step(dtype) * y.abs() + (36 + blocks + 4) * 2.0 ** -23 * (a.abs() @ b.abs().t() + y.abs()) + torch.finfo(dtype).tiny
