"""The token-wise operators of a DiT block and their plain forms: layer norm (affine or AdaLN-modulated) with its gradient,
and linear layers in 8-bit floating point (e4m3, one scale per block of 128) with theirs.

A case is a dict of plain values.  `op` names the operator:

  norm          y = layer_norm(x) * gain + offset        gain, offset: weight, bias [C] or 1 + scale, shift [B, 1, C]
  norm_train    the same, and the gradients of x, gain and offset
  linear        y = x W^T + b, W held in e4m3 with one scale per 128 x 128 block, x quantised in the call, 1 x 128 blocks
  mlp           linear(quantise(gelu(linear(x)))), the hidden rows quantised from their 32-bit values
  linear_train  y = x W^T + b with W quantised in the call too, and the gradients of x, W and b: the gradient of y is quantised in
                blocks of 128 along what each product sums over, as x and W are
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
TINY = 2.0 ** -126          # the smallest scale: a block of zeros has it
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the text tokens of one prompt before the cross attention: latency
        dict(name="norm-512x1536", op="norm", mode="affine", batch=1, rows=512, cols=1536, dtype="bf16"),
        # AdaLN of every block at 480p, scale and shift in 32 bits and a slice of the six that the time embedding gives
        dict(name="modulate-32760x1536", op="norm", mode="modulate", batch=1, rows=32760, cols=1536, dtype="bf16"),
        # the same at 720p with 40 heads: the largest
        dict(name="modulate-75600x5120", op="norm", mode="modulate", batch=1, rows=75600, cols=5120, dtype="bf16"),
        # fine-tuning: the affine norm before the cross attention, forward and backward
        dict(name="norm-train-32760x1536", op="norm_train", mode="affine", batch=1, rows=32760, cols=1536, dtype="bf16"),
        # odd sizes, two samples with modulations of their own, 32 bits
        dict(name="modulate-train-2x4097x1001", op="norm_train", mode="modulate", batch=2, rows=4097, cols=1001, dtype="fp32"),
        # one row: the projections of a time embedding or of a pooled prompt
        dict(name="linear-1x5120x5120", op="linear", rows=1, n=5120, k=5120, bias=True, dtype="bf16"),
        # the projection of the text tokens into the model's width
        dict(name="linear-512x1536x4096", op="linear", rows=512, n=1536, k=4096, bias=True, dtype="bf16"),
        # ragged in every direction, half precision, no bias
        dict(name="linear-333x777x1000", op="linear", rows=333, n=777, k=1000, bias=False, dtype="fp16"),
        # Q, K, V and output projections at 480p and at 720p with 40 heads
        dict(name="linear-32760x1536x1536", op="linear", rows=32760, n=1536, k=1536, bias=True, dtype="bf16"),
        dict(name="linear-75600x5120x5120", op="linear", rows=75600, n=5120, k=5120, bias=True, dtype="bf16"),
        # the feed-forward of a block at 480p
        dict(name="mlp-32760x1536x8960", op="mlp", rows=32760, n=8960, k=1536, bias=True, dtype="bf16"),
        # fine-tuning a projection of it
        dict(name="linear-train-8190x8960x1536", op="linear_train", rows=8190, n=8960, k=1536, bias=True, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm; one in two is a multiple of 16."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v = (v + 8) // 16 * 16
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_train", "linear", "linear", "mlp", "linear_train"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"]) if op.startswith("norm") else rng.choice(["bf16", "bf16", "fp16"])
    if op.startswith("norm"):
        batch, cols = rng.randint(1, 4), _spread(rng, 64, 8192)
        rows = _spread(rng, 1, max(1, min(75600, 100_000_000 // (cols * batch))))
        return dict(op=op, mode=rng.choice(["affine", "modulate"]), batch=batch, rows=rows, cols=cols, dtype=dtype)
    n, k = _spread(rng, 128, 8960), _spread(rng, 128, 8960)
    most = {"linear": 1.5e12, "mlp": 0.6e12, "linear_train": 0.3e12}[op] / (2 * n * k)
    rows = _spread(rng, 1, int(max(1, min(32760, most))))
    return dict(op=op, rows=rows, n=n, k=k, bias=rng.random() < 0.5, dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"].startswith("norm"):
        B, S, C = case["batch"], case["rows"], case["cols"]
        # a residual stream: every channel with a mean and a spread of its own
        x = (randn(B, S, C) * (0.5 + randn(C).abs()) + randn(C)).to(dt)
        s = {"op": case["op"], "x": x, "eps": 1e-6, "weight": None, "bias": None, "scale": None, "shift": None}
        if case["mode"] == "affine":
            s["weight"], s["bias"] = (1 + 0.1 * randn(C)).to(dt), (0.1 * randn(C)).to(dt)
        else:
            six = 0.3 * randn(B, 6, C)
            s["shift"], s["scale"] = six.chunk(6, dim=1)[:2]
        if case["op"] == "norm_train":
            s["dy"] = randn(B, S, C).to(dt)
        return s

    M, N, K = case["rows"], case["n"], case["k"]
    s = {"op": case["op"], "x": (randn(M, K) * (0.5 + randn(K).abs())).to(dt)}
    if case["op"] == "linear_train":
        s["x"].requires_grad_(True)
        s["weight"] = (0.02 * randn(N, K)).to(dt).requires_grad_(True)
        s["bias"] = (0.1 * randn(N)).to(dt).requires_grad_(True) if case["bias"] else None
        s["dy"] = (0.01 * randn(M, N)).to(dt)
        return s
    s["w_q"], s["w_scale"] = _stored_weight(0.02 * randn(N, K))
    s["bias"] = (0.1 * randn(N)).to(dt) if case["bias"] else None
    if case["op"] == "mlp":
        s["w2_q"], s["w2_scale"] = _stored_weight(0.02 * randn(K, N))
        s["bias2"] = (0.1 * randn(K)).to(dt) if case["bias"] else None
    return s


def run(state):
    op = state["op"]
    if own:
        from svoo_b200 import linear, ops
        if op == "norm":
            return ops.layer_norm(state["x"], state["weight"], state["bias"], state["scale"], state["shift"], state["eps"])
        if op == "norm_train":
            y, mean, rstd = ops.layer_norm(state["x"], state["weight"], state["bias"], state["scale"], state["shift"], state["eps"],
                                           return_stats=True)
            dx, dgain, doffset = ops.layer_norm_backward(state["dy"], state["x"], mean, rstd, state["weight"], state["scale"])
            return {"y": y, "dx": dx, "dgain": dgain, "doffset": doffset}
        if op == "linear":
            return linear.linear_fp8(state["x"], linear.Fp8Weight(state["w_q"], state["w_scale"]), state["bias"])
        if op == "mlp":
            return linear.mlp_fp8(state["x"], linear.Fp8Weight(state["w_q"], state["w_scale"]), state["bias"],
                                  linear.Fp8Weight(state["w2_q"], state["w2_scale"]), state["bias2"])
        y = linear.linear_fp8(state["x"], state["weight"], state["bias"])
        leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
    if op == "norm":
        return _plain_norm(state)[0]
    if op == "norm_train":
        return _plain_norm_train(state)
    with torch.no_grad():
        dt, x = state["x"].dtype, state["x"].float()
        if op == "linear_train":
            return _plain_linear_train(state, x, dt)
        y = _along_rows(x) @ _read_weight(state["w_q"], state["w_scale"]).t()
        y = y if state["bias"] is None else y + state["bias"].float()
        if op == "mlp":
            h = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
            y = _along_rows(h) @ _read_weight(state["w2_q"], state["w2_scale"]).t()
            y = y if state["bias2"] is None else y + state["bias2"].float()
        return y.to(dt)


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + s["eps"])
    gain = s["weight"].float() if s["weight"] is not None else 1.0 + s["scale"].float()
    offset = s["bias"].float() if s["weight"] is not None else s["shift"].float()
    xhat = d * rstd
    return (xhat * gain + offset).to(s["x"].dtype), xhat, rstd, gain


def _plain_norm_train(s):
    y, xhat, rstd, gain = _plain_norm(s)
    dy = s["dy"].float()
    w = dy * gain
    dx = (w - w.mean(-1, keepdim=True) - xhat * (w * xhat).mean(-1, keepdim=True)) * rstd
    affine = s["weight"] is not None
    dims = (0, 1) if affine else (1,)
    kind = s["weight"].dtype if affine else s["scale"].dtype
    return {"y": y, "dx": dx.to(s["x"].dtype), "dgain": (dy * xhat).sum(dims, keepdim=not affine).to(kind),
            "doffset": dy.sum(dims, keepdim=not affine).to(kind)}


def _e4m3(blocks, amax):
    """Values of `blocks` in e4m3 and the scale of each block, whose largest magnitude `amax` broadcasts."""
    scale = (amax / torch.full_like(amax, E4M3_MAX)).clamp_min(TINY)      # a quotient, not a product with 1 / 448
    return (blocks / scale).to(torch.float8_e4m3fn), scale


def _padded(x, rows):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 128, 0, -x.shape[0] % rows))


def _along_rows(x):
    """x [R, C] quantised in blocks of 1 x 128, as the values it then stands for."""
    R, C = x.shape
    b = _padded(x, 1).view(R, -1, 128)
    q, scale = _e4m3(b, b.abs().amax(-1, keepdim=True))
    return (q.float() * scale).view(R, -1)[:, :C]


def _square_blocks(w):
    """w [N, K] in e4m3 and its scales [ceil(N / 128), ceil(K / 128)]."""
    N, K = w.shape
    p = _padded(w, 128)
    b = p.view(p.shape[0] // 128, 128, -1, 128)
    q, scale = _e4m3(b, b.abs().amax((1, 3), keepdim=True))
    return q.view(p.shape)[:N, :K], scale[:, 0, :, 0].contiguous()


def _stored_weight(w):
    """The same with rows a multiple of 16 bytes apart, as a program keeps it."""
    N, K = w.shape
    q, scale = _square_blocks(w)
    kept = torch.zeros(N, -(-K // 16) * 16, dtype=torch.float8_e4m3fn, device=w.device)
    kept[:, :K] = q
    return kept[:, :K], scale


def _read_weight(q, scale):
    N, K = q.shape
    return q.float() * scale.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def _plain_linear_train(s, x, dt):
    dy = s["dy"].float()
    w = _read_weight(*_square_blocks(s["weight"].float()))
    y = _along_rows(x) @ w.t()
    y = y if s["bias"] is None else y + s["bias"].float()
    dx = _along_rows(dy) @ w
    dw = _along_rows(dy.t().contiguous()) @ _along_rows(x.t().contiguous()).t()
    grads = [dx.to(dt), dw.to(dt)] + ([] if s["bias"] is None else [dy.sum(0).to(dt)])
    return [y.to(dt), *grads]


# ---- what the operators are, in 64 bits ------------------------------------------------------------------------------

def _rounded_e4m3(v):
    """v to the nearest value of e4m3, ties to even: steps of 2^-3 of the binade, of 2^-9 below 2^-6."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _exact_blocks(x, height):
    """x in 64 bits as its blocks of height x 128 in e4m3 stand for it; scales and quotients are 32-bit numbers."""
    R, C = x.shape
    rb, cb = -(-R // height), -(-C // 128)
    big = x.new_zeros(rb * height, cb * 128)
    big[:R, :C] = x
    b = big.reshape(rb, height, cb, 128).transpose(1, 2)
    top = b.abs().flatten(2).max(-1).values[:, :, None, None]
    scale = torch.clamp((top / 448).float().double(), min=2.0 ** -126)
    b = _rounded_e4m3((b / scale).float().double()) * scale
    return b.transpose(1, 2).reshape(rb * height, cb * 128)[:R, :C]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    x = s["x"].detach().double()
    if op.startswith("norm"):
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        sd = (var + s["eps"]).sqrt()
        z = (x - mean) / sd
        a, b = (s["weight"], s["bias"]) if case["mode"] == "affine" else (1 + s["scale"].double(), s["shift"])
        a, b = a.double(), b.double()
        y = z * a + b
        if op == "norm":
            return y
        dy = s["dy"].double()
        u = dy * a
        n = x.shape[-1]
        dx = (n * u - u.sum(-1, keepdim=True) - z * (u * z).sum(-1, keepdim=True)) / (n * sd)
        if case["mode"] == "affine":
            return {"y": y, "dx": dx, "dgain": torch.einsum("bsc,bsc->c", dy, z), "doffset": torch.einsum("bsc->c", dy)}
        return {"y": y, "dx": dx, "dgain": torch.einsum("bsc,bsc->bc", dy, z)[:, None], "doffset": torch.einsum("bsc->bc", dy)[:, None]}
    bias = 0.0 if s["bias"] is None else s["bias"].detach().double()
    if op == "linear_train":
        w, dy = _exact_blocks(s["weight"].detach().double(), 128), s["dy"].double()
        y = torch.einsum("mk,nk->mn", _exact_blocks(x, 1), w) + bias
        dx = torch.einsum("mn,nk->mk", _exact_blocks(dy, 1), w)
        dw = torch.einsum("nm,km->nk", _exact_blocks(dy.t(), 1), _exact_blocks(x.t(), 1))
        return [y, dx, dw] + ([] if s["bias"] is None else [dy.sum(0)])
    wide = [torch.kron(t.double(), torch.ones(128, 128, dtype=torch.float64, device=DEV)) for t in [s["w_scale"], s.get("w2_scale")] if t is not None]
    w = s["w_q"].double() * wide[0][: case["n"], : case["k"]]
    y = torch.einsum("mk,nk->mn", _exact_blocks(x, 1), w) + bias
    if op == "mlp":
        t = math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)
        h = y * torch.special.expit(2 * t)
        w2 = s["w2_q"].double() * wide[1][: case["k"], : case["n"]]
        y = torch.einsum("mn,kn->mk", _exact_blocks(h.float().double(), 1), w2)
        y = y if s["bias2"] is None else y + s["bias2"].double()
    return y


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"].startswith("norm"):
        cells = case["batch"] * case["rows"] * case["cols"]
        train = case["op"] == "norm_train"
        params = case["cols"] * (2 * e if case["mode"] == "affine" else 8 * case["batch"])
        return {"bytes": cells * e * (4 if train else 2) + params * (2 if train else 1), "flops": cells * (20 if train else 8)}
    M, N, K = case["rows"], case["n"], case["k"]
    b = N * e if case["bias"] else 0
    if case["op"] == "linear":
        return {"bytes": M * K * e + N * K + M * N * e + b, "flops": 2 * M * N * K}
    if case["op"] == "mlp":
        return {"bytes": 2 * M * K * e + 2 * N * K + b + (K * e if case["bias"] else 0), "flops": 4 * M * N * K}
    # x, W, dy in; y, dx, dW, db out
    return {"bytes": 2 * (M * K + N * K + M * N) * e + 2 * b, "flops": 6 * M * N * K}
