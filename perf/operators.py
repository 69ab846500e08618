"""The 8-bit activation path of a Linear layer: its operators in plain form, and the calls of the
framework that compute the same.

An activation matrix X [M, K] is held as int8 numbers q and one fp32 scale per row (token):
X ~ q * scale. Two operators make that form and two read it:

  quantize  q = round(127 x / A), scale = A / 127, A = max_k |x| of the row      (saving a checkpoint)
  norm      h = x + residual; y = h * rstd * w, rstd = 1 / sqrt(mean(h^2) + eps); y in int8 form
  linear    Y = max((q_x q_w^T) * (scale_x scale_w) + b, 0) and its ReLU mask       (int8 products)
  dw        dW = dZ^T (q_x * scale_x): the weight gradient from the 8-bit checkpoint of X

and `norm_bwd` is the gradient of the norm (the rounding to int8 counts as the identity):
dx = rstd (w dy - xhat mean(w dy xhat)) + dh, dw = sum over rows of dy xhat, xhat = h rstd.

Roundings that are part of the operators' definitions: h is rounded to its type and everything
after uses the rounded h; a = fl32(h * w); q is the integer nearest to the real number 127 a / A
(ties to even) with A = max |a|, on which rstd has no influence; the linear's result is
z = fl32(fl32(fl32(acc) * fl32(scale_x scale_w)) + b) with acc the exact integer sum. So the int8
numbers and the mask words are the same from any correct implementation, and they are returned as
the whole numbers they are, with the scales beside them.
"""
import math

import torch

own = False

EPS = 1e-6
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a serving loop: the norm before a 4096-wide layer, and that layer
        dict(name="norm_token", op="norm", m=1, k=4096, dtype="bf16", residual=True),
        dict(name="linear_token", op="linear", m=1, n=4096, k=4096, relu=False, bias=True, out="bf16"),
        # a few tokens (a small batch of sequences, one token each)
        dict(name="linear_few", op="linear", m=40, n=4096, k=4096, relu=True, bias=True, out="bf16"),
        # sizes that divide by nothing
        dict(name="linear_ragged", op="linear", m=1000, n=1397, k=777, relu=False, bias=False, out="fp32"),
        dict(name="norm_bwd_ragged", op="norm_bwd", m=333, k=1416, dtype="fp32", dh=False),
        # the first layer of the MLP training step (batch 128, 784 -> 256)
        dict(name="quantize_mlp", op="quantize", m=128, k=784, dtype="fp32"),
        dict(name="dw_mlp", op="dw", m=128, n=256, k=784),
        # the forward benchmark's layer (8192 rows, 4096 x 4096) with its mask kept for training
        dict(name="linear_batch", op="linear", m=8192, n=4096, k=4096, relu=True, bias=True, out="bf16"),
        # the training step's batch (16384 rows, 4096 x 4096)
        dict(name="norm_batch", op="norm", m=16384, k=4096, dtype="bf16", residual=True),
        dict(name="quantize_batch", op="quantize", m=16384, k=4096, dtype="bf16"),
        dict(name="norm_bwd_batch", op="norm_bwd", m=16384, k=4096, dtype="bf16", dh=True),
        dict(name="dw_batch", op="dw", m=16384, n=4096, k=4096),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "norm", "norm_bwd", "linear", "linear", "dw"])
    k = _log(rng, 16, 12288)
    if rng.random() < 0.5:
        k = max(16, k // 16 * 16)  # half of the widths are the multiples of 16 that layers have
    m = _log(rng, 1, 16384)
    if op in ("quantize", "norm", "norm_bwd"):
        m = min(m, 16384 * 4096 // k)
        c = dict(op=op, m=m, k=k, dtype=rng.choice(["bf16", "bf16", "fp32"]))
        if c["dtype"] == "fp32":
            c["m"] = max(1, m // 2)
        if op == "norm":
            c["residual"] = rng.random() < 0.7
        if op == "norm_bwd":
            c["dh"] = rng.random() < 0.7
        return c
    n = _log(rng, 16, 12288)
    if op == "linear":
        m = max(1, min(m, 8192 * 4096 * 4096 // (n * k)))
        relu = rng.random() < 0.5
        return dict(op=op, m=m, n=n, k=k, relu=relu, bias=relu or rng.random() < 0.5,
                    out=rng.choice(["bf16", "bf16", "fp32"]))
    n = n // 8 * 8  # rows of dZ start on 16 bytes
    m = max(1, min(m, 16384 * 4096 * 4096 // (n * k)))
    return dict(op=op, m=m, n=n, k=k)


# ------------------------------------------------------------------------------------ inputs
def _rows16(q):
    """An int8 matrix whose rows start on 16 bytes, as the quantising calls lay it out."""
    m, k = q.shape
    buf = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.int8, device=q.device)
    buf[:, :k] = q
    return buf[:, :k]


def _to_int8(x):
    a = x.float().abs().amax(1)
    s = a / 127
    q = torch.round(x.float() / s.clamp_min(1e-30)[:, None]).clamp_(-127, 127).to(torch.int8)
    return _rows16(q), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    c = case

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    def activations(m, k):
        # channels of different sizes, a few of them large, as in a residual stream
        x = randn(m, k) * torch.exp(0.5 * randn(k))
        if m > 2:
            x[m // 2] = 0  # a padded position
        return x

    st = {"case": dict(c)}
    op = c["op"]
    if op in ("quantize", "norm", "norm_bwd"):
        dt = DT[c["dtype"]]
        st["x"] = activations(c["m"], c["k"]).to(dt)
    if op in ("norm", "norm_bwd"):
        st["weight"] = 1 + 0.1 * randn(c["k"])
    if op == "norm":
        st["residual"] = activations(c["m"], c["k"]).to(dt) if c["residual"] else None
    if op == "norm_bwd":
        st["dy"] = (1e-3 * randn(c["m"], c["k"])).to(dt)
        st["dh"] = (1e-3 * randn(c["m"], c["k"])).to(dt) if c["dh"] else None
        st["rstd"] = torch.rsqrt(st["x"].float().square().mean(1) + EPS)
    if op in ("linear", "dw"):
        st["xq"], st["xs"] = _to_int8(activations(c["m"], c["k"]))
    if op == "linear":
        st["wq"], st["ws"] = _to_int8(0.02 * randn(c["n"], c["k"]))
        st["b"] = 0.01 * randn(c["n"]) if c["bias"] else None
    if op == "dw":
        dz = 1e-3 * randn(c["m"], c["n"])
        st["dz"] = (dz * (randn(c["m"], c["n"]) > 0)).to(torch.bfloat16)  # behind a ReLU
    return st


# ------------------------------------------------------------------------------------ the operators
def run(state):
    c = state["case"]
    return (_calls if own else _plain)[c["op"]](c, state)


def _own_quantize(c, st):
    from c3_b200 import quant
    q, scale = quant.quantize_rows(st["x"])
    return {"q": q, "scale": scale}


def _own_norm(c, st):
    from c3_b200 import norm
    q, scale, h, rstd = norm.rms_norm_int8(st["x"], st["weight"], EPS, residual=st["residual"])
    return {"q": q, "scale": scale, "h": h, "rstd": rstd}


def _own_norm_bwd(c, st):
    from c3_b200 import norm
    dx, dweight = norm.rms_norm_backward(st["dy"], st["x"], st["weight"], st["rstd"], dh=st["dh"])
    return {"dx": dx, "dweight": dweight}


def _own_linear(c, st):
    from c3_b200 import linear
    y, mask = linear.forward_int8(st["xq"], st["xs"], st["wq"], st["ws"], st["b"], relu=c["relu"],
                                  out_dtype=DT[c["out"]])
    return {"y": y, "mask": mask} if c["relu"] else {"y": y}


def _own_dw(c, st):
    from c3_b200 import linear
    return {"dw": linear.grad_weight_int8(st["dz"], st["xq"], st["xs"])}


_calls = {"quantize": _own_quantize, "norm": _own_norm, "norm_bwd": _own_norm_bwd, "linear": _own_linear,
          "dw": _own_dw}


def _nearest(a, big):
    """round(127 a / A) with ties to even, in 64 bits: a quotient of two 32-bit floats that is not
    a tie is further from one than a 64-bit division can lose."""
    b = big.double()[:, None]
    return torch.where(b > 0, torch.round(a.double() * 127 / b), 0.0).to(torch.int8)


def _plain_quantize(c, st):
    x = st["x"].float()
    big = x.abs().amax(1)
    return {"q": _nearest(x, big), "scale": big / 127}


def _plain_norm(c, st):
    h = st["x"]
    if st["residual"] is not None:
        h = (h.float() + st["residual"].float()).to(h.dtype)
    f = h.float()
    rstd = 1 / torch.sqrt(f.square().mean(1) + EPS)
    a = f * st["weight"]
    big = a.abs().amax(1)
    return {"q": _nearest(a, big), "scale": big * rstd / 127, "h": h, "rstd": rstd}


def _plain_norm_bwd(c, st):
    h, dy, r = st["x"].float(), st["dy"].float(), st["rstd"][:, None]
    xhat = h * r
    g = dy * st["weight"]
    dx = (g - xhat * (g * xhat).mean(1, keepdim=True)) * r
    if st["dh"] is not None:
        dx = dx + st["dh"].float()
    return {"dx": dx.to(st["x"].dtype), "dweight": (dy * xhat).sum(0)}


def _plain_linear(c, st):
    # the integer sums pass 2^24: products and sums in 64 bits are exact
    acc = (st["xq"].double() @ st["wq"].double().t()).float()
    z = acc * (st["xs"][:, None] * st["ws"][None, :])
    if st["b"] is not None:
        z = z + st["b"]
    if not c["relu"]:
        return {"y": z.to(DT[c["out"]])}
    m, n = z.shape
    bits = torch.zeros((m, (n + 31) // 32 * 32), dtype=torch.int64, device=z.device)
    bits[:, :n] = z > 0
    words = (bits.view(m, -1, 32) << torch.arange(32, device=z.device)).sum(2)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return {"y": z.clamp_min(0).to(DT[c["out"]]), "mask": words}


def _plain_dw(c, st):
    x = st["xq"].float() * st["xs"][:, None]
    return {"dw": (st["dz"].float().t() @ x).to(torch.bfloat16)}


_plain = {"quantize": _plain_quantize, "norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "linear": _plain_linear,
          "dw": _plain_dw}


# ------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    op, m, k = c["op"], c["m"], c["k"]
    if op in ("quantize", "norm", "norm_bwd"):
        e = 2 if c["dtype"] == "bf16" else 4
        if op == "quantize":
            return {"bytes": m * k * (e + 1) + 4 * m, "flops": 3 * m * k}
        if op == "norm":  # x (and residual in, h out), q, scale, rstd, weight
            return {"bytes": m * k * (e * (3 if c["residual"] else 1) + 1) + 8 * m + 4 * k, "flops": 7 * m * k}
        return {"bytes": m * k * e * (4 if c["dh"] else 3) + 4 * m + 8 * k, "flops": 10 * m * k}
    n = c["n"]
    if op == "linear":
        e = 2 if c["out"] == "bf16" else 4
        mask = 4 * m * ((n + 31) // 32) if c["relu"] else 0
        return {"bytes": m * k + n * k + e * m * n + mask + 4 * (m + 2 * n), "flops": 2 * m * n * k}
    return {"bytes": 2 * m * n + m * k + 4 * m + 2 * n * k, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return {"q": None, "scale": st["x"].double().abs().max(dim=1).values / 127.0}
    if op in ("norm", "norm_bwd"):
        x, w = st["x"].double(), st["weight"].double()
        k = x.shape[1]
    if op == "norm":
        h = x
        if st["residual"] is not None:
            h = x + st["residual"].double()
            x = (st["x"].float() + st["residual"].float()).to(st["x"].dtype).double()  # the stored sum
        rstd = torch.pow((x * x).sum(1) / k + EPS, -0.5)
        scale = (x * w).abs().max(dim=1).values * rstd / 127.0
        return {"q": None, "scale": scale, "h": h, "rstd": rstd}
    if op == "norm_bwd":
        dy, r = st["dy"].double(), st["rstd"].double()
        dot = torch.einsum("mk,mk,k->m", dy, x, w)
        dx = dy * w * r[:, None] - x * (dot * r.pow(3) / k)[:, None]
        if st["dh"] is not None:
            dx += st["dh"].double()
        return {"dx": dx, "dweight": torch.einsum("mk,mk,m->k", dy, x, r)}
    xd = st["xq"].double() * st["xs"].double()[:, None]
    if op == "dw":
        return {"dw": torch.mm(st["dz"].double().t(), xd)}
    y = torch.mm(xd, (st["wq"].double() * st["ws"].double()[:, None]).t())
    if st["b"] is not None:
        y += st["b"].double()
    if not case["relu"]:
        return {"y": y}
    return {"y": torch.relu(y), "mask": None}
