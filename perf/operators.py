"""The operators around a frozen four-bit trunk and its trained norms, as measured cases.

``layer_norm``  layer norm over the last axis, forward, and forward + backward with the gradients of
                its weight and bias summed over all rows
``mx_quant``    OCP microscaled four-bit floats (e2m1 elements, one e8m0 scale per 32 of a row):
                quantise a matrix and read it back
``mx_linear``   y = x W^T + b on the block-scaled matrix instructions, W kept in four bits, x
                quantised in the call; with ``train`` also the gradient of x
``clip``        global gradient norm over many tensors and clipping by it

``own`` False computes each operator in elementary torch operations, True calls the framework's.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


_framework = None


def _ops():
    global _framework
    if _framework is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "hy-video-prfl_amd"))
        from prfl_amd import ops
        _framework = ops
    return _framework


# ------------------------------------------------------------------------------------- cases ----
def listed():
    return [
        # the first norm over the 257 image tokens of an I2V sample: latency
        dict(name="ln_image_tokens", op="layer_norm", rows=257, cols=1280, x="fp32", y="bf16",
             w="fp32", affine=True, train=False, pad=0),
        # the affine norm before the cross-attention of a 720p x 81-frame sample, fp32 residual
        dict(name="ln_720p", op="layer_norm", rows=73920, cols=5120, x="fp32", y="bf16", w="fp32",
             affine=True, train=False, pad=0),
        # a trained norm of odd width over a ragged batch, everything in fp16
        dict(name="ln_train_odd", op="layer_norm", rows=1003, cols=1021, x="fp16", y="fp16",
             w="fp16", affine=True, train=True, pad=0),
        # a trained norm over a 480p x 81-frame sample in bf16 with fp32 weights
        dict(name="ln_train_480p", op="layer_norm", rows=32760, cols=5120, x="bf16", y="bf16",
             w="fp32", affine=True, train=True, pad=0),
        # activations of a short ragged batch whose width is no multiple of the scale's block
        dict(name="mx_quant_ragged", op="mx_quant", rows=333, cols=1000, x="fp32"),
        # the feed-forward weight of a 14B block, quantised when a trunk is frozen
        dict(name="mx_quant_weight", op="mx_quant", rows=13824, cols=5120, x="bf16"),
        # a projection for a single token (the time embedding of one sample)
        dict(name="mx_linear_token", op="mx_linear", m=1, n=5120, k=5120, x="bf16", bias=True,
             train=False),
        # the text projection of 512 prompt tokens
        dict(name="mx_linear_text", op="mx_linear", m=512, n=5120, k=4096, x="bf16", bias=True,
             train=False),
        # the feed-forward up-projection of a 480p x 81-frame sample through the frozen trunk
        dict(name="mx_linear_480p", op="mx_linear", m=32760, n=13824, k=5120, x="bf16", bias=True,
             train=False),
        # an attention projection of the reward trunk in training: the gradient passes through it
        dict(name="mx_linear_train", op="mx_linear", m=8190, n=5120, k=5120, x="bf16", bias=True,
             train=True),
        # a reward head's few gradients, already below the limit: latency, nothing to scale
        dict(name="clip_head", op="clip", tensors=12, width=1280, g="fp32", out="", clipped=False),
        # two 14B blocks' bf16 gradients, clipped into the fp32 ones that the optimizer reads
        dict(name="clip_blocks", op="clip", tensors=54, width=5120, g="bf16", out="fp32",
             clipped=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm", "mx_quant", "mx_linear", "mx_linear", "clip"])
    if op == "layer_norm":
        cols = _log_int(rng, 8, 16384)
        if rng.random() < 0.5:
            cols = max(8, cols // 8 * 8)
        rows = _log_int(rng, 1, min(73920, 160_000_000 // cols))
        x = rng.choice(["fp32", "bf16", "fp16"])
        return dict(op=op, rows=rows, cols=cols, x=x,
                    y=rng.choice([x, "bf16" if x == "fp32" else x]), w=rng.choice(["fp32", x]),
                    affine=rng.random() < 0.8, train=rng.random() < 0.5,
                    pad=rng.choice([0, 0, 8, 3]))
    if op == "mx_quant":
        cols = _log_int(rng, 8, 14000)
        return dict(op=op, rows=_log_int(rng, 1, min(73920, 70_000_000 // cols)), cols=cols,
                    x=rng.choice(["fp32", "bf16", "fp16"]))
    if op == "mx_linear":
        k, n = _log_int(rng, 64, 14000), _log_int(rng, 8, 14000)
        if rng.random() < 0.5:
            k, n = -(-k // 32) * 32, -(-n // 32) * 32
        train = rng.random() < 0.4
        m = _log_int(rng, 1, min(32760, int((1.1e12 if train else 2.3e12) / (k * n))))
        return dict(op=op, m=m, n=n, k=k, x=rng.choice(["bf16", "bf16", "fp32", "fp16"]),
                    bias=rng.random() < 0.7, train=train)
    g = rng.choice(["fp32", "bf16", "fp16"])
    clipped = rng.random() < 0.7
    return dict(op=op, tensors=rng.randint(1, 60), width=_log_int(rng, 33, 4000), g=g,
                out=rng.choice([g, "fp32"]) if clipped else "", clipped=clipped)


def _clip_shapes(c):
    """Square weights, one wide one and vectors in turn, as a block's parameters lie."""
    d = c["width"]
    kinds = [(d, d), (d,), (d, d), (d,), (d, d), (1,), (2 * d + 1, d), (2 * d + 1,), (d,)]
    return [kinds[i % len(kinds)] for i in range(c["tensors"])]


# ------------------------------------------------------------------------------------ inputs ----
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 13)


def _activations(g, rows, cols, dtype):
    """Rows of different scale with a mean of their own, as residual streams have, some of them
    padding."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    size = torch.exp(torch.randn(rows, 1, generator=g, device=DEV) * 0.7)
    mean = torch.randn(rows, 1, generator=g, device=DEV) * 0.5
    x = (x + mean) * size
    x[3::97] = 0.0
    return x.to(dtype)


def _upstream(g, rows, cols, dtype):
    """A gradient of such rows: none where they are padding."""
    dy = torch.randn(rows, cols, generator=g, device=DEV)
    dy[3::97] = 0.0
    return dy.to(dtype)


def _tile(codes, scales):
    """e2m1 codes [R, K] and e8m0 bytes [R, K / 32], K a multiple of 32, in the layout in which a
    program keeps them: 64 rows x 128 columns at a time, as [row half][column half][lane] pieces
    of 32 codes, lane = 32 * (second 32 columns) + row, and the four pieces' scales side by side."""
    r, k = codes.shape
    rp, kp = -(-r // 64) * 64, -(-k // 128) * 128
    c = torch.zeros(rp, kp, dtype=torch.uint8, device=codes.device)
    c[:r, :k] = codes
    c = c.view(rp, kp // 2, 2)
    c = c[..., 0] | (c[..., 1] << 4)
    # [group, row half, row, step, column half, block, byte]
    c = c.view(rp // 64, 2, 32, kp // 128, 2, 2, 16).permute(0, 3, 1, 4, 5, 2, 6)
    s = torch.zeros(rp, kp // 32, dtype=torch.uint8, device=codes.device)
    s[:r, :k // 32] = scales
    s = s.view(rp // 64, 2, 32, kp // 128, 2, 2).permute(0, 3, 5, 2, 1, 4)
    return (c.reshape(rp // 64, kp // 128, 4, 64, 16).contiguous(),
            s.reshape(rp // 64, kp // 128, 64, 4).contiguous())


def _untile(q, s):
    """The values of a tiled matrix with its padding, fp32."""
    g, t = q.shape[:2]
    c = torch.stack((q & 15, q >> 4), -1).view(g, t, 2, 2, 2, 32, 32)
    c = c.permute(0, 2, 5, 1, 3, 4, 6).reshape(g * 64, t * 128)
    e = s.view(g, t, 2, 32, 2, 2).permute(0, 4, 3, 1, 5, 2).reshape(g * 64, t * 4)
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6],
                         device=q.device)
    v = table[c.long()].view(g * 64, t * 4, 32)
    return torch.ldexp(v, (e.int() - 127).unsqueeze(-1)).view(g * 64, t * 128)


def _mx(x):
    """(element values, exponents) of x [R, K] in 32 bits: 32 of a row share 2^e, e = floor(log2
    of the largest) - 2, elements to the nearest of 0 .5 1 1.5 2 3 4 6, ties to the even code."""
    r, k = x.shape
    kp = -(-k // 32) * 32
    v = torch.zeros(r, kp, device=x.device)
    v[:, :k] = x
    v = v.view(r, kp // 32, 32)
    e = (torch.frexp(v.abs().amax(-1, keepdim=True))[1] - 3).clamp_(min=-127)
    e = torch.where(v.abs().amax(-1, keepdim=True) == 0, torch.full_like(e, -127), e)
    v = torch.ldexp(v, -e)
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = ((a / step).round() * step).clamp(max=6.0)
    return torch.copysign(a, v), e.squeeze(-1)


def _mx_values(x):
    v, e = _mx(x.float())
    return torch.ldexp(v, e.unsqueeze(-1)).view(x.shape[0], -1)[:, :x.shape[1]]


def prepare(case, seed):
    g, c = _gen(seed), dict(case)
    if c["op"] == "layer_norm":
        wide = _activations(g, c["rows"], c["cols"] + c["pad"], DTYPES[c["x"]])
        c["xt"] = wide[:, :c["cols"]]
        c["eps"] = 1e-6
        c["wt"] = c["bt"] = None
        if c["affine"]:
            c["wt"] = (1 + 0.2 * torch.randn(c["cols"], generator=g, device=DEV)).to(DTYPES[c["w"]])
            c["bt"] = (0.2 * torch.randn(c["cols"], generator=g, device=DEV)).to(DTYPES[c["w"]])
        if c["train"]:
            c["dy"] = _upstream(g, c["rows"], c["cols"], DTYPES[c["y"]])
    elif c["op"] == "mx_quant":
        c["xt"] = _activations(g, c["rows"], c["cols"], DTYPES[c["x"]])
    elif c["op"] == "mx_linear":
        c["xt"] = _activations(g, c["m"], c["k"], DTYPES[c["x"]])
        v, e = _mx(_weight(c, g))
        code = torch.bucketize(v.abs(), torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.],
                                                     device=DEV))
        code = code + 8 * torch.signbit(v)
        c["wq"], c["ws"] = _tile(code.to(torch.uint8).view(c["n"], -1), (e + 127).to(torch.uint8))
        c["bt"] = _bias(c, g)
        if c["train"]:
            c["dy"] = _upstream(g, c["m"], c["n"], torch.bfloat16)
    else:
        c["gt"] = [(torch.randn(s, generator=g, device=DEV)
                    * torch.exp(torch.randn((), generator=g, device=DEV))).to(DTYPES[c["g"]])
                   for s in _clip_shapes(c)]
        c["max_norm"] = 1.0 if c["clipped"] else 1e9
        c["outs"] = [torch.empty_like(t, dtype=DTYPES[c["out"]]) for t in c["gt"]] \
            if c["out"] else None
    return c


def _weight(c, g):
    return torch.randn(c["n"], c["k"], generator=g, device=DEV) / math.sqrt(c["k"])


def _bias(c, g):
    return (0.1 * torch.randn(c["n"], generator=g, device=DEV)).to(torch.bfloat16) \
        if c["bias"] else None


# --------------------------------------------------------------------------------- one pass ----
def run(state):
    if own:
        return _run_own(state)
    return {"layer_norm": _plain_layer_norm, "mx_quant": _plain_mx_quant,
            "mx_linear": _plain_mx_linear, "clip": _plain_clip}[state["op"]](state)


def _run_own(s):
    ops = _ops()
    if s["op"] == "layer_norm":
        y, mean, rstd = ops.layer_norm_fwd(s["xt"], s["wt"], s["bt"], s["eps"],
                                           out_dtype=DTYPES[s["y"]])
        if not s["train"]:
            return {"y": y}
        dx, dw, db = ops.layer_norm_bwd(s["dy"], s["xt"], mean, rstd, s["wt"],
                                        want_db=s["bt"] is not None)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if s["op"] == "mx_quant":
        q, e = ops.quant_mxfp4(s["xt"])
        return {"values": ops.dequant_mxfp4(q, e, s["rows"], s["cols"])}
    if s["op"] == "mx_linear":
        y = ops.linear_mxfp4(s["xt"], s["wq"], s["ws"], s["n"], s["bt"])
        if not s["train"]:
            return {"y": y}
        return {"y": y, "dx": ops.linear_mxfp4_dx(s["dy"], s["wq"], s["ws"], s["k"])}
    norm = ops.clip_grads(s["gt"], s["max_norm"], out=s["outs"])
    return {"norm": norm, "grads": s["outs"] or s["gt"]}


def _plain_layer_norm(s):
    x = s["xt"].float()
    d = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + s["eps"])
    xhat = d * rstd
    y = xhat if s["wt"] is None else xhat * s["wt"].float() + s["bt"].float()
    y = y.to(DTYPES[s["y"]])
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy if s["wt"] is None else dy * s["wt"].float()
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    dw = db = None
    if s["wt"] is not None:
        dw, db = (dy * xhat).sum(0), dy.sum(0)
    return {"y": y, "dx": dx.to(DTYPES[s["x"]]), "dw": dw, "db": db}


def _plain_mx_quant(s):
    return {"values": _mx_values(s["xt"]).to(torch.bfloat16)}


def _plain_mx_linear(s):
    w = _untile(s["wq"], s["ws"])[:s["n"], :s["k"]]
    y = _mx_values(s["xt"]) @ w.t()
    if s["bt"] is not None:
        y = y + s["bt"].float()
    y = y.to(torch.bfloat16)
    if not s["train"]:
        return {"y": y}
    return {"y": y, "dx": (s["dy"].float() @ w).to(torch.bfloat16)}


def _plain_clip(s):
    norm = torch.stack([t.double().square().sum() for t in s["gt"]]).sum().sqrt().float()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    if s["outs"] is None:
        return {"norm": norm, "grads": [t.copy_(t.float() * coef) for t in s["gt"]]}
    return {"norm": norm, "grads": [o.copy_(t.float() * coef) for t, o in zip(s["gt"], s["outs"])]}


# ------------------------------------------------------------------------- what it cannot save ----
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


def work(case):
    c = case
    if c["op"] == "layer_norm":
        n, v = c["rows"] * c["cols"], c["cols"] * SIZE[c["w"]] * 2 * c["affine"]
        b = n * (SIZE[c["x"]] + SIZE[c["y"]]) + v
        if c["train"]:
            b += n * (SIZE[c["x"]] + SIZE[c["y"]]) + c["cols"] * 8 * c["affine"]
        return {"bytes": b, "flops": n * (20 if c["train"] else 8)}
    if c["op"] == "mx_quant":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (SIZE[c["x"]] + 2), "flops": 4 * n}
    if c["op"] == "mx_linear":
        m, n, k = c["m"], c["n"], c["k"]
        b = m * k * SIZE[c["x"]] + n * k * 17 / 32 + m * n * 2 + 2 * n * c["bias"]
        if c["train"]:
            b += m * n * 2 + m * k * 2
        return {"bytes": b, "flops": 2 * m * n * k * (2 if c["train"] else 1)}
    n = sum(math.prod(s) for s in _clip_shapes(c))
    return {"bytes": n * (SIZE[c["g"]] + (SIZE[c["out"]] if c["clipped"] else 0)), "flops": 3 * n}


# ------------------------------------------------------------------------------- in 64 bits ----
def _exact_mx(x):
    """Microscaled values of x [R, K] in 64 bits, by the definition's grid: the code whose interval
    between midpoints holds the scaled value."""
    r, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(r, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2)
    a = v.abs() / scale
    # a tie goes to the even code: the midpoints above odd codes belong to the code above
    out = torch.zeros_like(a)
    for mid, low, high, up in ((.25, 0, .5, False), (.75, .5, 1, True), (1.25, 1, 1.5, False),
                               (1.75, 1.5, 2, True), (2.5, 2, 3, False), (3.5, 3, 4, True),
                               (5., 4, 6, False)):
        out = torch.where((a >= mid) if up else (a > mid), torch.full_like(a, high), out)
    return (out * torch.sign(v) * scale).view(r, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "layer_norm":
        x = s["xt"].double().requires_grad_(s["train"])
        leaves = [x]
        w = b = None
        if s["affine"]:
            w, b = s["wt"].double(), s["bt"].double()
            if s["train"]:
                leaves += [w.requires_grad_(), b.requires_grad_()]
        y = torch.nn.functional.layer_norm(x, (s["cols"],), w, b, s["eps"])
        if not s["train"]:
            return {"y": y}
        got = list(torch.autograd.grad(y, leaves, s["dy"].double())) + [None, None]
        return {"y": y.detach(), "dx": got[0], "dw": got[1], "db": got[2]}
    if s["op"] == "mx_quant":
        return {"values": _exact_mx(s["xt"])}
    if s["op"] == "mx_linear":
        g = _gen(seed)
        _activations(g, s["m"], s["k"], DTYPES[s["x"]])
        w = _exact_mx(_weight(s, g))
        y = _exact_mx(s["xt"]) @ w.t()
        if s["bt"] is not None:
            y += s["bt"].double()
        if not s["train"]:
            return {"y": y}
        return {"y": y, "dx": s["dy"].double() @ w}
    norm = math.sqrt(math.fsum(float(t.double().norm()) ** 2 for t in s["gt"]))
    coef = min(1.0, s["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=torch.float64, device=DEV),
            "grads": [t.double() * coef for t in s["gt"]]}
