"""The block's norm kernels element by element against the formulas in 64 bits, at widths that reach every variant.

Tolerances, u = 2^-24, U = 2^-8 (bf16).  A lane adds at most 80 products and the wave or workgroup joins them in at
most 12 levels more, so a mean, a mean square and what a root, a quotient and two products add to them stay within
A = 128 u of the sums of magnitudes:
  ln    xhat: d = A u (r (|x| + mean |x|) + |xhat|), and U |xhat| more where it is rounded to bf16 (bf16 x, modulated)
        y: U |y| + |a| d + A u (|xhat a| + |b|)
        dx: A u r (|g| + mean |g| + |xhat| mean |g xhat|) + r (d mean |g xhat| + |xhat| mean (|g| d)) + u |dx|
  rms   n = bf16(x r): U |n| + A u |n|;  a rotation of pairs passes the errors of both on, with |cos| and |sin|
        dx: the gradient of n is rounded to bf16, U |dn|, which passes through the sum over the row
  sums over the rows: (rows + A) u sum |.| besides the terms' own errors
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
u, U, A = 2.0 ** -24, 2.0 ** -8, 128
TINY = 2.0 ** -133


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


def rand(*s, seed):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed)).to(DEV)


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    lim = (U if got.dtype == BF16 else u) * want.abs() + tol * (1 + U) + TINY
    assert (err <= lim).all(), (what, float((err / lim).max()))


# whole and ragged last chunks of 20 and of 8 a lane, and widths that the column-fixed backward does not take
@pytest.mark.parametrize("L", (1, 17, 77))
@pytest.mark.parametrize("C", (4, 200, 256, 1280, 1540, 2048, 2052, 2304, 4864, 5116, 5120))
@pytest.mark.parametrize("t", (F32, BF16))
@pytest.mark.parametrize("affine", (False, True))
def test_layer_norm_of_the_block(ops, C, L, t, affine):
    x = (2 * rand(L, C, seed=C) + rand(L, 1, seed=C + 1)).to(t)
    p, q = 0.2 * rand(C, seed=C + 2), 0.2 * rand(C, seed=C + 3)
    dy = rand(L, C, seed=C + 4).to(BF16)
    kw = dict(w=1 + p, b=q) if affine else dict(scale=p, shift=q)
    y, m, r0 = ops.ln_mod_fwd(x, **kw)
    a = (1 + p).double() if affine else 1 + p.double()
    X = x.double()
    mu = X.mean(-1, keepdim=True)
    r = 1 / ((X - mu).square().mean(-1, keepdim=True) + 1e-6).sqrt()
    xh = (X - mu) * r
    d = A * u * (r * (X.abs() + X.abs().mean(-1, keepdim=True)) + xh.abs())
    low = 0 if affine or t == F32 else U * xh.abs()
    within(y, xh * a + q.double(), a.abs() * (d + low) + A * u * ((xh * a).abs() + q.abs()), "y")
    within(m, mu.squeeze(-1), A * u * X.abs().mean(-1), "mean")
    base = rand(L, C, seed=C + 5)
    for accumulate in (False, True):
        dx = base.clone()
        s0, s1 = ops.ln_mod_bwd(dy, x, m, r0, dx, accumulate=accumulate, **({"w": 1 + p} if affine else {"scale": p}))
        D = dy.double()
        g = D * a
        gx = (g * xh).abs().mean(-1, keepdim=True)
        want = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        tol = A * u * r * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * gx) \
            + r * (d * gx + xh.abs() * (g.abs() * d).mean(-1, keepdim=True))
        within(dx, want + accumulate * base.double(), tol + accumulate * u * (want.abs() + base.double().abs()), "dx")
        within(s0, (D * xh).sum(0), (L + A) * u * (D * xh).abs().sum(0) + (D.abs() * (d + low)).sum(0), "d scale")
        within(s1, D.sum(0), (L + A) * u * D.abs().sum(0), "d shift")


def rotate(v, c, s, back=False):
    e, o = v[..., 0::2], v[..., 1::2]
    s = -s if back else s
    return torch.stack((e * c - o * s, e * s + o * c), -1).flatten(-2)


@pytest.mark.parametrize("C", (128, 256, 384, 1280, 2048, 4992, 5120))
@pytest.mark.parametrize("rope", (False, True))
@pytest.mark.parametrize("osc", (1.0, 0.1275))
def test_rms_norm_and_rope(ops, C, rope, osc):
    L, grid = 77, (2, 5, 7)                                  # 70 rotated rows and 7 behind them
    x, do = (3 * rand(L, C, seed=C)).to(BF16), rand(L, C, seed=C + 1).to(BF16)
    w = 1 + 0.2 * rand(C, seed=C + 2)
    ang = torch.outer(torch.arange(1024.0, dtype=torch.float64), 1e4 ** (-torch.arange(64.0, dtype=torch.float64) / 64))
    tab = ops.rope_table(torch.polar(torch.ones_like(ang), ang), DEV)
    osc = float(torch.tensor(osc, dtype=F32))
    y, r0 = ops.rms_rope_fwd(x, w, 1e-6, tab if rope else None, grid if rope else (0, 0, 0), out_scale=osc)
    dx, dw = ops.rms_rope_bwd(do, x, r0, w, tab if rope else None, grid if rope else (0, 0, 0), out_scale=osc)
    c, s = torch.ones(L, C // 2, device=DEV).double(), torch.zeros(L, C // 2, device=DEV).double()
    if rope:
        row, pair = torch.arange(70), torch.arange(64)
        at = torch.where(pair < 22, (row // 35)[:, None], torch.where(pair < 43, (row // 7 % 5)[:, None], (row % 7)[:, None]))
        cs = tab.cpu()[at, pair].to(DEV).double().repeat(1, C // 128, 1)
        c[:70], s[:70] = cs[..., 0], cs[..., 1]
    X, W = x.double(), w.double()
    r = 1 / (X.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    n = X * r
    within(y, rotate(n * W, c, s) * osc, (U + A * u) * rotate((n * W).abs(), c.abs(), -s.abs()).abs() * osc
           + (U + A * u) * osc * (rotate((n * W).abs(), c.abs(), s.abs())).abs(), "y")
    dy = rotate(do.double() * osc, c, s, back=True)
    size = rotate((do.double() * osc).abs(), c.abs(), s.abs()).abs() + rotate((do.double() * osc).abs(), c.abs(), -s.abs()).abs()
    dn, tn = dy * W, A * u * size * W.abs() + U * (dy * W).abs()
    m = (dn * n).mean(-1, keepdim=True)
    want = r * (dn - n * m)
    tol = r * (tn + n.abs() * (tn * n.abs()).mean(-1, keepdim=True)
               + A * u * (dn.abs() + n.abs() * (dn * n).abs().mean(-1, keepdim=True)))
    within(dx, want, tol, "dx")
    within(dw, (dy * n).sum(0), ((L + A) * u * (size * n.abs()) + (U + A * u) * (dy * n).abs()).sum(0), "dw")


def test_misaligned_rows_take_the_other_kernels(ops):
    """views that the 16-byte kernels do not take give the aligned call's values to the same tolerances"""
    C, L = 1280, 40
    w, p = 1 + 0.1 * rand(C, seed=1), 0.1 * rand(C, seed=2)
    wide = rand(L, C + 8, seed=3)
    x, dy = wide[:, 4:C + 4], rand(L, C + 4, seed=4).to(BF16)[:, 4:]
    y, m, r = ops.ln_mod_fwd(x, scale=p, shift=p)
    want = ops.ln_mod_fwd(x.contiguous(), scale=p, shift=p)
    assert torch.equal(y, want[0]) and torch.equal(m, want[1]) and torch.equal(r, want[2])
    got, ref = torch.zeros(L, C, device=DEV), torch.zeros(L, C, device=DEV)
    a = ops.ln_mod_bwd(dy, x, m, r, got, scale=p, accumulate=False)
    b = ops.ln_mod_bwd(dy.contiguous(), x.contiguous(), m, r, ref, scale=p, accumulate=False)
    assert ((got - ref).abs() <= 8 * A * u * (1 + ref.abs()) * float(r.max())).all()
    assert all(((g - f).abs() <= 8 * A * u * L * (1 + f.abs())).all() for g, f in zip(a, b))
