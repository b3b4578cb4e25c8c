"""layer_norm_fwd / layer_norm_bwd on the MI355X against the formulas in 64 bits.

Tolerances, per element, u = 2^-24 and U = eps(type) / 2 (half a step of the output):
a sum over a row is at most 16 terms a thread, 6 levels of a wave and 16 waves deep, so a mean is
within 38 u of the mean of magnitudes, and a variance, a root and a product add less than 20 u
more: A = 64 covers the chain.
  y:   U |y| + A u (|w| (r (|x| + mean |x|) + |xhat|) + |b|)
  dx:  U |dx| + A u r (|g| + mean |g| + |xhat| mean |g xhat|) + r (d |m2| + |xhat| mean (|g| d)),
       d = A u (r (|x| + mean |x|) + |xhat|) the error of xhat
  dw:  (rows + 64) u sum |dy xhat| + sum |dy| d;   db: (rows + 64) u sum |dy|
"""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
u = 2.0 ** -24
A = 64


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


def reference(x, w, b, eps, dy=None):
    """y (and dx, dw, db) in 64 bits with the bounds' ingredients."""
    x = x.double()
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    d = A * u * (r * (x.abs() + x.abs().mean(-1, keepdim=True)) + xh.abs())
    out = dict(y=xh * w + b, ty=w.abs() * d + A * u * b.abs(), mean=mu.squeeze(-1), rstd=r.squeeze(-1))
    if dy is not None:
        dy = dy.double()
        g = dy * w
        m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        out["dx"] = r * (g - m1 - xh * m2)
        out["tdx"] = A * u * r * (g.abs() + g.abs().mean(-1, keepdim=True)
                                  + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) \
            + r * (d * m2.abs() + xh.abs() * (g.abs() * d).mean(-1, keepdim=True))
        rows = x.numel() // C
        f = lambda t: t.reshape(rows, C).sum(0)  # noqa: E731
        out["dw"], out["db"] = f(dy * xh), f(dy)
        out["tdw"] = (rows + 64) * u * f((dy * xh).abs()) + f(dy.abs() * d)
        out["tdb"] = (rows + 64) * u * f(dy.abs())
    return out


def within(got, want, tol, what):
    U = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else u
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    err = (got.double() - want).abs()
    lim = U * want.abs() + tol * (1 + U) + tiny
    bad = ~(err <= lim)
    assert not bad.any(), (what, int(bad.sum()), float((err / lim).max()))


def inputs(shape, dtype, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) + mean * torch.randn(*shape[:-1], 1, generator=g)
    w = 1 + 0.3 * torch.randn(shape[-1], generator=g)
    b = 0.3 * torch.randn(shape[-1], generator=g)
    dy = torch.randn(*shape, generator=g)
    return x.to(dtype).to(DEV), w.to(DEV), b.to(DEV), dy.to(DEV)


def check(ops, x, w, b, dy, eps=1e-6, out_dtype=None):
    yt = out_dtype or x.dtype
    dy = dy.to(yt)
    ref = reference(x, w, b, eps, dy)
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, eps, out_dtype=out_dtype)
    assert y.dtype == yt and y.shape == x.shape and mean.shape == x.shape[:-1] == rstd.shape
    within(y, ref["y"], ref["ty"], "y")
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w, want_dw=True)
    assert dx.dtype == x.dtype and dx.shape == x.shape and dw.dtype == db.dtype == F32
    within(dx, ref["dx"], ref["tdx"], "dx")
    within(dw, ref["dw"], ref["tdw"], "dw")
    within(db, ref["db"], ref["tdb"], "db")


@pytest.mark.parametrize("xt,yt", itertools.product((F32, BF16, F16), repeat=2))
def test_types(ops, xt, yt):
    x, w, b, dy = inputs((37, 328), xt)
    check(ops, x, w, b, dy, out_dtype=yt)
    check(ops, x, w.to(BF16), b.to(BF16), dy, out_dtype=yt)
    check(ops, x, w.to(F16), b.to(F16), dy, out_dtype=yt)


# one element to the widest row; every number of chunks a thread and waves a row can have, odd
# widths whose rows lie at every alignment
@pytest.mark.parametrize("xt", (F32, BF16, F16))
@pytest.mark.parametrize("C", (1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 257, 511, 513, 1021, 1024, 1280, 2047,
                               2049, 4095, 5120, 6145, 8191, 8193, 16383, 16384))
def test_widths(ops, C, xt):
    x, w, b, dy = inputs((5, C), xt, seed=C)
    check(ops, x, w, b, dy)


# rows that end inside a lane's vector, at a wave's end, in its last chunk and one past it
@pytest.mark.parametrize("xt,yt", ((F32, BF16), (BF16, BF16), (F16, F32)))
@pytest.mark.parametrize("C", (4, 5, 6, 33, 127, 129, 250, 260, 500, 516, 519, 770, 776, 1031, 1288, 1540, 1654, 2056,
                               4104, 5003, 6076, 8200, 12001))
def test_rows_that_end_inside_a_vector(ops, C, xt, yt):
    x, w, b, dy = inputs((21, C), xt, seed=C)
    check(ops, x, w, b, dy, out_dtype=yt)
    wide, _, _, dwide = inputs((13, C + 3), xt, seed=C + 1)
    check(ops, wide[:, 2:C + 2], w, None, dwide[:, 1:C + 1])
    y, m, r = ops.layer_norm_fwd(x, w, b, out_dtype=yt)
    again = ops.layer_norm_fwd(x, w, b, out_dtype=yt)[0]
    assert torch.equal(y, again)
    for a, c in zip(ops.layer_norm_bwd(dy, x, m, r, w), ops.layer_norm_bwd(dy, x, m, r, w)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("C", (5, 100, 517, 1654, 6076))
def test_a_value_that_is_no_number_stays_in_its_row(ops, C):
    x, w, b, dy = inputs((40, C), BF16, seed=C)
    y0, m, r = ops.layer_norm_fwd(x, w, b)
    dx0 = ops.layer_norm_bwd(dy, x, m, r, w)[0]
    for col in (0, C // 2, C - 2, C - 1):
        for v in (math.nan, math.inf, -math.inf):
            bad, dbad = x.clone(), dy.clone()
            bad[7, col], dbad[9, col] = v, v
            y, m1, r1 = ops.layer_norm_fwd(bad, w, b)
            assert y[7].isnan().all() and torch.equal(y[:7], y0[:7]) and torch.equal(y[8:], y0[8:])
            dx, dw, db = ops.layer_norm_bwd(dbad, x, m, r, w)
            assert not dx[9].isfinite().any()
            assert torch.equal(dx[:9], dx0[:9]) and torch.equal(dx[10:], dx0[10:])
            keep = torch.arange(C, device=DEV) != col
            assert not db[col].isfinite() and dw[keep].isfinite().all() and db[keep].isfinite().all()


@pytest.mark.parametrize("rows", (1, 2, 3, 4, 5, 15, 16, 17, 32, 33, 63, 64, 65, 511, 512, 513, 2047, 2049, 8200))
def test_rows(ops, rows):
    for C, t in ((64, F16), (200, BF16), (700, BF16), (1280, BF16), (5, F32)):
        x, w, b, dy = inputs((rows, C), t, seed=rows)
        check(ops, x, w, b, dy)


def test_without_weight_or_bias(ops):
    x, w, b, dy = inputs((33, 257), BF16)
    check(ops, x, None, None, dy)
    check(ops, x, w, None, dy)
    check(ops, x, None, b, dy)


def test_leading_axes_strides_and_alignment(ops):
    x, w, b, dy = inputs((3, 4, 5, 96), BF16)
    check(ops, x, w, b, dy)
    check(ops, x.transpose(0, 2), w, b, dy.transpose(0, 2))          # leading axes out of order
    check(ops, x.transpose(1, 3)[..., :3], w[:3], b[:3], dy.transpose(1, 3)[..., :3])
    check(ops, x[0, 0].expand(4, 5, 96), w, b, dy[0, :4])            # one batch's rows for all
    for off in (1, 2, 5):                                           # column slices of a wider buffer
        wide, _, _, dwide = inputs((31, 300), F16, seed=off)
        check(ops, wide[:, off:off + 260], inputs((1, 260), F32)[1], None, dwide[:, off:off + 260])
    one = inputs((1, 96), F32)[3][:, :1].expand(2, 96)              # dy of a sum: strides 0
    check(ops, x[0, 0, :2], w, b, one)
    flat = torch.randn(96 * 2 + 1, device=DEV)
    check(ops, x[0, 0], flat[1:97], flat[97:], dy[0, 0])            # misaligned weights


@pytest.mark.parametrize("t", (F32, BF16))
def test_far_mean_and_large_values(ops, t):
    """a mean far above the spread costs the digits that x itself has not, and no more"""
    x, w, b, dy = inputs((17, 1000), t, mean=0)
    check(ops, x * 0.01 + 100, w, b, dy)
    check(ops, x * 1e15, w, b, dy)
    check(ops, x * 1e-12, w, b, dy, eps=1e-30)


def test_constant_rows(ops):
    x, w, b, dy = inputs((6, 130), BF16)
    x[1] = 0
    x[4] = 3
    check(ops, x, w, b, dy)
    y, _, rstd = ops.layer_norm_fwd(x, w, b, 1e-6)
    assert torch.equal(y[4], b.to(BF16)) and torch.equal(y[1], b.to(BF16))


def test_nan_and_inf_stay_in_their_row(ops):
    x, w, b, dy = inputs((9, 200), F32)
    clean = ops.layer_norm_fwd(x, w, b)
    x[3, 7], x[5, 100] = float("nan"), float("inf")
    y, mean, rstd = ops.layer_norm_fwd(x, w, b)
    dx, _, _ = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    rows = [i for i in range(9) if i not in (3, 5)]
    assert torch.equal(y[rows], clean[0][rows]) and y[[3, 5]].isnan().all()
    assert dx[rows].isfinite().all() and dx[[3, 5]].isnan().all()


def test_empty(ops):
    x = torch.empty(0, 3, 48, device=DEV, dtype=BF16)
    w = torch.ones(48, device=DEV)
    y, mean, rstd = ops.layer_norm_fwd(x, w)
    dx, dw, db = ops.layer_norm_bwd(x, x, mean, rstd, w)
    assert y.shape == dx.shape == x.shape and not dw.any() and not db.any()


def test_one_axis(ops):
    x, w, b, dy = inputs((1, 300), BF16)
    check(ops, x[0], w, b, dy[0])


def test_wanted_outputs_only(ops):
    x, w, b, dy = inputs((70, 300), F32)
    _, mean, rstd = ops.layer_norm_fwd(x, w, b)
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    none = ops.layer_norm_bwd(dy, x, mean, rstd, w, want_dx=False, want_dw=False, want_db=False)
    assert none == (None, None, None)
    only = ops.layer_norm_bwd(dy, x, mean, rstd, w, want_dx=False, want_db=False)
    assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
    only = ops.layer_norm_bwd(dy, x, mean, rstd, w, want_dw=False)
    assert only[1] is None and torch.equal(only[0], dx) and torch.equal(only[2], db)


def test_same_bits_every_time_and_on_another_stream(ops):
    x, w, b, dy = inputs((3000, 640), BF16)

    def both():
        y, m, r = ops.layer_norm_fwd(x, w, b)
        return (y,) + ops.layer_norm_bwd(dy.to(BF16), x, m, r, w)
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got))


def test_captured_and_replayed(ops):
    x, w, b, dy = inputs((515, 1021), F16)
    dy = dy.to(F16)

    def step():
        y, m, r = ops.layer_norm_fwd(x, w, b)
        return (y,) + ops.layer_norm_bwd(dy, x, m, r, w)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        x.copy_(torch.randn(515, 1021, device=DEV) + k)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, got)), k


def test_two_graphs_replayed_in_turn(ops):
    """each holds its own workspace: replays in any order, and eager calls between, change nothing"""
    from prfl_amd import custom_ops

    def build(seed):
        x, w, b, dy = inputs((700, 384), BF16, seed=seed)
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        dy = dy.to(BF16)

        def step():
            y = custom_ops.layer_norm(*leaves, 1e-6)
            return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.clone() for t in step()]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        return graph, got, want, (leaves, dy)           # what the graph reads lives as long as it
    a, b = build(1), build(2)
    x, w, bb, dy = inputs((900, 640), F32)
    for order in ((a, b), (b, a), (a, a, b)):
        for graph, *_ in order:
            graph.replay()
        _, m, r = ops.layer_norm_fwd(x, w, bb)
        ops.layer_norm_bwd(dy, x, m, r, w)
        torch.cuda.synchronize()
        for _, got, want, _ in (a, b):
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_autograd_op(ops):
    """prfl::layer_norm: gradients in the leaves' own types, against the formulas and differences"""
    from prfl_amd import custom_ops
    x, w, b, dy = inputs((4, 11, 130), F32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b.to(F32))]
    y = custom_ops.layer_norm(*leaves, 1e-6, None)
    got = torch.autograd.grad(y, leaves, dy)
    ref = reference(x, w, b, 1e-6, dy)
    within(y.detach(), ref["y"], ref["ty"], "y")
    for g, k in zip(got, ("dx", "dw", "db")):
        within(g, ref[k], ref["t" + k], k)
    # central differences of sum(dy y): truncation falls with h^2, rounding is 1 / h of y's error
    h, v = 2.0 ** -6, torch.randn(4, 11, 130, generator=torch.Generator().manual_seed(9)).to(DEV)
    with torch.no_grad():
        up, dn = (reference(x + s * h * v, w, b, 1e-6)["y"] for s in (1, -1))
        slope = ((up - dn) * dy.double()).sum() / (2 * h)
    assert abs(float((got[0].double() * v.double()).sum() - slope)) < 1e-3 * float(
        (got[0].double() * v.double()).abs().sum())
    # weights of another type than x, and a leaf that wants no gradient
    wb = w.to(BF16).requires_grad_()
    y = custom_ops.layer_norm(x.to(BF16), wb, b.to(BF16), 1e-6, F32)
    assert y.dtype == F32
    y.backward(dy)
    assert wb.grad.dtype == BF16
    torch.library.opcheck(torch.ops.prfl.layer_norm, (leaves[0], leaves[1], leaves[2], 1e-6, None))
