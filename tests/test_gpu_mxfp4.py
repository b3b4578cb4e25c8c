"""Microscaled fp4 on the MI355X: quantisation bit for bit against the definition in 64 bits, the
product against 64 bits.

Tolerances of the product: elements times elements are exact in fp32 (3 bits each), so y differs
from the exact sum by the fp32 additions, at most one step 2^-23 of the partial magnitudes each
(K of them), and by one rounding to bf16 (2^-8):  2^-8 |y| + (K + 1) 2^-23 (sum |x w| + |b|).
Where every partial sum is a multiple of 1/4 below 2^22 the additions are exact, and y has to be
the exact sum rounded to bf16 (one more rounding in fp32 with the bias left out)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


def mx_reference(x):
    """(values, scale bytes) of x [M, K] on the CPU in 64 bits, by search over the eight elements"""
    x = x.detach().cpu().double()
    M, K = x.shape
    v = torch.nn.functional.pad(x, (0, -K % 32)).view(M, -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -149))) - 2
    e = torch.where(top.isfinite() & (top > 0), e, torch.zeros_like(e) - 127).clamp(min=-127)
    a = (v.abs() / torch.exp2(e)).nan_to_num(0, 0, 0)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    code = torch.zeros(a.shape, dtype=torch.long)
    for c in range(1, 8):
        mid = (grid[c] + grid[c - 1]) / 2
        code = torch.where((a > mid) | ((a == mid) & (c % 2 == 0)), torch.full_like(code, c), code)
    val = torch.copysign(grid[code], v) * torch.exp2(e)
    bad = ~top.isfinite()
    val = torch.where(bad, torch.full_like(val, math.nan), val)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(-1).to(torch.uint8)
    return val.view(M, -1)[:, :K], byte


def untile_scales(s, M, K):
    G, S = s.shape[:2]
    t = s.cpu().view(G, S, 2, 32, 2, 2).permute(0, 4, 3, 1, 5, 2).reshape(G * 64, S * 4)
    return t[:M, :-(-K // 32)], t


def untile_codes(q):
    G, S = q.shape[:2]
    c = torch.stack((q.cpu() & 15, q.cpu() >> 4), -1).view(G, S, 2, 2, 2, 32, 32)
    return c.permute(0, 2, 5, 1, 3, 4, 6).reshape(G * 64, S * 128)


def same(a, b):
    a, b = a.detach().cpu().double(), b.double()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))


def check_quant(ops, x):
    M, K = x.shape
    q, s = ops.quant_mxfp4(x)
    val, byte = mx_reference(x)
    got, whole = untile_scales(s, M, K)
    assert torch.equal(got, byte)
    codes = untile_codes(q)
    assert not codes[M:].any() and not codes[:, K:].any()          # the padding is zeros
    assert not whole[M:].any() and not whole[:, -(-K // 32):].any()
    assert same(ops.dequant_mxfp4(q, s, M, K, F32), val)
    assert same(ops.dequant_mxfp4(q, s, M, K), val)                # exact in bf16 too
    return q, s


@pytest.mark.parametrize("t", (F32, BF16, F16))
@pytest.mark.parametrize("M,K", [(1, 1), (1, 31), (2, 32), (3, 33), (63, 64), (64, 128), (65, 129),
                                 (7, 1000), (130, 257), (257, 1280), (31, 5120)])
def test_quantise(ops, M, K, t):
    g = torch.Generator().manual_seed(M * 1000 + K)
    x = torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))
    check_quant(ops, x.to(t).to(DEV))


def test_every_tie_and_border(ops):
    """quarters around all midpoints, at scales over the whole exponent range"""
    base = torch.arange(-32, 32).float() / 4
    rows = []
    for e in (-149, -140, -127, -126, -100, -3, 0, 5, 60, 100, 124):
        r = base.view(2, 32).clone()
        r[:, 0] = 7.75
        rows.append(torch.ldexp(r.double(), torch.tensor(e)).float().view(-1))
    check_quant(ops, torch.stack(rows).to(DEV))


def test_ends_of_the_range(ops):
    big = torch.finfo(F32).max
    x = torch.zeros(8, 64)
    x[0, 3], x[0, 40] = big, -big
    x[1, 1] = 1e-45
    x[2, :32] = torch.tensor(2.0 ** -126)
    x[3, 5] = 2.0 ** -125
    x[4, :] = -0.0
    x[5, 2] = 2.0 ** 127
    x[6, 33] = 1 - 2.0 ** -24
    check_quant(ops, x.to(DEV))
    check_quant(ops, x.to(BF16).to(DEV))
    y = torch.zeros(3, 40)
    y[0, 1], y[1, 2], y[2, 39] = 65504, 6e-8, -2.0 ** -14
    check_quant(ops, y.to(F16).to(DEV))


def test_nonfinite_blocks(ops):
    for t in (F32, BF16, F16):
        x = torch.randn(5, 96)
        x[0, 3], x[1, 40], x[4, 95] = math.nan, math.inf, -math.inf
        q, s = check_quant(ops, x.to(t).to(DEV))
        w, ws = ops.quant_mxfp4(torch.randn(10, 96, device=DEV))
        y = ops.linear_mxfp4(x.to(t).to(DEV), w, ws, 10)
        assert y[[0, 1, 4]].isnan().all() and y[[2, 3]].isfinite().all()


def test_strided_and_misaligned_rows(ops):
    wide = torch.randn(70, 300, device=DEV)
    for t in (F32, BF16, F16):
        w = wide.to(t)
        check_quant(ops, w[:, 1:1 + 131])
        check_quant(ops, w[::2, 8:264])
        check_quant(ops, w.t())
        check_quant(ops, w[:1].expand(5, 300))


def test_empty(ops):
    q, s = ops.quant_mxfp4(torch.empty(0, 64, device=DEV))
    assert q.shape == (0, 1, 4, 64, 16) and s.shape == (0, 1, 64, 4)
    assert ops.dequant_mxfp4(q, s, 0, 64).shape == (0, 64)
    w, ws = ops.quant_mxfp4(torch.randn(10, 64, device=DEV))
    assert ops.linear_mxfp4(torch.empty(2, 0, 64, device=DEV), w, ws, 10).shape == (2, 0, 10)
    assert ops.linear_mxfp4_dx(torch.empty(0, 10, device=DEV, dtype=BF16), w, ws, 64).shape == (0, 64)


def product(x, w, b):
    xv, wv = mx_reference(x)[0].to(DEV), mx_reference(w)[0].to(DEV)
    y, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if b is not None:
        y, size = y + b.double(), size + b.double().abs()
    return y, size


def check_linear(ops, x, w, b):
    K, N = x.shape[-1], w.shape[0]
    wq, ws = ops.quant_mxfp4(w)
    y = ops.linear_mxfp4(x, wq, ws, N, b)
    ref, size = product(x, w, b)
    assert y.dtype == BF16 and y.shape == (x.shape[0], N)
    assert ((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (K + 1) * 2.0 ** -23 * size).all()
    return y


def matrices(M, N, K, seed=0):
    g = torch.Generator().manual_seed(seed + M * 31 + N * 7 + K)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    w = torch.randn(N, K, generator=g) / math.sqrt(K)
    b = torch.randn(N, generator=g).to(BF16)
    return x.to(DEV), w.to(DEV), b.to(DEV)


# single rows, a few, every tile's edges, widths in and out of the blocks of 32 / 64 / 128 / 256
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 64, 32), (1, 5120, 1280), (2, 100, 100), (4, 33, 4096),
                                   (5, 1280, 640), (16, 513, 384), (31, 257, 96), (32, 256, 512),
                                   (33, 320, 513), (64, 64, 128), (65, 129, 257), (127, 255, 1000),
                                   (128, 128, 256), (129, 300, 640), (255, 511, 896), (256, 256, 1024),
                                   (257, 513, 1152), (300, 1280, 2048), (512, 768, 640),
                                   (1000, 1000, 1000), (2049, 520, 320), (5300, 5376, 128),
                                   (6000, 5000, 200), (9, 200, 14000), (1, 100, 33000), (33, 64, 9000),
                                   (65, 6209, 257), (127, 6400, 130), (129, 5119, 640), (257, 2500, 1152),
                                   (32, 12320, 384), (21, 17000, 96), (300, 100, 14000), (2000, 100, 513),
                                   (1500, 500, 2600), (1500, 500, 2400), (16385, 20, 40)])
def test_linear(ops, M, N, K):
    x, w, b = matrices(M, N, K)
    check_linear(ops, x.to(BF16), w, b)
    check_linear(ops, x, w, None)
    check_linear(ops, x.to(F16), w.to(BF16), b)


def exact_matrices(M, N, K, seed=0):
    """elements of e2m1 with a 4 or a 6 in every block, so that all scales are 2^0"""
    g = torch.Generator().manual_seed(seed + M + N + K)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6])

    def one(r):
        m = grid[torch.randint(0, 8, (r, K), generator=g)] * (1 - 2.0 * torch.randint(0, 2, (r, K), generator=g))
        m[:, ::32] = 4.0
        return m
    return one(M).to(DEV), one(N).to(DEV)


@pytest.mark.parametrize("M,N,K", [(1, 160, 5120), (3, 512, 1024), (17, 96, 640), (40, 130, 2048),
                                   (130, 258, 4096), (300, 200, 5120), (512, 512, 128), (770, 1030, 1152),
                                   (6, 320, 5120), (64, 320, 2200), (5500, 5632, 640), (5500, 5600, 384),
                                   (512, 1280, 2688), (384, 2048, 640), (1023, 129, 4100), (12, 16500, 300),
                                   (4096, 4096, 5120), (3900, 4000, 5000), (4091, 3975, 5003), (4095, 4097, 8192)])
def test_linear_to_the_bit(ops, M, N, K):
    x, w = exact_matrices(M, N, K)
    y = ops.linear_mxfp4(x.to(BF16), *ops.quant_mxfp4(w), N)
    assert torch.equal(y, (x.double() @ w.double().t()).float().to(BF16))


@pytest.mark.parametrize("M,N,K", [(1, 8, 32), (3, 100, 100), (33, 1280, 96), (300, 333, 260), (512, 640, 1000),
                                   (1, 1, 1), (2, 13312, 96), (1, 5120, 5120), (32, 65, 129), (33, 64, 33),
                                   (64, 1000, 640), (65, 4100, 31), (129, 257, 2049), (2000, 33, 200),
                                   (2000, 200, 1100), (1030, 133, 1111), (8200, 64, 160), (40, 300, 16400),
                                   (1500, 320, 1280), (4100, 97, 999), (3, 64, 40000), (64, 70, 33000)])
def test_gradient_of_x(ops, M, N, K):
    """dx = dy W: K bf16 products a row, fp32 sums, one rounding"""
    _, w, _ = matrices(M, N, K)
    dy = torch.randn(M, N, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    wq, ws = ops.quant_mxfp4(w)
    dx = ops.linear_mxfp4_dx(dy, wq, ws, K)
    wv = mx_reference(w)[0].to(DEV)
    ref, size = dy.double() @ wv, dy.double().abs() @ wv.abs()
    assert dx.dtype == BF16 and dx.shape == (M, K)
    assert ((dx.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (N + 1) * 2.0 ** -23 * size).all()
    wide = torch.zeros(M, N + 5, dtype=BF16, device=DEV)
    wide[:, 3:3 + N] = dy
    assert torch.equal(ops.linear_mxfp4_dx(wide[:, 3:3 + N], wq, ws, K), dx)
    for t in (F32, F16):                       # taken in bf16
        assert torch.equal(ops.linear_mxfp4_dx(dy.to(t), wq, ws, K), ops.linear_mxfp4_dx(dy.to(t).to(BF16), wq, ws, K))
    same_row = dy[:1].expand(M, N)
    assert torch.equal(ops.linear_mxfp4_dx(same_row, wq, ws, K), ops.linear_mxfp4_dx(same_row.contiguous(), wq, ws, K))


def test_gradient_of_x_takes_what_a_row_holds(ops):
    """one row's NaN or infinity reaches no other row; a NaN block of W reaches its columns of dx alone"""
    _, w, _ = matrices(70, 300, 200)
    wq, ws = ops.quant_mxfp4(w)
    for M in (5, 40, 70, 4000):
        dy = torch.randn(M, 300, generator=torch.Generator().manual_seed(M)).to(BF16).to(DEV)
        want = ops.linear_mxfp4_dx(dy, wq, ws, 200)
        bad = dy.clone()
        bad[M // 2, 17] = math.nan
        bad[M - 1, 299] = math.inf
        got = ops.linear_mxfp4_dx(bad, wq, ws, 200)
        keep = torch.ones(M, dtype=torch.bool, device=DEV)
        keep[M // 2] = keep[M - 1] = False
        assert torch.equal(got[keep], want[keep])
        assert got[M // 2].isnan().all() and not got[M - 1].isfinite().any()
    w[3, 40] = math.nan
    wq, ws = ops.quant_mxfp4(w)
    for M in (5, 70, 4000):
        got = ops.linear_mxfp4_dx(torch.ones(M, 300, dtype=BF16, device=DEV), wq, ws, 200)
        assert got[:, 32:64].isnan().all() and got[:, :32].isfinite().all() and got[:, 64:].isfinite().all()


def test_leading_axes_and_strides(ops):
    x, w, b = matrices(30, 200, 160)
    wq, ws = ops.quant_mxfp4(w)
    want = ops.linear_mxfp4(x, wq, ws, 200, b)
    assert torch.equal(ops.linear_mxfp4(x.view(2, 3, 5, 160), wq, ws, 200, b).view(30, 200), want)
    assert torch.equal(ops.linear_mxfp4(x[4], wq, ws, 200, b), want[4])
    wide = torch.randn(30, 171, device=DEV)
    wide[:, 7:167] = x
    assert torch.equal(ops.linear_mxfp4(wide[:, 7:167], wq, ws, 200, b), want)
    assert torch.equal(ops.linear_mxfp4(x.view(5, 6, 160).transpose(0, 1), wq, ws, 200, b),
                       want.view(5, 6, 200).transpose(0, 1))


def test_a_row_is_the_same_in_any_batch(ops):
    """a padded or a larger batch changes no row's result beyond the order of its fp32 sums"""
    x, w, b = matrices(300, 384, 1024)
    wq, ws = ops.quant_mxfp4(w)
    whole = ops.linear_mxfp4(x, wq, ws, 384, b)
    ref, size = product(x, w, b)
    for m in (1, 4, 9, 32, 40, 128, 256):
        part = ops.linear_mxfp4(x[:m], wq, ws, 384, b)
        lim = 2.0 ** -8 * ref[:m].abs() + 1025 * 2.0 ** -23 * size[:m]
        assert ((part.double() - ref[:m]).abs() <= lim).all()
        assert torch.equal(part, ops.linear_mxfp4(x[:m].clone(), wq, ws, 384, b))
    assert torch.equal(whole, ops.linear_mxfp4(x, wq, ws, 384, b))


def test_zero_rows_give_the_bias(ops):
    x, w, b = matrices(70, 130, 192)
    x[5] = 0
    x[69] = 0
    y = ops.linear_mxfp4(x, *ops.quant_mxfp4(w), 130, b)
    assert torch.equal(y[5], b) and torch.equal(y[69], b)


def test_captured_replayed_and_on_another_stream(ops):
    for M in (1, 20, 300, 1500):
        x, w, b = matrices(M, 640, 512)
        wq, ws = ops.quant_mxfp4(w)
        dy = torch.randn(M, 640, device=DEV).to(BF16)

        def step():
            return ops.linear_mxfp4(x, wq, ws, 640, b), ops.linear_mxfp4_dx(dy, wq, ws, 512)
        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, got))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        for k in range(3):
            x.copy_(torch.randn(M, 512, device=DEV) * (k + 1))
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(want, got)), (M, k)


def test_two_graphs_replayed_in_turn(ops):
    built = []
    for M in (300, 40, 3):
        x, w, b = matrices(M, 384, 640)
        wq, ws = ops.quant_mxfp4(w)
        want = ops.linear_mxfp4(x, wq, ws, 384, b)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.linear_mxfp4(x, wq, ws, 384, b)
        built.append((graph, got, want, (x, wq, ws, b)))
    for order in ((0, 1, 2), (2, 0, 1, 0), (1, 1, 2)):
        for i in order:
            built[i][1].zero_()
            built[i][0].replay()
        ops.linear_mxfp4(built[0][3][0] * 2, *built[0][3][1:3], 384)
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(built[i][1], built[i][2])


def test_weights_with_a_nan_block(ops):
    """its own column of y is NaN, and no other"""
    for M in (2, 50, 200):
        x, w, b = matrices(M, 150, 200)
        w[70, 40] = math.nan
        y = ops.linear_mxfp4(x, *ops.quant_mxfp4(w), 150, b)
        bad = y.isnan()
        assert bad[:, 70].all() and int(bad.sum()) == M


def test_autograd_op(ops):
    from prfl_amd import custom_ops
    x, w, b = matrices(12, 72, 96)
    wq, ws = ops.quant_mxfp4(w)
    xl, bl = x.view(3, 4, 96).detach().requires_grad_(), b.detach().requires_grad_()
    y = custom_ops.linear_mxfp4(xl, wq, ws, 72, bl)
    dy = torch.randn(3, 4, 72, generator=torch.Generator().manual_seed(3)).to(BF16).to(DEV)
    dx, db = torch.autograd.grad(y, (xl, bl), dy)
    assert dx.dtype == F32 and dx.shape == xl.shape and db.dtype == BF16
    assert torch.equal(dx.view(12, 96), ops.linear_mxfp4_dx(dy.view(12, 72), wq, ws, 96).float())
    ref = dy.double().view(12, 72).sum(0)
    assert ((db.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 12 * 2.0 ** -24 * dy.double().abs().view(
        12, 72).sum(0)).all()
    assert torch.autograd.grad(custom_ops.linear_mxfp4(xl, wq, ws, 72, None), xl, dy)[0].shape == xl.shape
    w2, ws2 = ops.quant_mxfp4(w[:71])                             # a width that the column sums pad
    b2 = b[:71].clone().requires_grad_()
    db = torch.autograd.grad(custom_ops.linear_mxfp4(xl, w2, ws2, 71, b2), b2, dy[..., :71])[0]
    assert ((db.double() - ref[:71]).abs() <= 2.0 ** -8 * ref[:71].abs() + 12 * 2.0 ** -24 * dy.double().abs().view(
        12, 72).sum(0)[:71]).all()
    none = custom_ops.linear_mxfp4(xl[:0], wq, ws, 72, bl)
    dx, db = torch.autograd.grad(none.sum(), (xl, bl))
    assert not dx.any() and not db.any()
    torch.library.opcheck(torch.ops.prfl.linear_mxfp4, (xl, wq, ws, 72, bl))
