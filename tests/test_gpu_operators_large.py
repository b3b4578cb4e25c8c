"""Layer norm, microscaled fp4 and clipping over tensors whose offsets pass 32 bits: the last rows of a
large call are, bit for bit, those of a call on them alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
ROWS, COLS = 420_032, 5120                     # 2.15e9 elements; whole groups of 64 rows


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    yield _ops
    torch.cuda.empty_cache()


@pytest.fixture(scope="module")
def big():
    assert ROWS * COLS > 2 ** 31
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.empty(ROWS, COLS, dtype=BF16, device=DEV)
    for part in x.split(32768):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV))
    yield x
    del x
    torch.cuda.empty_cache()


def test_layer_norm(ops, big):
    w, b = torch.randn(COLS, device=DEV), torch.randn(COLS, device=DEV)
    y, m, r = ops.layer_norm_fwd(big, w, b)
    tail, tm, tr = ops.layer_norm_fwd(big[-300:], w, b)
    assert torch.equal(y[-300:], tail) and torch.equal(m[-300:], tm) and torch.equal(r[-300:], tr)
    dx = ops.layer_norm_bwd(y, big, m, r, w, want_dw=False, want_db=False)[0]
    assert torch.equal(dx[-300:], ops.layer_norm_bwd(tail, big[-300:], tm, tr, w)[0])
    assert torch.equal(dx[:300], ops.layer_norm_bwd(y[:300], big[:300], m[:300], r[:300], w)[0])


def test_layer_norm_of_far_rows(ops, big):
    far = big.view(-1).as_strided((70, 1000), (30_700_001, 1), 3)
    assert 69 * far.stride(0) > 2 ** 30 and far.stride(0) * 2 * 70 > 2 ** 32
    dy = torch.randn(70, 1000, device=DEV).to(BF16)
    y, m, r = ops.layer_norm_fwd(far)
    near = far.contiguous()
    assert torch.equal(y, ops.layer_norm_fwd(near)[0])
    for a, c in zip(ops.layer_norm_bwd(dy, far, m, r, None, want_dw=True),
                    ops.layer_norm_bwd(dy, near, m, r, None, want_dw=True)):
        assert torch.equal(a, c)


def test_quantise_and_read_back(ops, big):
    q, s = ops.quant_mxfp4(big)
    tq, ts = ops.quant_mxfp4(big[-640:])
    assert torch.equal(q[-10:], tq) and torch.equal(s[-10:], ts)
    v = ops.dequant_mxfp4(q, s, ROWS, COLS)
    assert torch.equal(v[-640:], ops.dequant_mxfp4(tq, ts, 640, COLS))
    assert torch.equal(v[:64], ops.dequant_mxfp4(q[:1], s[:1], 64, COLS))


def test_linear(ops, big):
    """x and y of 2.15e9 elements, with a short and a long K: the last 8192 rows are those of a call on them
    (every tile adds K in the same order)"""
    b = torch.randn(COLS, device=DEV).to(BF16)
    for k in (96, COLS):
        x = big.view(-1)[:ROWS * k].view(ROWS, k)
        wq, ws = ops.quant_mxfp4(torch.randn(COLS, k, device=DEV))
        y = ops.linear_mxfp4(x, wq, ws, COLS, b)
        assert torch.equal(y[-8192:], ops.linear_mxfp4(x[-8192:], wq, ws, COLS, b))
        assert torch.equal(y[:8192], ops.linear_mxfp4(x[:8192], wq, ws, COLS, b))


def test_linear_of_far_rows(ops, big):
    far = big.view(-1).as_strided((70, 1000), (30_700_001, 1), 5)
    near = far.contiguous()
    wq, ws = ops.quant_mxfp4(torch.randn(500, 1000, device=DEV))
    vq, vs = ops.quant_mxfp4(torch.randn(1000, 300, device=DEV))
    for m in (1, 2, 40, 70):
        assert torch.equal(ops.linear_mxfp4(far[-m:], wq, ws, 500), ops.linear_mxfp4(near[-m:], wq, ws, 500))
        assert torch.equal(ops.linear_mxfp4_dx(far[-m:], vq, vs, 300), ops.linear_mxfp4_dx(near[-m:], vq, vs, 300))


def test_clip(ops, big):
    """powers of two, so that every product and sum is exact: sum of squares n, factor 1/2 to the bit"""
    g = torch.ones(ROWS * COLS, dtype=BF16, device=DEV)
    n = g.numel()
    assert float(ops.grads_sumsq([g])) == n
    ops.clip_grads([g], 0.5, eps=0.0, sumsq=torch.ones(1, dtype=torch.float64, device=DEV))
    assert bool((g == 0.5).all())
    norm = ops.clip_grads([g], 1e9)
    assert abs(float(norm) - (n / 4) ** 0.5) <= 2.0 ** -23 * (n / 4) ** 0.5
    assert bool((g == 0.5).all())
