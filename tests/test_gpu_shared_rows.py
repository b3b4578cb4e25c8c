"""Products whose rows lie over one another in memory: a broadcast gradient (stride 0, as the sum over tokens
hands back) and overlapping windows (a stride below the row), against the same values in rows of their own, in 64 bits.

Tolerances: products of bf16 (and of e2m1) are exact in fp32, so an element is within one step 2^-23 of the partial
magnitudes for each of its n additions, and one rounding to bf16 (2^-8)."""
import pytest
import torch

from test_gpu_mxfp4 import mx_reference

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


def shared(rows, cols, stride, seed=0):
    """[rows, cols] with `stride` elements from row to row"""
    flat = rand(cols + (rows - 1) * stride, seed=seed)
    return flat.as_strided((rows, cols), (stride, 1))


def within(got, a, b):
    """got = a b^T of [m, n] and [k, n] matrices"""
    ref, size = a.double() @ b.double().t(), a.double().abs() @ b.double().abs().t()
    U = 2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24
    assert ((got.double() - ref).abs() <= U * ref.abs() + (a.shape[1] + 1) * 2.0 ** -23 * size).all()


# over and under the sizes at which the 256-wide tiles take over
@pytest.mark.parametrize("stride", (0, 8, 128))
@pytest.mark.parametrize("M,N,K", [(70, 64, 96), (2000, 200, 1100), (4096, 256, 1536), (4097, 320, 1544), (8190, 640, 1280)])
def test_gradient_through_an_fp4_linear(ops, M, N, K, stride):
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(K)).to(DEV) / N ** 0.5
    wq, ws = ops.quant_mxfp4(w)
    dy = shared(M, N, stride, seed=M)
    dx = ops.linear_mxfp4_dx(dy, wq, ws, K)
    within(dx, dy, mx_reference(w)[0].to(DEV).t())


@pytest.mark.parametrize("M", (70, 4096))
def test_sum_over_tokens_through_autograd(ops, M):
    from prfl_amd import custom_ops
    w = torch.randn(256, 1536, generator=torch.Generator().manual_seed(1)).to(DEV) / 16
    wq, ws = ops.quant_mxfp4(w)
    x = rand(M, 1536).requires_grad_()
    v = rand(256, seed=2)
    custom_ops.linear_mxfp4(x, wq, ws, 256, None).sum(0).backward(v)
    within(x.grad, v.expand(M, 256), mx_reference(w)[0].to(DEV).t())


@pytest.mark.parametrize("stride", (0, 8, 128))
def test_bf16_products(ops, stride):
    x, w, dy = rand(4096, 256), rand(1536, 256, seed=1), rand(4096, 1536, seed=2)
    xs, ws, ds = shared(4096, 256, stride, 3), shared(1536, 256, stride, 4), shared(4096, 1536, stride, 5)
    within(ops.linear(xs, w), xs, w)
    within(ops.linear(x, ws), x, ws)
    within(ops.linear_t(xs, w.t().contiguous()), xs, w)
    within(ops.linear_dx(ds, w), ds, w.t())
    within(ops.linear_dx(dy, ws), dy, ws.t())
    x, dy = rand(256, 2560, seed=6), rand(256, 2560, seed=7)
    xs, ds = shared(256, 2560, stride, 8), shared(256, 2560, stride, 9)
    within(ops.linear_dw(ds, x), ds.t(), x.t())
    within(ops.linear_dw(dy, xs), dy.t(), xs.t())
