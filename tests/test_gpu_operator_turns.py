"""Calls that take a kernel through more than one turn: wide layer norm rows of which a workgroup gets several, lists
of more than a thousand gradients, and a bias gradient over views at any alignment."""
import itertools

import pytest
import torch

from test_gpu_grads import check_clip, grads
from test_gpu_layer_norm import check, inputs

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


# one launch with one workgroup, one row a workgroup, and several rows for each of them
@pytest.mark.parametrize("rows", (2, 4, 5, 300, 700))
@pytest.mark.parametrize("C", (5120, 6077, 8192, 8200, 12001, 16384))
@pytest.mark.parametrize("xt,yt", itertools.product((F32, BF16, F16), repeat=2))
def test_wide_rows(ops, C, rows, xt, yt):
    x, w, b, dy = inputs((rows, C), xt, seed=C + rows)
    check(ops, x, w, b, dy, out_dtype=yt)


@pytest.mark.parametrize("rows,C", ((40000, 64), (20000, 392), (9000, 1280), (5000, 5120), (3000, 9000)))
@pytest.mark.parametrize("t", (F32, BF16))
def test_many_turns(ops, rows, C, t):
    x, w, b, dy = inputs((rows, C), t, seed=C)
    check(ops, x, w, b, dy)


@pytest.mark.parametrize("count", (1024, 1025, 3000))
def test_clip_of_very_many_tensors(ops, count):
    src = grads([(i * 37 % 300 + 1,) for i in range(count)], (F32, BF16, F16), seed=count)
    got = [t.clone() for t in src]
    check_clip(got, ops.clip_grads(got, 0.1), src, 0.1)
    out = [torch.full_like(t, 7, dtype=F32) for t in src]
    check_clip(out, ops.clip_grads(src, 0.1, out=out), src, 0.1)


@pytest.mark.parametrize("M,N", ((1, 1), (3, 7), (64, 8), (65, 129), (1000, 333), (8190, 640), (70001, 40)))
def test_bias_gradient(ops, M, N):
    from prfl_amd import custom_ops
    wq, ws = ops.quant_mxfp4(torch.randn(N, 32, device=DEV))
    x, bias = torch.randn(M, 32, device=DEV), torch.zeros(N, device=DEV, dtype=BF16, requires_grad=True)
    flat = torch.randn(M * N + 3, generator=torch.Generator().manual_seed(N)).to(BF16).to(DEV)
    for off in (0, 1, 3):                                            # dense, at any alignment
        dy = flat[off:off + M * N].view(M, N)
        db, = torch.autograd.grad(custom_ops.linear_mxfp4(x, wq, ws, N, bias), bias, dy)
        want, size = dy.double().sum(0), dy.double().abs().sum(0)
        assert ((db.double() - want).abs() <= 2.0 ** -8 * want.abs() + M * 2.0 ** -24 * size).all()
    db, = torch.autograd.grad(custom_ops.linear_mxfp4(x, wq, ws, N, bias).sum(0), bias, flat[:N])   # one row for all
    want = flat[:N].double() * M
    assert ((db.double() - want).abs() <= 2.0 ** -8 * want.abs() + M * 2.0 ** -24 * want.abs()).all()
