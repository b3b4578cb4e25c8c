"""Calls of clip_grads / clip_grads_ beside an optimizer and at the ends of the range."""
import pytest
import torch

from test_gpu_grads import check_clip, grads

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


@pytest.mark.parametrize("overlap", (False, True))
def test_clipped_into_the_buffers_that_the_optimizer_keeps(ops, overlap):
    """bf16 gradients clipped into the fp32 ones that step(zero_grad=True) left zeroed: every step takes them"""
    from prfl_amd import optim
    model = torch.nn.Module()
    model.blocks = torch.nn.ModuleList([torch.nn.Linear(33, 20).to(DEV), torch.nn.Linear(20, 7).to(DEV)])
    params = list(model.parameters())
    twins = [p.detach().clone().requires_grad_() for p in params]
    opt, ref = optim.AdamW(params, lr=1e-2, overlap=overlap), torch.optim.AdamW(twins, lr=1e-2, weight_decay=0.01)
    if overlap:
        opt.attach(model)
    for p in params:
        p.grad = torch.zeros_like(p)
    for k in range(4):
        opt.wait()                                       # its zeroing of the buffers precedes the clip
        src = grads([tuple(p.shape) for p in params], (BF16,), seed=k)
        norm = ops.clip_grads(src, 0.5, out=[p.grad for p in params])
        check_clip([p.grad for p in params], norm, src, 0.5)
        for t, p in zip(twins, params):
            t.grad = p.grad.clone()
        opt.step(zero_grad=True)
        ref.step()
        opt.synchronize()
        for t, p in zip(twins, params):
            assert int(opt._pstep[p]) == k + 1
            # four updates of at most 10 lr each, each within 64 roundings, and the roundings of p itself
            assert ((p - t).abs() <= 4 * (0.1 * 64 + p.abs()) * 2.0 ** -24).all()


def test_clipping_in_place_wakes_no_parameter_that_had_no_gradient(ops):
    """a buffer that the optimizer zeroed and no backward touched stays passed over after a clip in place"""
    from prfl_amd import optim
    params = [torch.nn.Parameter(torch.randn(50, device=DEV)) for _ in range(2)]
    opt = optim.AdamW(params, lr=1e-2)
    for p in params:
        p.grad = torch.randn_like(p)
    optim.clip_grads_(params, 0.1)
    opt.step(zero_grad=True)
    opt.synchronize()
    keep = params[1].detach().clone()
    (params[0] ** 2).sum().backward()
    optim.clip_grads_(params, 0.1)
    opt.step(zero_grad=True)
    opt.synchronize()
    assert torch.equal(params[1], keep) and opt._pstep[params[0]] == 2 and opt._pstep[params[1]] == 1


def clipped64(src, max_norm, eps):
    total = sum(float((t.double() ** 2).sum()) for t in src) ** 0.5
    c = min(1.0, max_norm / (total + eps)) if total + eps else 1.0
    return total, [t.double() * c for t in src]


# The factor takes at most three roundings (norm, sum, quotient) and the product one; the sum under the norm is in 64
# bits.  The output's type rounds once more, and a subnormal result is within one step of the smallest.
@pytest.mark.parametrize("t,to", [(F32, None), (BF16, None), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("size,max_norm", [(1e38, 1.0), (1e38, 1e-3), (1e38, 1e30), (1e38, 1e-20), (1e38, float("inf")),
                                           (1e34, 1e-5), (1e33, 1e-12), (1e20, 1e-30), (1e-3, 1e-40), (1e5, 1e-40)])
def test_norms_and_factors_outside_fp32(ops, t, to, size, max_norm):
    """a norm past the largest fp32, and a factor below its smallest normal: the clipped values are ordinary numbers"""
    src = [s.clamp(-3, 3) * torch.tensor(size, device=DEV, dtype=t) for s in grads([(3000,), (77, 33), (1,)], (t,))]
    assert all(s.isfinite().all() for s in src)
    max_norm, eps = torch.tensor([max_norm, 1e-6], dtype=F32).tolist()          # as the kernel gets them
    total, want = clipped64(src, max_norm, eps)
    got = [s.clone() for s in src]
    out = None if to is None else [torch.full_like(s, 7, dtype=to) for s in src]
    norm = float(ops.clip_grads(got, max_norm, out=out))
    assert norm == float("inf") if total > torch.finfo(F32).max else abs(norm - total) <= 2.0 ** -23 * total
    for o, w in zip(got if out is None else out, want):
        U, fi = torch.finfo(o.dtype).eps / 2, torch.finfo(o.dtype)
        err = (o.double() - w).abs()
        assert (err <= (U + 4.1 * 2.0 ** -24) * w.abs() + fi.smallest_normal * fi.eps).all(), float(err.max())


def test_nothing_to_scale_and_nothing_allowed(ops):
    """zero gradients stay zero whatever the limit, also where limit, norm and eps are all zero"""
    for max_norm in (0.0, 1.0, float("inf")):
        for eps in (0.0, 1e-6):
            got = [torch.zeros(40, device=DEV), torch.zeros(5, 5, device=DEV, dtype=BF16)]
            assert float(ops.clip_grads(got, max_norm, eps=eps)) == 0
            assert not any(g.any() for g in got)
