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
