"""The operators as one training step uses them: trained norms around frozen fp4 projections,
autograd through both, gradients clipped over all tensors, one AdamW update.

Every stage is held to the formula on the values that entered it (the kernels' own activations and
upstream gradients), so the bounds are those of one operator each; the whole is held to the plain
chain of the same roundings."""
import math

import pytest
import torch

from test_gpu_grads import check_clip
from test_gpu_layer_norm import reference, within
from test_gpu_mxfp4 import mx_reference

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


class Block(torch.nn.Module):
    """x + W2 gelu(W1 norm(x)): norm trained, W1 and W2 frozen in fp4"""

    def __init__(self, dim, hidden, seed):
        super().__init__()
        from prfl_amd import ops
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
        self.weight = torch.nn.Parameter(1 + 0.2 * r(dim))
        self.bias = torch.nn.Parameter(0.2 * r(dim))
        self.w = [r(hidden, dim) / math.sqrt(dim), r(dim, hidden) / math.sqrt(hidden)]
        self.q = [ops.quant_mxfp4(w) for w in self.w]
        self.b = [(0.1 * r(hidden)).to(BF16), (0.1 * r(dim)).to(BF16)]

    def forward(self, x, seen=None):
        from prfl_amd import custom_ops as c
        h = c.layer_norm(x, self.weight, self.bias, 1e-6, BF16)
        a = c.linear_mxfp4(h, *self.q[0], self.w[0].shape[0], self.b[0])
        g = torch.nn.functional.gelu(a, approximate="tanh")
        y = c.linear_mxfp4(g, *self.q[1], self.w[1].shape[0], self.b[1])
        if seen is not None:
            for t in (h, a, g, y):
                t.retain_grad()
            seen += [x, h, a, g, y]
        return x + y


@pytest.mark.parametrize("rows,dim,hidden", [(1, 96, 320), (75, 256, 640), (300, 200, 520)])
def test_step_through_a_frozen_trunk(rows, dim, hidden):
    from prfl_amd import ops, optim
    blocks = torch.nn.ModuleList([Block(dim, hidden, s) for s in (1, 2)])
    x = torch.randn(rows, dim, generator=torch.Generator().manual_seed(rows)).to(DEV).requires_grad_()
    seen = [[], []]
    z = x
    for b, s in zip(blocks, seen):
        z = b(z, s)
        z.retain_grad()
    loss = (z * z).mean()
    loss.backward()

    out_grad = z.grad
    for b, (xin, h, a, g, y) in reversed(list(zip(blocks, seen))):
        assert torch.equal(y.grad, out_grad.to(BF16))
        for (inp, out, k) in ((g, y, 1), (h, a, 0)):
            wv = mx_reference(b.w[k])[0].to(DEV)
            xv = mx_reference(inp)[0].to(DEV)
            n, kk = wv.shape
            ref, size = xv @ wv.t() + b.b[k].double(), xv.abs() @ wv.abs().t() + b.b[k].double().abs()
            assert ((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (kk + 1) * 2.0 ** -23 * size).all()
            d = out.grad.double()
            ref, size = d @ wv, d.abs() @ wv.abs()
            assert ((inp.grad.double() - ref).abs() <= 2.0 ** -8 * ref.abs()
                    + (n + 1) * 2.0 ** -23 * size).all()
        ref = reference(xin.detach(), b.weight.detach(), b.bias.detach(), 1e-6, h.grad)
        within(h.detach(), ref["y"], ref["ty"], "y")
        within(b.weight.grad, ref["dw"], ref["tdw"], "dw")
        within(b.bias.grad, ref["db"], ref["tdb"], "db")
        # the block's input takes the norm's gradient and the residual's: one fp32 addition more
        got = xin.grad.double() - out_grad.double()
        tol = ref["tdx"] + 2.0 ** -24 * (2 * ref["dx"].abs() + 2 * out_grad.double().abs())
        assert ((got - ref["dx"]).abs() <= tol).all()
        out_grad = xin.grad

    params = list(blocks.parameters())
    keep = [p.grad.clone() for p in params]
    limit = 0.5 * float(ops.grads_sumsq(keep).sqrt())
    norm = optim.clip_grads_(params, limit)
    check_clip([p.grad for p in params], norm, keep, limit)
    before = [p.detach().clone() for p in params]
    optim.AdamW(params, lr=1e-3).step()
    assert all(not torch.equal(p, b) and p.isfinite().all() for p, b in zip(params, before))


def test_a_token_alone_matches_its_row_of_the_batch():
    """served one at a time: the norm gives a row the same bits in any batch, so its quantised
    operand is the same too, and the product differs by the order of its fp32 sums at most"""
    from prfl_amd import custom_ops as c, ops
    b = Block(256, 640, 1)
    x = torch.randn(40, 256, generator=torch.Generator().manual_seed(0)).to(DEV)
    with torch.no_grad():
        h = c.layer_norm(x, b.weight, b.bias, 1e-6, BF16)
        one = [c.layer_norm(x[i:i + 1], b.weight, b.bias, 1e-6, BF16) for i in range(40)]
        assert torch.equal(torch.cat(one), h)
        a = torch.cat([ops.linear_mxfp4(t, *b.q[0], 640, b.b[0]) for t in one])
    xv, wv = mx_reference(h)[0].to(DEV), mx_reference(b.w[0])[0].to(DEV)
    ref, size = xv @ wv.t() + b.b[0].double(), xv.abs() @ wv.abs().t() + b.b[0].double().abs()
    assert ((a.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 257 * 2.0 ** -23 * size).all()
