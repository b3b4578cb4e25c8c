"""AdamW with moments on the host where not all of them can be pinned: the same updates to the bit."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
SHAPES = [(3000,), (257, 33), (5,), (1024, 64), (7, 11), (300, 300), (64,)]


def limit_pinning(monkeypatch, elements):
    """as if `elements` fp32 values could be pinned and then no more"""
    from prfl_amd import optim
    empty, left = torch.empty, [elements]

    def limited(*a, pin_memory=False, **k):
        if pin_memory:
            if a[0] > left[0]:
                raise RuntimeError("HIP error: out of memory\nmore of the message")
            left[0] -= a[0]
        return empty(*a, pin_memory=pin_memory, **k)
    monkeypatch.setattr(optim.torch, "empty", limited)


@pytest.mark.parametrize("slab", (1 << 29, 1 << 17, 4096))
@pytest.mark.parametrize("limit", (0, 20_000, 150_000, 1 << 40))
@pytest.mark.parametrize("overlap,duplex", ((False, True), (True, True), (True, False)))
def test_moments_that_cannot_be_pinned(monkeypatch, slab, limit, overlap, duplex):
    from prfl_amd import optim
    g = torch.Generator().manual_seed(7)
    base = [torch.randn(s, generator=g) for s in SHAPES]
    a, b = ([torch.nn.Parameter(t.clone().to(DEV)) for t in base] for _ in range(2))
    oa = optim.AdamW(a, lr=1e-2)
    monkeypatch.setattr(optim, "SLAB", slab)
    limit_pinning(monkeypatch, limit)
    ob = optim.AdamW(b, lr=1e-2, state_on_host=True, overlap=overlap, ring_slots=2)
    ob.duplex = duplex
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        ob.init_state()
    told = [w for w in seen if "pageable" in str(w.message)]
    assert len(told) == bool(ob._pageable) and ("more of the message" not in str(told[0].message) if told else True)
    if limit == 1 << 40:
        assert not ob._pageable and all(m.is_pinned() and v.is_pinned() for m, v in ob.state.values())
    if limit == 0:
        assert len(ob._pageable) == len(b) and not any(m.is_pinned() for m, _ in ob.state.values())
    for k in range(4):
        ob.wait()
        for p, q, t in zip(a, b, base):
            p.grad = torch.randn(t.shape, generator=g).to(DEV)
            q.grad = p.grad.clone()
        oa.step()
        ob.step()
    ob.synchronize()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for s, t in zip(oa.state[p], ob.state[q]):
            assert torch.equal(s.flatten().cpu(), t)
    again = optim.AdamW(b, lr=1e-2, state_on_host=True)
    again.load_state_dict(ob.state_dict())
    for q in b:
        assert all(torch.equal(s, t) for s, t in zip(ob.state[q], again.state[q]))


def test_slabs_waste_nothing_of_note():
    """moments lie side by side: as many slabs as their sum takes"""
    from prfl_amd import optim
    params = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (1000, 513, 77, 4096, 129)]
    opt = optim.AdamW(params, state_on_host=True)
    opt.init_state()
    need = sum(2 * (-(-p.numel() // 64) * 64) for p in params)
    assert {m.untyped_storage().nbytes() for pair in opt.state.values() for m in pair} == {4 * need}
    assert opt._host.need == 0 and all(m.is_pinned() and not m.any() for pair in opt.state.values() for m in pair)


class Toy(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.emb = torch.nn.Linear(16, 640)
        self.blocks = torch.nn.ModuleList([torch.nn.Linear(640, 640) for _ in range(5)])
        self.head = torch.nn.Linear(640, 3)

    def forward(self, x):
        x = self.emb(x)
        for b in self.blocks:
            x = torch.tanh(b(x))
        return self.head(x)


@pytest.mark.parametrize("limit", (0, 2_000_000))
@pytest.mark.parametrize("keep", (False, True))
def test_forward_behind_an_update_from_the_thread(monkeypatch, limit, keep):
    """forwards wait block by block for updates that are still to be issued; gradients may be dropped or are zeroed"""
    from prfl_amd import optim
    torch.manual_seed(0)
    ma = Toy().to(DEV)
    mb = Toy().to(DEV)
    mb.load_state_dict(ma.state_dict())
    x = torch.randn(32, 16, device=DEV)
    oa = optim.AdamW(list(ma.parameters()), lr=1e-2)
    monkeypatch.setattr(optim, "SLAB", 1 << 19)
    limit_pinning(monkeypatch, limit)
    ob = optim.AdamW(list(mb.parameters()), lr=1e-2, state_on_host=True, overlap=True, ring_slots=2)
    ob.attach(mb)
    with pytest.warns(UserWarning, match="pageable"):
        ob.init_state()
    assert ob._pageable and (limit == 0 or len(ob._pageable) < len(ob.params))
    for k in range(5):
        la, lb = ma(x).square().mean(), mb(x).square().mean()
        assert torch.equal(la, lb), k
        la.backward()
        lb.backward()
        if k == 2:                                       # a gradient that does not lie in order
            g = mb.blocks[3].weight.grad
            mb.blocks[3].weight.grad = g.t().contiguous().t()
        oa.step()
        ob.step(zero_grad=keep)
        oa.zero_grad()
        if not keep:
            ob.zero_grad()
        elif k == 2:
            ob.wait()
            assert not any(p.grad.any() for p in mb.parameters())
            assert not any(ob._fresh(p) for p in mb.parameters())
    ob.synchronize()
    for p, q in zip(ma.parameters(), mb.parameters()):
        assert torch.equal(p, q)
        for s, t in zip(oa.state[p], ob.state[q]):
            assert torch.equal(s.flatten().cpu(), t)


def test_what_fails_in_the_thread_is_raised_where_it_is_waited_for(monkeypatch):
    from prfl_amd import optim
    params = [torch.nn.Parameter(torch.zeros(100, device=DEV)) for _ in range(3)]
    limit_pinning(monkeypatch, 0)
    opt = optim.AdamW(params, state_on_host=True, overlap=True)
    with pytest.warns(UserWarning, match="pageable"):
        opt.init_state()
    for p in params:
        p.grad = torch.ones_like(p)

    def broken(*a, **k):
        raise ValueError("no update")
    monkeypatch.setattr(optim.ops, "adamw_", broken)
    opt.step()
    with pytest.raises(ValueError, match="no update"):
        opt.wait()
    with pytest.raises(ValueError, match="no update"):
        opt.synchronize()
