"""layer_norm, the fp4 operators and gradient clipping on the CPU host: registered ops and their
fake shapes, no CPU kernel, and every refusal before anything is launched (Python checks on fake
device tensors, C entries by their return code)."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64
NEW = ["layer_norm", "layer_norm_backward", "linear_mxfp4", "linear_mxfp4_backward"]


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import custom_ops, ops as _ops  # noqa: F401
    return _ops


def test_registered_without_a_cpu_kernel(ops):
    for name in NEW:
        assert str(getattr(torch.ops.prfl, name).default._schema).startswith(f"prfl::{name}(")
    x = torch.zeros(3, 8)
    with pytest.raises(NotImplementedError):
        torch.ops.prfl.layer_norm(x, None, None, 1e-5, None)
    with pytest.raises(NotImplementedError):
        torch.ops.prfl.linear_mxfp4(x, x, x, 8, None)
    for f in (lambda: ops.layer_norm_fwd(x), lambda: ops.quant_mxfp4(x), lambda: ops.clip_grads([x], 1.0),
              lambda: ops.grads_sumsq([x])):
        with pytest.raises(RuntimeError, match="MI355X"):
            f()


def test_fake_shapes(ops):
    with FakeTensorMode():
        x = torch.empty(2, 5, 96, device="cuda", dtype=BF16)
        y, m, r = torch.ops.prfl.layer_norm(x, None, None, 1e-5, F32)
        assert y.shape == x.shape and y.dtype == F32 and m.shape == r.shape == (2, 5)
        dx, dw, db = torch.ops.prfl.layer_norm_backward(y, x, m, r, None, True, False, True)
        assert dx.shape == x.shape and dx.dtype == BF16 and dw.numel() == 0 and db.shape == (96,)
        q, s = (torch.empty(*v, device="cuda", dtype=torch.uint8) for v in ((2, 1, 4, 64, 16), (2, 1, 64, 4)))
        y = torch.ops.prfl.linear_mxfp4(x, q, s, 100, None)
        assert y.shape == (2, 5, 100) and y.dtype == BF16
        dx, db = torch.ops.prfl.linear_mxfp4_backward(y, q, s, 96, True, True)
        assert dx.shape == (2, 5, 96) and db.shape == (100,) and db.dtype == F32


def refuses(f, what=ValueError):
    with pytest.raises(what):
        f()


def test_layer_norm_refusals(ops):
    with FakeTensorMode():
        E = lambda *s, t=F32: torch.empty(s, device="cuda", dtype=t)  # noqa: E731
        x, m = E(4, 32), E(4)
        refuses(lambda: ops.layer_norm_fwd(E()))
        refuses(lambda: ops.layer_norm_fwd(E(4, 0)))
        refuses(lambda: ops.layer_norm_fwd(E(4, 16385)))
        refuses(lambda: ops.layer_norm_fwd(E(4, 32, t=F64)))
        refuses(lambda: ops.layer_norm_fwd(x, out_dtype=F64))
        refuses(lambda: ops.layer_norm_fwd(x, E(31)))
        refuses(lambda: ops.layer_norm_fwd(x, E(32), E(1, 32)))
        refuses(lambda: ops.layer_norm_fwd(x, E(32), E(32, t=BF16)))
        refuses(lambda: ops.layer_norm_fwd(x, E(32, t=F64)))
        refuses(lambda: ops.layer_norm_fwd(x, eps=-1.0))
        refuses(lambda: ops.layer_norm_fwd(x, eps=float("nan")))
        refuses(lambda: ops.layer_norm_fwd(x, torch.empty(32)), RuntimeError)
        refuses(lambda: ops.layer_norm_fwd(x, torch.empty(32, device="cuda:1")))
        refuses(lambda: ops.layer_norm_bwd(E(4, 31), x, m, m))
        refuses(lambda: ops.layer_norm_bwd(x, x, E(3), m))
        refuses(lambda: ops.layer_norm_bwd(x, x, m, E(4, t=BF16)))
        refuses(lambda: ops.layer_norm_bwd(x, x, m, m, E(8)))
        refuses(lambda: ops.layer_norm_bwd(x, x, m, m, E(32, t=F64)))
        refuses(lambda: ops.layer_norm_bwd(E(4, 32, t=F64), x, m, m))


def test_mxfp4_refusals(ops):
    with FakeTensorMode():
        E = lambda *s, t=F32: torch.empty(s, device="cuda", dtype=t)  # noqa: E731
        U = lambda *s: E(*s, t=torch.uint8)  # noqa: E731
        q, s = U(2, 1, 4, 64, 16), U(2, 1, 64, 4)                 # a [65..128, 1..128] matrix
        refuses(lambda: ops.quant_mxfp4(E(8)))
        refuses(lambda: ops.quant_mxfp4(E(8, 0)))
        refuses(lambda: ops.quant_mxfp4(E(8, 8, t=F64)))
        refuses(lambda: ops.dequant_mxfp4(q, s, 64, 100))
        refuses(lambda: ops.dequant_mxfp4(q, s, 100, 129))
        refuses(lambda: ops.dequant_mxfp4(q, s, 100, 100, F16))
        refuses(lambda: ops.dequant_mxfp4(q, U(2, 1, 4, 64), 100, 100))
        refuses(lambda: ops.dequant_mxfp4(E(2, 1, 4, 64, 16), s, 100, 100))
        refuses(lambda: ops.dequant_mxfp4(q.transpose(2, 3).contiguous().transpose(2, 3), s, 100, 100))
        refuses(lambda: ops.linear_mxfp4(E(), q, s, 100))
        refuses(lambda: ops.linear_mxfp4(E(3, 0), q, s, 100))
        refuses(lambda: ops.linear_mxfp4(E(3, 200), q, s, 100))
        refuses(lambda: ops.linear_mxfp4(E(3, 100, t=F64), q, s, 100))
        refuses(lambda: ops.linear_mxfp4(E(3, 100), q, s, 129))
        refuses(lambda: ops.linear_mxfp4(E(3, 100), q, s, 0))
        refuses(lambda: ops.linear_mxfp4(E(3, 100), q, s, 100, E(100)))
        refuses(lambda: ops.linear_mxfp4(E(3, 100), q, s, 100, E(99, t=BF16)))
        refuses(lambda: ops.linear_mxfp4(E(3, 100), q, s, 100, E(200, t=BF16)[::2]))
        refuses(lambda: ops.linear_mxfp4(E(3, 100), q, torch.empty(2, 1, 64, 4, dtype=torch.uint8,
                                                                  device="cuda:1"), 100))
        refuses(lambda: ops.linear_mxfp4_dx(E(3, 100, t=BF16), q, s, 129))
        refuses(lambda: ops.linear_mxfp4_dx(E(3, 129, t=BF16), q, s, 100))
        refuses(lambda: ops.linear_mxfp4_dx(E(3, 100, t=F64), q, s, 100))


def test_shapes_that_only_one_direction_refused(ops):
    with FakeTensorMode():
        E = lambda *s, t=F32: torch.empty(s, device="cuda", dtype=t)  # noqa: E731
        U = lambda *s: E(*s, t=torch.uint8)  # noqa: E731
        refuses(lambda: ops.layer_norm_bwd(E(), E(), E(), E()))
        refuses(lambda: ops.layer_norm_bwd(E(4, 0), E(4, 0), E(4), E(4)))
        refuses(lambda: ops.layer_norm_bwd(E(4, 16385), E(4, 16385), E(4), E(4)))
        q, s = U(2, 1, 4, 64, 16), U(2, 1, 64, 4)
        refuses(lambda: ops.linear_mxfp4_dx(E(), q, s, 100))
        refuses(lambda: ops.linear_mxfp4_dx(E(3, 0, t=BF16), q[:0], s[:0], 100))
        wide = (1 << 24) + 1
        refuses(lambda: ops.quant_mxfp4(E(1, wide)))
        refuses(lambda: ops.dequant_mxfp4(U(1, 131073, 4, 64, 16), U(1, 131073, 64, 4), 1, wide))
        refuses(lambda: ops.linear_mxfp4(E(1, wide), U(1, 131073, 4, 64, 16), U(1, 131073, 64, 4), 1))
        refuses(lambda: ops.linear_mxfp4(E(1, 8), U(262145, 1, 4, 64, 16), U(262145, 1, 64, 4), wide))
        refuses(lambda: ops.linear_mxfp4_dx(E(1, wide), U(262145, 1, 4, 64, 16), U(262145, 1, 64, 4), 8))
        refuses(lambda: ops.linear_mxfp4_dx(E(1, 8), U(1, 131073, 4, 64, 16), U(1, 131073, 64, 4), wide))


def test_clip_refusals(ops):
    refuses(lambda: ops.clip_grads([], 1.0))
    with FakeTensorMode():
        E = lambda *s, t=F32: torch.empty(s, device="cuda", dtype=t)  # noqa: E731
        a = [E(4, 4), E(3)]
        refuses(lambda: ops.clip_grads(a, -1.0))
        refuses(lambda: ops.clip_grads(a, float("nan")))
        refuses(lambda: ops.clip_grads(a, 1.0, eps=-1e-6))
        refuses(lambda: ops.clip_grads([E(4, t=F64)], 1.0))
        refuses(lambda: ops.clip_grads([E(4, 8)[:, :4]], 1.0))             # gaps
        refuses(lambda: ops.clip_grads([E(1).expand(4)], 1.0))             # one element four times
        refuses(lambda: ops.clip_grads([a[0], torch.empty(3, device="cuda:1")], 1.0))
        refuses(lambda: ops.clip_grads(a, 1.0, out=[E(4, 4)]))
        refuses(lambda: ops.clip_grads(a, 1.0, out=[E(4, 4), E(4)]))
        refuses(lambda: ops.clip_grads(a, 1.0, out=[E(4, 4).t(), E(3)]))
        refuses(lambda: ops.clip_grads(a, 1.0, out=[E(4, 4), E(3, t=BF16)]))
        refuses(lambda: ops.grads_sumsq([torch.empty(4, device="cuda", dtype=torch.int32)]))


def test_overlapping_gradients_are_refused(ops, monkeypatch):
    """by address: the check needs real memory, so CPU tensors stand in for the device's"""
    from prfl_amd import _lib
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "call_on", lambda *a: pytest.fail("launched"))
    flat = torch.zeros(100)
    refuses(lambda: ops.clip_grads([flat, flat], 1.0))
    refuses(lambda: ops.clip_grads([flat[:50], flat[49:]], 1.0))
    refuses(lambda: ops.clip_grads([flat[60:], flat[20:40], flat[:10], flat[39:50], flat[90:91]], 1.0))
    refuses(lambda: ops.clip_grads([flat[:50]], 1.0, out=[flat[20:70]]))
    refuses(lambda: ops.clip_grads([flat[:50]], 1.0, out=[flat[:50]]))
    refuses(lambda: ops.clip_grads([flat[:5]], 1.0, sumsq=torch.zeros(1)))
    refuses(lambda: ops.clip_grads([flat[:5]], 1.0, sumsq=torch.zeros(2, dtype=F64)))


def test_gradients_apart_are_taken(ops, monkeypatch):
    from prfl_amd import _lib
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    calls = []
    monkeypatch.setattr(_lib, "call_on", lambda *a: calls.append(a))
    flat, half = torch.zeros(100), torch.zeros(64, dtype=BF16)
    ops.clip_grads([flat[60:], flat[20:40].view(4, 5).t(), flat[:0], flat[:10], flat[40:60], half[1:33], half[33:]], 1.0)
    ops.clip_grads([flat[:10], half[:8]], 1.0, out=[flat[10:20], flat[20:28]])
    ops.clip_grads([flat[30:30], flat[:50]], 1.0, out=[flat[:0], flat[50:]])
    assert len(calls) == 3


def test_tensors_clipped_into_count_as_written(ops, monkeypatch):
    from prfl_amd import _lib
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "call_on", lambda *a: 0)
    grads, out = [torch.ones(5, dtype=BF16), torch.ones(3, dtype=BF16)], [torch.zeros(5), torch.zeros(3)]
    ops.clip_grads(grads, 1.0, out=out)
    assert [t._version for t in grads + out] == [0, 0, 1, 1]
    ops.clip_grads(grads, 1.0)
    assert [t._version for t in grads] == [0, 0]


def test_sparse_gradients_are_refused(ops, monkeypatch):
    from prfl_amd import _lib
    monkeypatch.setattr(_lib, "require_gpu", lambda *t: None)
    monkeypatch.setattr(_lib, "call_on", lambda *a: pytest.fail("launched"))
    refuses(lambda: ops.clip_grads([torch.zeros(3), torch.eye(3).to_sparse()], 1.0))
    refuses(lambda: ops.grads_sumsq([torch.eye(3).to_sparse_csr()]))
    refuses(lambda: ops.clip_grads([torch.zeros(3)], 1.0, out=[torch.zeros(3).to_sparse()]))


def test_empty_list_of_gradients(ops):
    from prfl_amd import optim
    assert float(optim.clip_grads_([torch.nn.Parameter(torch.zeros(2))])) == 0
    refuses(lambda: ops.grads_sumsq([]))


def test_c_entries_refuse(ops):
    """bad arguments come back as hipErrorInvalidValue (1) before any launch; p is never read"""
    from prfl_amd import _lib
    lib = _lib.load()
    mem = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(mem) + 63) // 64 * 64

    def ln(x=p, xt=0, ldx=32, rows=4, C=32, wt=0, eps=1e-5, y=p, yt=0, ldy=32, mean=p):
        return lib.prfl_layer_norm_fwd(x, xt, ldx, rows, C, p, p, wt, eps, y, yt, ldy, mean, p, None)
    for bad in (dict(x=None), dict(y=None), dict(mean=None), dict(xt=3), dict(xt=-1), dict(yt=3), dict(wt=3),
                dict(C=0), dict(C=16385), dict(rows=-1), dict(ldy=31), dict(ldx=-1), dict(eps=-1.0),
                dict(eps=float("nan"))):
        assert ln(**bad) == 1, bad
    assert ln(rows=0) == 0
    bwd = lambda **k: lib.prfl_layer_norm_bwd(  # noqa: E731
        *{**dict(dy=p, yt=0, lddy=32, x=p, xt=0, ldx=32, mean=p, rstd=p, rows=4, C=32, w=p, wt=0, dx=p,
                 lddx=32, dw=p, db=p, part=p, st=None), **k}.values())
    for bad in (dict(part=None, rows=100), dict(C=16385), dict(xt=3), dict(lddx=31), dict(dy=None), dict(rows=-1)):
        assert bwd(**bad) == 1, bad
    assert lib.prfl_layer_norm_parts(-1, 32, 0) == 0 and lib.prfl_layer_norm_parts(4, 0, 0) == 0

    quant = lambda x=p, t=0, ld=32, M=4, K=32, q=p, s=p: lib.prfl_quant_mxfp4(x, t, ld, M, K, q, s, None)  # noqa: E731
    for bad in (dict(x=None), dict(t=3), dict(M=-1), dict(K=0), dict(q=p + 1), dict(s=p + 2), dict(q=None),
                dict(K=(1 << 24) + 1), dict(M=1 << 40)):
        assert quant(**bad) == 1, bad
    assert quant(M=0) == 0
    deq = lambda q=p, s=p, M=4, K=32, o=p, ld=32: lib.prfl_dequant_mxfp4(q, s, M, K, o, 0, ld, None)  # noqa: E731
    for bad in (dict(q=None), dict(o=None), dict(ld=31), dict(M=-1), dict(q=p + 8)):
        assert deq(**bad) == 1, bad
    mm = lambda xq=p, xs=p, wq=p, ws=p, y=p, ld=8, M=2, N=8, K=32: lib.prfl_gemm_mxfp4(  # noqa: E731
        xq, xs, wq, ws, None, y, ld, M, N, K, None)
    for bad in (dict(xq=None), dict(xq=p + 8), dict(ws=p + 1), dict(y=None), dict(ld=7), dict(N=0), dict(M=-1),
                dict(K=0)):
        assert mm(**bad) == 1, bad
    assert mm(M=0) == 0
    lin = lambda x=p, t=0, ld=32, wq=p, ws=p, y=p, ldy=8, M=2, N=8, K=32, w=None, nb=0: lib.prfl_linear_mxfp4(  # noqa: E731
        x, t, ld, wq, ws, None, y, ldy, M, N, K, w, nb, None)
    assert lib.prfl_linear_mxfp4_ws_bytes(2, 32) == 0
    assert lib.prfl_linear_mxfp4_ws_bytes(65, 129) == 2 * 2 * 4352
    for bad in (dict(x=None), dict(t=3), dict(t=-1), dict(wq=p + 8), dict(ws=p + 1), dict(y=None), dict(ldy=7),
                dict(N=0), dict(M=-1), dict(K=0), dict(ld=-1), dict(M=65, K=129),
                dict(M=65, K=129, w=p, nb=2 * 2 * 4352 - 1), dict(M=65, K=129, w=p + 8, nb=2 * 2 * 4352)):
        assert lin(**bad) == 1, bad
    assert lin(M=0) == 0

    ldx = lambda dy=p, t=0, ld=8, wq=p, ws=p, dx=p, lddx=32, M=2, N=8, K=32: lib.prfl_linear_mxfp4_dx(  # noqa: E731
        dy, t, ld, wq, ws, dx, lddx, M, N, K, None)
    for bad in (dict(dy=None), dict(t=3), dict(t=-1), dict(ld=-1), dict(wq=None), dict(wq=p + 8), dict(ws=None),
                dict(dx=None), dict(lddx=31), dict(M=-1), dict(N=0), dict(K=0), dict(M=65536 * 64),
                dict(N=(1 << 24) + 1), dict(K=(1 << 24) + 1)):
        assert ldx(**bad) == 1, bad
    assert ldx(M=0) == 0
    direct = lib.prfl_linear_mxfp4_dx_direct
    assert direct(1, 8, 32) == 1 and not (direct(0, 8, 32) or direct(1, 0, 32) or direct(32760, 5120, 5120))

    n, t = (ctypes.c_int64 * 2)(4, 5), (ctypes.c_int32 * 2)(0, 1)
    at, none = (ctypes.c_void_p * 2)(p, p), (ctypes.c_void_p * 2)(p, None)
    assert lib.prfl_grads_parts(n, 2) == 2
    ss = lambda at=at, n=n, t=t, c=2, parts=2, s=p: lib.prfl_grads_sumsq(at, n, t, c, p, parts, s, None)  # noqa: E731
    for bad in (dict(at=none), dict(parts=1), dict(c=-1), dict(s=None), dict(t=(ctypes.c_int32 * 2)(0, 3)),
                dict(n=(ctypes.c_int64 * 2)(4, -1))):
        assert ss(**bad) == 1, bad
    cl = lambda at=at, out=None, c=2, ot=-1, s=p, w=None, parts=0, m=1.0, e=1e-6: lib.prfl_grads_clip(  # noqa: E731
        at, out, n, t, c, ot, s, w, parts, m, e, p, None)
    for bad in (dict(at=none), dict(out=none, ot=0), dict(ot=0), dict(out=at), dict(out=at, ot=3), dict(m=-1.0),
                dict(m=float("nan")), dict(e=-1.0), dict(c=-1), dict(s=None), dict(s=None, w=p, parts=1),
                dict(s=None, parts=2)):
        assert cl(**bad) == 1, bad
