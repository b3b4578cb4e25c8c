"""grads_sumsq / clip_grads / optim.clip_grads_ on the MI355X.

Tolerances: the squares are summed in 64 bits, so the norm is the 64-bit one rounded once
(2^-24, plus 2^-40 for the sum).  The factor max_norm / (norm + eps) takes three roundings and the
product one more, then one of the output's type: (U + 4.1 2^-24) of the value, and half a step of
the smallest where it is subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
u = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from prfl_amd import ops as _ops
    return _ops


def grads(shapes, dtypes, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(size * torch.randn(s, generator=g)).to(dtypes[i % len(dtypes)]).to(DEV)
            for i, s in enumerate(shapes)]


def norm64(ts):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))


def check_clip(got, norm, src, max_norm, eps=1e-6):
    want = norm64(src)
    assert abs(float(norm) - want) <= want * u * 1.001
    c = min(1.0, max_norm / (want + eps))
    for o, s in zip(got, src):
        U, fi = torch.finfo(o.dtype).eps / 2, torch.finfo(o.dtype)
        ref = s.double() * c
        err = (o.double() - ref).abs()
        assert (err <= (U + 4.1 * u) * ref.abs() + fi.smallest_normal * fi.eps).all(), (o.dtype, o.shape)


SHAPES = [(1,), (3,), (7, 5), (128, 130), (16384,), (16385,), (32768,), (40, 41, 42), (255,), (70000,)]


@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize("max_norm", (0.5, 1e6))
def test_in_place(ops, dtypes, max_norm):
    src = grads(SHAPES, dtypes)
    got = [t.clone() for t in src]
    norm = ops.clip_grads(got, max_norm)
    assert norm.shape == () and norm.dtype == F32
    check_clip(got, norm, src, max_norm)
    if max_norm > 1e5:
        assert all(torch.equal(a, b) for a, b in zip(got, src))


@pytest.mark.parametrize("to", (F32, BF16, F16))
def test_into_other_tensors(ops, to):
    src = grads(SHAPES, (F32, BF16, F16))
    keep = [t.clone() for t in src]
    for max_norm in (2.0, 1e6):
        out = [torch.full_like(t, 7, dtype=to) for t in src]
        norm = ops.clip_grads(src, max_norm, out=out)
        check_clip(out, norm, src, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(src, keep))


@pytest.mark.parametrize("count", (1, 127, 128, 129, 300))
def test_many_tensors(ops, count):
    """launches of 128 tensors, empty ones among them"""
    src = grads([(i * 37 % 900,) for i in range(count)], (F32, BF16), seed=count)
    if not sum(t.numel() for t in src):
        src[0] = torch.ones(3, device=DEV)
    got = [t.clone() for t in src]
    check_clip(got, ops.clip_grads(got, 0.1), src, 0.1)


def test_large_tensor_and_chunks(ops):
    src = grads([(5120, 5120), (2048 * 16384 + 17,)], (BF16,))
    got = [t.clone() for t in src]
    check_clip(got, ops.clip_grads(got, 1.0), src, 1.0)


def test_views_at_any_alignment(ops):
    """gradients as views of a flat buffer: neighbours stay as they were"""
    for t in (F32, BF16, F16):
        flat = torch.randn(5000, device=DEV).to(t)
        keep = flat.clone()
        views = [flat[1:1000], flat[1001:1003], flat[1005:4999]]
        norm = ops.clip_grads(views, 0.25)
        check_clip(views, norm, [keep[1:1000], keep[1001:1003], keep[1005:4999]], 0.25)
        for i in (0, 1000, 1003, 1004, 4999):
            assert flat[i] == keep[i]


def test_axes_in_another_order(ops):
    src = [torch.randn(30, 50, device=DEV).t(), torch.randn(4, 5, 6, 7, device=DEV).to(
        memory_format=torch.channels_last)]
    got = [t.clone() for t in src]
    check_clip(got, ops.clip_grads(got, 1.0), src, 1.0)


def test_far_ranges(ops):
    """squares outside fp32: the sum is in 64 bits"""
    for size in (1e25, 1e-25):
        src = grads([(1000,), (77, 33)], (F32,), size=size)
        assert abs(float(ops.clip_grads([t.clone() for t in src], 1.0)) / norm64(src) - 1) <= 1.001 * u
    s = ops.grads_sumsq(grads([(1000,)], (F32,), size=1e25))
    assert s.dtype == torch.float64 and s.shape == (1,) and s.isfinite().all()


def test_nonfinite(ops):
    src = grads([(500,), (40,)], (F32,))
    src[0][3] = float("inf")
    got = [t.clone() for t in src]
    assert float(ops.clip_grads(got, 1.0)) == math.inf
    assert got[0][3].isnan() and not got[1].any()          # inf * 0; finite * 0
    src[0][3] = float("nan")
    got = [t.clone() for t in src]
    assert math.isnan(float(ops.clip_grads(got, 1.0)))
    assert all(t.isnan().all() for t in got)


def test_zero_gradients_and_zero_limit(ops):
    got = [torch.zeros(100, device=DEV), torch.zeros(0, device=DEV)]
    assert float(ops.clip_grads(got, 1.0)) == 0 and not got[0].any()
    assert float(ops.clip_grads([torch.zeros(0, device=DEV)], 1.0)) == 0
    got = grads([(10,)], (F32,))
    ops.clip_grads(got, 0.0)
    assert not got[0].any()


def test_sum_of_shards(ops):
    """two ranks' shards: their sums of squares added, each clips its own by the whole norm"""
    a, b = grads([(1000,), (30, 9)], (F32,)), grads([(777,)], (F32,), seed=5)
    total = ops.grads_sumsq(a) + ops.grads_sumsq(b)
    want = norm64(a + b)
    for part in (a, b):
        got = [t.clone() for t in part]
        norm = ops.clip_grads(got, 1.0, sumsq=total)
        assert abs(float(norm) - want) <= 1.001 * u * want
        for o, s in zip(got, part):
            assert ((o - s.double() / (want + 1e-6)).abs() <= 5.2 * u * s.abs().double()).all()


def test_same_bits_and_another_stream(ops):
    src = grads([(5000, 333)] * 5, (BF16,))
    want = ops.grads_sumsq(src)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.grads_sumsq(src)
    side.synchronize()
    assert torch.equal(want, got)


def test_captured_and_replayed(ops):
    src = grads(SHAPES, (F32, BF16))
    buf = [t.clone() for t in src]
    out = [torch.empty_like(t, dtype=F32) for t in src]
    ops.clip_grads(buf, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(buf, 1.0, out=out)
        ops.clip_grads(buf, 3.0)
    for k in range(3):
        for t, s in zip(buf, src):
            t.copy_(s * (k + 1))
        keep = [t.clone() for t in buf]
        graph.replay()
        torch.cuda.synchronize()
        check_clip(out, norm, keep, 1.0)
        check_clip(buf, norm, keep, 3.0)


def test_optimizer_entry(ops):
    from prfl_amd import optim
    params = [torch.nn.Parameter(torch.randn(33, 65, device=DEV)), torch.nn.Parameter(
        torch.randn(65, device=DEV)), torch.nn.Parameter(torch.randn(4, device=DEV))]
    for p in params[:2]:
        p.grad = torch.randn_like(p)
    src = [p.grad.clone() for p in params[:2]]
    norm = optim.clip_grads_(params, 0.5)
    check_clip([p.grad for p in params[:2]], norm, src, 0.5)
    # as clip_grad_norm_ does, to rounding
    for p, s in zip(params, src):
        p.grad = s.clone()
    old = optim.clip_grad_norm_(params, 0.5)
    assert abs(float(old) / float(norm) - 1) < 1e-6
    assert float(optim.clip_grads_([torch.nn.Parameter(torch.zeros(3, device=DEV))], 1.0)) == 0
