"""Tensor-level wrappers over the C ABI (shapes, strides and dtypes checked here).

All tensors are 2-D row-major views ``[rows, cols]`` with unit column stride; row strides are
passed through, so q/k/v slices of the fused QKV output need no copy.
"""
import array
import math

import torch

from . import _lib
from ._lib import F32, I32, I64, P, call, ptr, stream_ptr

BF16 = torch.bfloat16
EPI_BF16, EPI_GELU, EPI_RESID, EPI_F32, EPI_DGELU = range(5)


def _ld(t):
    assert t.dim() == 2 and t.stride(1) == 1, (tuple(t.shape), t.stride())
    return t.stride(0)


def gemm(a, b, c, M, N, K, a_kmajor=True, b_kmajor=True, epilogue=EPI_BF16, bias=None,
         gate=None, res=None, aux=None, accumulate=False, tile=0):
    """C[m][n] = sum_k A(m,k) B(n,k) (+ epilogue); see include/prfl_hip.h.  tile: 0 = by shape,
    128 / 256 (four-wave) / 512 (8-wave 256 tile) = forced (prfl_gemm_bf16_tiled)."""
    _lib.require_gpu(a, b, c)
    assert a.dtype == BF16 and b.dtype == BF16
    assert bias is None or (bias.dtype == BF16 and bias.is_contiguous())
    assert gate is None or (gate.dtype == torch.float32 and gate.is_contiguous())
    call("prfl_gemm_bf16_tiled", ptr(a), I64(_ld(a)), I32(int(a_kmajor)), ptr(b), I64(_ld(b)),
         I32(int(b_kmajor)), ptr(c), I64(_ld(c)), I64(M), I64(N), I64(K), I32(epilogue),
         ptr(bias), ptr(gate), ptr(res), I64(_ld(res) if res is not None else 0),
         I32(int(res is not None and res.dtype == BF16)), ptr(aux),
         I64(_ld(aux) if aux is not None else 0), I32(int(accumulate)), I32(tile), stream_ptr())
    return c


def linear(x, w, bias=None, epilogue=EPI_BF16, out=None, gate=None, res=None, aux=None, tile=0):
    """y = x @ w^T (+bias) with x [M,K] bf16, w [N,K] bf16 (nn.Linear layout)."""
    M, K = x.shape
    N = w.shape[0]
    if out is None:
        dt = torch.float32 if epilogue in (EPI_RESID, EPI_F32) else BF16
        out = torch.empty(M, N, dtype=dt, device=x.device)
    return gemm(x, w, out, M, N, K, True, True, epilogue, bias, gate, res, aux, tile=tile)


def linear_t(x, wt, bias=None, epilogue=EPI_BF16, out=None, gate=None, res=None, aux=None):
    """linear() on the transposed weight wt [K, N] (cast_bf16_t of the nn.Linear weight): the
    weight is then an MN-major GEMM operand; results bit-identical to linear(x, wt.t())."""
    M, K = x.shape
    N = wt.shape[1]
    if out is None:
        dt = torch.float32 if epilogue in (EPI_RESID, EPI_F32) else BF16
        out = torch.empty(M, N, dtype=dt, device=x.device)
    return gemm(x, wt, out, M, N, K, True, False, epilogue, bias, gate, res, aux)


def linear_dx(dy, w, out=None, epilogue=EPI_BF16, aux=None):
    """dX[M,K] = dY[M,N] @ W[N,K] (bf16 out; DGELU epilogue multiplies by gelu'(aux))."""
    M, N = dy.shape
    K = w.shape[1]
    if out is None:
        out = torch.empty(M, K, dtype=BF16, device=dy.device)
    return gemm(dy, w, out, M, K, N, True, False, epilogue, aux=aux)


def linear_dw(dy, x, out=None, accumulate=False):
    """dW[N,K] = dY[M,N]^T @ X[M,K] in fp32 (accumulate=True adds into `out`)."""
    M, N = dy.shape
    K = x.shape[1]
    if out is None:
        out = torch.empty(N, K, dtype=torch.float32, device=dy.device)
    return gemm(dy, x, out, N, K, M, False, False, EPI_F32, accumulate=accumulate)


FP8 = torch.float8_e4m3fn   # OCP e4m3 (gfx950), not the MI300 fnuz variant


def quant_rows_fp8(x, q=None, scale=None):
    """Per-row e4m3 quantisation: scale[m] = amax_m / 448, q = e4m3(x * 448 / amax_m).
    x [M, K] bf16 or fp32 (row-strided), K % 8 == 0, K <= 16384."""
    _lib.require_gpu(x)
    M, K = x.shape
    if q is None:
        q = torch.empty(M, K, dtype=FP8, device=x.device)
    if scale is None:
        scale = torch.empty(M, dtype=torch.float32, device=x.device)
    assert x.dtype in (BF16, torch.float32) and q.dtype == FP8
    call("prfl_quant_rows_fp8", ptr(x), I32(int(x.dtype == torch.float32)), I64(_ld(x)), I64(M),
         I64(K), ptr(q), I64(_ld(q)), ptr(scale), stream_ptr())
    return q, scale


def linear_fp8(xq, xs, wq, ws, bias=None, epilogue=EPI_BF16, out=None, gate=None, res=None,
               aux=None):
    """y = (xs * xq) @ (ws * wq)^T (+bias, epilogue) on the block-scaled fp8 MFMA: xq [M,K],
    wq [N,K] e4m3 with per-row fp32 scales xs [M], ws [N]."""
    _lib.require_gpu(xq, wq)
    assert xq.dtype == FP8 and wq.dtype == FP8
    assert bias is None or (bias.dtype == BF16 and bias.is_contiguous())
    assert gate is None or (gate.dtype == torch.float32 and gate.is_contiguous())
    M, K = xq.shape
    N = wq.shape[0]
    if out is None:
        dt = torch.float32 if epilogue == EPI_RESID else BF16
        out = torch.empty(M, N, dtype=dt, device=xq.device)
    call("prfl_gemm_fp8", ptr(xq), I64(_ld(xq)), ptr(xs), ptr(wq), I64(_ld(wq)), ptr(ws),
         ptr(out), I64(_ld(out)), I64(M), I64(N), I64(K), I32(epilogue), ptr(bias), ptr(gate),
         ptr(res), I64(_ld(res) if res is not None else 0),
         I32(int(res is not None and res.dtype == BF16)), ptr(aux),
         I64(_ld(aux) if aux is not None else 0), stream_ptr())
    return out


def cast_bf16(src, dst=None):
    """fp32 -> bf16 (round to nearest even); dst may be a contiguous slice of a larger buffer.
    A weight already stored in bf16 (a frozen trunk, train.store_frozen_bf16) is returned as
    it is, or copied into dst: its bits are what the cast of its fp32 master would give."""
    _lib.require_gpu(src)
    src = src.contiguous()
    if src.dtype == BF16:
        if dst is None:
            return src
        assert dst.is_contiguous() and dst.numel() == src.numel()
        return dst.view(src.shape).copy_(src)
    if dst is None:
        dst = torch.empty(src.shape, dtype=BF16, device=src.device)
    assert dst.is_contiguous() and dst.numel() == src.numel()
    call("prfl_cast_f32_bf16", ptr(src), ptr(dst), I64(src.numel()), stream_ptr())
    return dst


def cast_bf16_t(w, dst=None):
    """fp32 nn.Linear weight w [N, K] -> bf16 w^T [K, N] (prfl_cast_f32_bf16_t); dst may be a
    column block of a wider row-major buffer (its row stride is dst.stride(0))."""
    _lib.require_gpu(w)
    w = w.contiguous()
    N, K = w.shape
    if dst is None:
        dst = torch.empty(K, N, dtype=BF16, device=w.device)
    assert dst.shape == (K, N) and dst.stride(1) == 1
    call("prfl_cast_f32_bf16_t", ptr(w), I64(N), I64(K), I64(K), ptr(dst), I64(dst.stride(0)),
         stream_ptr())
    return dst


def colsum_reduce(part, out=None, accumulate=False):
    P_, N = part.shape
    if out is None:
        out = torch.empty(N, dtype=torch.float32, device=part.device)
        accumulate = False
    call("prfl_colsum_reduce", ptr(part), I64(P_), I64(N), ptr(out), I32(int(accumulate)),
         stream_ptr())
    return out


def colsum(x, out=None, accumulate=False):
    """sum over rows of a bf16 [L, N] matrix -> fp32 [N]."""
    L, N = x.shape
    rp = call_int("prfl_colsum_rows_per_part")
    part = torch.empty((L + rp - 1) // rp, N, dtype=torch.float32, device=x.device)
    call("prfl_colsum_bf16", ptr(x), I64(_ld(x)), I64(L), I64(N), ptr(part), stream_ptr())
    return colsum_reduce(part, out, accumulate)


_int_cache = {}


def call_int(name):
    if name not in _int_cache:
        _int_cache[name] = getattr(_lib.load(), name)()
    return _int_cache[name]


def gate_bwd(dx, y, gate, dy_out=None, want_gate=True, want_bias=True):
    """x_out = x + y*gate: dy = bf16(dx*gate), d gate = sum dx*y, d bias = sum dy."""
    L, N = dx.shape
    rp = call_int("prfl_colsum_rows_per_part")
    nb = (L + rp - 1) // rp
    if dy_out is None:
        dy_out = torch.empty(L, N, dtype=BF16, device=dx.device)
    pg = torch.empty(nb, N, dtype=torch.float32, device=dx.device) if (want_gate and y is not None) else None
    pb = torch.empty(nb, N, dtype=torch.float32, device=dx.device) if want_bias else None
    call("prfl_gate_bwd", ptr(dx), I64(_ld(dx)), ptr(y), I64(_ld(y) if y is not None else 0),
         ptr(gate), I64(L), I64(N), ptr(dy_out), I64(_ld(dy_out)), ptr(pg), ptr(pb), stream_ptr())
    dgate = colsum_reduce(pg) if pg is not None else None
    dbias = colsum_reduce(pb) if pb is not None else None
    return dy_out, dgate, dbias


def ln_mod_fwd(x, scale=None, shift=None, w=None, b=None, eps=1e-6, out=None):
    """bf16(LN(x)*(1+scale)+shift) or bf16(LN(x)*w+b); returns (out, mean, rstd)."""
    L, C = x.shape
    if out is None:
        out = torch.empty(L, C, dtype=BF16, device=x.device)
    mean = torch.empty(L, dtype=torch.float32, device=x.device)
    rstd = torch.empty(L, dtype=torch.float32, device=x.device)
    call("prfl_ln_mod_fwd", ptr(x), I32(int(x.dtype == BF16)), I64(_ld(x)), I64(L), I64(C),
         ptr(scale), ptr(shift), ptr(w), ptr(b), F32(eps), ptr(out), I64(_ld(out)), ptr(mean),
         ptr(rstd), stream_ptr())
    return out, mean, rstd


def ln_mod_bwd(dy, x, mean, rstd, dx, scale=None, w=None, accumulate=True):
    """dx (+)= LN backward; returns (sum dy*xhat, sum dy) — (d scale, d shift) or (d w, d b)."""
    L, C = x.shape
    rp = call_int("prfl_norm_rows_per_part")
    nb = (L + rp - 1) // rp
    p0 = torch.empty(nb, C, dtype=torch.float32, device=x.device)
    p1 = torch.empty(nb, C, dtype=torch.float32, device=x.device)
    call("prfl_ln_mod_bwd", ptr(dy), I64(_ld(dy)), ptr(x), I32(int(x.dtype == BF16)), I64(_ld(x)),
         ptr(mean), ptr(rstd), I64(L), I64(C), ptr(scale), ptr(w), ptr(dx), I64(_ld(dx)),
         I32(int(accumulate)), ptr(p0), ptr(p1), stream_ptr())
    return colsum_reduce(p0), colsum_reduce(p1)


# softmax_scale * log2(e) of head_dim 128: the out_scale that turns norm_q's output into the q
# operand of the *_l2q attention entries (attn_fwd / attn_bwd with q_log2=True)
L2Q_SCALE = 1.4426950408889634 / math.sqrt(128)


def rms_rope_fwd(x, w, eps=1e-6, rope_tab=None, grid=(0, 0, 0), out=None, out_scale=1.0, row0=0):
    """bf16(rope(bf16(x * rsqrt(mean x^2 + eps)) * w) * out_scale); row r is token row0 + r of
    the grid (row0 > 0: a sequence-parallel rank's shard, model.py:89-96)."""
    L, C = x.shape
    if out is None:
        out = torch.empty(L, C, dtype=BF16, device=x.device)
    rstd = torch.empty(L, dtype=torch.float32, device=x.device)
    f, h, ww = grid
    call("prfl_rms_rope_fwd_pos", ptr(x), I64(_ld(x)), I64(L), I64(C), ptr(w), F32(eps),
         ptr(rope_tab), I64(f), I64(h), I64(ww), I64(row0), ptr(out), I64(_ld(out)), ptr(rstd),
         F32(out_scale), stream_ptr())
    return out, rstd


def rms_rope_bwd(dout, x, rstd, w, rope_tab=None, grid=(0, 0, 0), dx=None, out_scale=1.0, row0=0):
    """returns (dx bf16, d w fp32); out_scale and row0 as the forward's (dout is scaled by it)."""
    L, C = x.shape
    rp = call_int("prfl_norm_rows_per_part")
    p0 = torch.empty((L + rp - 1) // rp, C, dtype=torch.float32, device=x.device)
    if dx is None:
        dx = torch.empty(L, C, dtype=BF16, device=x.device)
    f, h, ww = grid
    call("prfl_rms_rope_bwd_pos", ptr(dout), I64(_ld(dout)), ptr(x), I64(_ld(x)), ptr(rstd),
         I64(L), I64(C), ptr(w), ptr(rope_tab), I64(f), I64(h), I64(ww), I64(row0), ptr(dx),
         I64(_ld(dx)), ptr(p0), F32(out_scale), stream_ptr())
    return dx, colsum_reduce(p0)


# the long-KV q_log2 forward reads V from its key-chunked transposed image (prfl_attn_v_to_vt +
# prfl_attn_fwd_l2q_vt_ws: one ds_read_b128 per V^T fragment; outputs bit-identical)
ATTN_VT = True     # 720p forward 84.11 -> 83.08 ms incl. the 0.29 ms transpose (profiles/r04_ab_attn_vt.txt)
# ... and (off) the long-KV q_log2 backward's dQ kernel its K^T fragments from K's VT image
# (prfl_attn_bwd_l2q_kt_ws; bit-identical, measured 0.3-0.5 % slower with the K transpose
# included: profiles/r04_ab_bwd_variants.txt)
ATTN_KT = False
VT_MIN_KEYS = 4096


def attn_fwd(q, k, v, num_heads, k_len=None, out=None, scale=None, q_log2=False):
    """q [Lq, H*128], k/v [Lk, H*128] (row-strided views) -> (o bf16 [Lq, H*128], lse2 [H, Lq]).
    q_log2: q is already multiplied by softmax_scale * log2(e) (rms_rope_fwd out_scale=L2Q_SCALE);
    scale is then unused (prfl_attn_fwd_l2q_ws; with Lk >= VT_MIN_KEYS and ATTN_VT, V is first
    rewritten into the VT layout and prfl_attn_fwd_l2q_vt_ws runs)."""
    Lq, C = q.shape
    Lk = k.shape[0]
    assert C == num_heads * 128, "head_dim must be 128"
    k_len = Lk if k_len is None else int(k_len)
    sc = scale if scale is not None else 1.0 / math.sqrt(128)
    if out is None:
        out = torch.empty(Lq, C, dtype=BF16, device=q.device)
    lse = torch.empty(num_heads, Lq, dtype=torch.float32, device=q.device)
    # scratch for the split-KV tail of long-KV launches (0 bytes when the grid has no tail)
    nb = _lib.load().prfl_attn_fwd_ws_bytes(1, Lq, Lk, num_heads, k_len)
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device) if nb > 0 else None
    head = (ptr(q), I64(_ld(q)), I64(0), ptr(k), I64(_ld(k)), I64(0), ptr(v), I64(_ld(v)), I64(0),
            ptr(out), I64(_ld(out)), I64(0), ptr(lse), I64(1), I64(Lq), I64(Lk), I64(num_heads),
            I64(k_len))
    if q_log2 and ATTN_VT and Lk >= VT_MIN_KEYS:
        vt = attn_v_to_vt(v, num_heads)
        call("prfl_attn_fwd_l2q_vt_ws", *head[:6], ptr(vt), *head[9:], ptr(ws), I64(nb), stream_ptr())
    elif q_log2:
        call("prfl_attn_fwd_l2q_ws", *head, ptr(ws), I64(nb), stream_ptr())
    else:
        call("prfl_attn_fwd_ws", *head, F32(sc), ptr(ws), I64(nb), stream_ptr())
    return out, lse


def attn_v_to_vt(v, num_heads):
    """v [Lk, H*128] (row-strided view) -> its VT image (prfl_attn_v_to_vt), a flat bf16 tensor"""
    Lk = v.shape[0]
    nb = _lib.load().prfl_attn_vt_bytes(1, Lk, num_heads)
    vt = torch.empty(nb // 2, dtype=BF16, device=v.device)
    call("prfl_attn_v_to_vt", ptr(v), I64(_ld(v)), I64(0), ptr(vt), I64(1), I64(Lk), I64(num_heads),
         stream_ptr())
    return vt


def attn_fwd_fp8(q, k, v, num_heads, k_len=None, out=None, scale=None, q_log2=False):
    """attn_fwd on the block-scaled e4m3 MFMA (config C5 self-attention): same arguments and
    outputs; q/k/v are quantised inside the call into a scratch buffer (~3 bytes per element)."""
    Lq, C = q.shape
    Lk = k.shape[0]
    assert C == num_heads * 128, "head_dim must be 128"
    k_len = Lk if k_len is None else int(k_len)
    sc = scale if scale is not None else 1.0 / math.sqrt(128)
    if out is None:
        out = torch.empty(Lq, C, dtype=BF16, device=q.device)
    lse = torch.empty(num_heads, Lq, dtype=torch.float32, device=q.device)
    nb = _lib.load().prfl_attn_fwd_fp8_ws_bytes(1, Lq, Lk, num_heads, k_len)
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device)
    head = (ptr(q), I64(_ld(q)), I64(0), ptr(k), I64(_ld(k)), I64(0), ptr(v), I64(_ld(v)), I64(0),
            ptr(out), I64(_ld(out)), I64(0), ptr(lse), I64(1), I64(Lq), I64(Lk), I64(num_heads),
            I64(k_len))
    if q_log2:
        call("prfl_attn_fwd_fp8_l2q", *head, ptr(ws), I64(nb), stream_ptr())
    else:
        call("prfl_attn_fwd_fp8", *head, F32(sc), ptr(ws), I64(nb), stream_ptr())
    return out, lse


def attn_bwd(q, k, v, o, do, lse, num_heads, k_len=None, dq=None, dk=None, dv=None, scale=None,
             q_log2=False):
    """Backward of attn_fwd; with q_log2 dq is the gradient w.r.t. the pre-scaled q."""
    Lq, C = q.shape
    Lk = k.shape[0]
    k_len = Lk if k_len is None else int(k_len)
    sc = scale if scale is not None else 1.0 / math.sqrt(128)
    dev = q.device
    dq = torch.empty(Lq, C, dtype=BF16, device=dev) if dq is None else dq
    dk = torch.empty(Lk, C, dtype=BF16, device=dev) if dk is None else dk
    dv = torch.empty(Lk, C, dtype=BF16, device=dev) if dv is None else dv
    delta = torch.empty(num_heads, Lq, dtype=torch.float32, device=dev)
    # scratch for the split tails of long-KV launches (0 bytes when the grids have no tail)
    nb = _lib.load().prfl_attn_bwd_ws_bytes(1, Lq, Lk, num_heads, k_len)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb > 0 else None
    head = (ptr(q), I64(_ld(q)), I64(0), ptr(k), I64(_ld(k)), I64(0), ptr(v), I64(_ld(v)), I64(0),
            ptr(o), I64(_ld(o)), I64(0), ptr(do), I64(_ld(do)), I64(0), ptr(lse), ptr(delta),
            ptr(dq), I64(_ld(dq)), I64(0), ptr(dk), I64(_ld(dk)), I64(0), ptr(dv), I64(_ld(dv)),
            I64(0), I64(1), I64(Lq), I64(Lk), I64(num_heads), I64(k_len))
    if q_log2 and ATTN_KT and Lk >= VT_MIN_KEYS:
        kt = attn_v_to_vt(k, num_heads)            # K in the VT layout for the dQ kernel
        call("prfl_attn_bwd_l2q_kt_ws", *head[:6], ptr(kt), *head[6:], ptr(ws), I64(nb), stream_ptr())
    elif q_log2:
        call("prfl_attn_bwd_l2q_ws", *head, ptr(ws), I64(nb), stream_ptr())
    else:
        call("prfl_attn_bwd_ws", *head, F32(sc), ptr(ws), I64(nb), stream_ptr())
    return dq, dk, dv


def query_pool_fwd(q, kv, num_heads, scale, nsplit=None):
    """Single-query attention pooling (csrc/pool.hip): q [N, E] bf16, kv [N, L, 2E] bf16 (k | v)
    -> (o bf16 [N, E], lse2 fp32 [N, H], o32 fp32 [N, E] = o before its bf16 rounding)."""
    _lib.require_gpu(q, kv)
    assert q.dtype == BF16 and kv.dtype == BF16 and kv.stride(2) == 1
    N, E = q.shape
    L = kv.shape[1]
    if nsplit is None:
        nsplit = call_int_args("prfl_query_pool_splits", I64(N), I64(L), I64(num_heads))
    hd = E // num_heads
    o = torch.empty(N, E, dtype=BF16, device=q.device)
    lse = torch.empty(N, num_heads, dtype=torch.float32, device=q.device)
    o32 = torch.empty(N, E, dtype=torch.float32, device=q.device)
    pm = torch.empty(N * num_heads * nsplit, dtype=torch.float32, device=q.device)
    pl = torch.empty_like(pm)
    po = torch.empty(N * num_heads * nsplit * hd, dtype=torch.float32, device=q.device)
    call("prfl_query_pool_fwd", ptr(q), I64(_ld(q)), ptr(kv), I64(kv.stride(1)), I64(kv.stride(0)),
         I64(N), I64(L), I64(num_heads), I64(E), F32(scale), ptr(o), I64(E), ptr(lse), ptr(o32),
         ptr(pm), ptr(pl), ptr(po), I64(nsplit), stream_ptr())
    return o, lse, o32


def query_pool_bwd(do, q, kv, o32, lse, num_heads, scale, nsplit=None):
    """-> (dq fp32 [N, E], dkv bf16 [N, L, 2E])."""
    N, E = q.shape
    L = kv.shape[1]
    if nsplit is None:
        nsplit = call_int_args("prfl_query_pool_splits", I64(N), I64(L), I64(num_heads))
    hd = E // num_heads
    dq = torch.empty(N, E, dtype=torch.float32, device=q.device)
    dkv = torch.empty(N, L, 2 * E, dtype=BF16, device=q.device)
    po = torch.empty(N * num_heads * nsplit * hd, dtype=torch.float32, device=q.device)
    call("prfl_query_pool_bwd", ptr(do), ptr(q), I64(_ld(q)), ptr(kv), I64(kv.stride(1)),
         I64(kv.stride(0)), ptr(o32), ptr(lse), I64(N), I64(L), I64(num_heads), I64(E), F32(scale),
         ptr(dq), I64(E), ptr(dkv), I64(2 * E), I64(L * 2 * E), ptr(po), I64(nsplit), stream_ptr())
    return dq, dkv


def call_int_args(name, *args):
    return getattr(_lib.load(), name)(*args)


def sumsq_(x, out):
    call("prfl_sumsq", ptr(x), I64(x.numel()), ptr(out), stream_ptr())


def scale_(x, factor):
    call("prfl_scale", ptr(x), I64(x.numel()), ptr(factor), stream_ptr())


def adamw_(p, g, m, v, lr, beta1, beta2, eps, weight_decay, step, zero_grad=False):
    """One AdamW step on p (m, v: its moments); zero_grad also sets g to 0 once read."""
    for t in (p, g, m, v):
        assert t.is_contiguous() and t.dtype == torch.float32
    call("prfl_adamw_zero_grad" if zero_grad else "prfl_adamw", ptr(p), ptr(g), ptr(m), ptr(v),
         I64(p.numel()), F32(lr), F32(beta1), F32(beta2), F32(eps), F32(weight_decay), I64(step),
         stream_ptr())


def rope_table(freqs_complex, device):
    """complex freqs [1024, 64] (model.py:521-526) -> fp32 (cos, sin) table on device."""
    t = torch.view_as_real(freqs_complex.to(torch.complex128)).to(torch.float32).contiguous()
    return t.to(device)


# ---------------------------------------------------------------- layer norm (csrc/layernorm.hip)
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _type(t, what):
    if t not in TYPES:
        raise ValueError(f"{what}: fp32, bf16 or fp16, got {t}")
    return TYPES[t]


def _one_device(what, first, *others):
    if not first.is_cuda:
        _lib.require_gpu(first)
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            _lib.require_gpu(t)
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    return dev


def _rows(t, C):
    """[..., C] as [rows, C] with unit column stride (a view where the strides allow it)."""
    t = t.reshape(-1, C) if t.dim() != 2 else t
    return t if t.stride(1) == 1 or C == 1 else t.contiguous()


def _last_axis(shape):
    C = shape[-1] if shape else 0
    if not 1 <= C <= 16384:
        raise ValueError(f"layer_norm: a last axis of 1 to 16384, got {tuple(shape)}")
    return C


def layer_norm_fwd(x, w=None, b=None, eps=1e-5, out_dtype=None):
    """LN over the last axis of x [..., C] (C <= 16384), times w plus b ([C] each, or None):
    returns (y in out_dtype or x's, mean, rstd fp32 of x's leading shape)."""
    shape = x.shape
    C = _last_axis(shape)
    dev = _one_device("layer_norm", x, w, b)
    ydt = x.dtype if out_dtype is None else out_dtype
    xt, yt, wt, pw, pb = _type(x.dtype, "layer_norm x"), _type(ydt, "layer_norm out_dtype"), 0, None, None
    if w is not None:
        wt = _type(w.dtype, "layer_norm w")
        w = w.contiguous()
        pw = w.data_ptr()
    if b is not None:
        wt = _type(b.dtype, "layer_norm w")
        b = b.contiguous()
        pb = b.data_ptr()
    if ((w is not None and w.shape != (C,)) or (b is not None and b.shape != (C,))
            or (pw is not None and pb is not None and w.dtype != b.dtype)):
        raise ValueError(f"layer_norm: w and b are [{C}] of one type")
    if not eps >= 0:
        raise ValueError(f"layer_norm: eps is not negative, got {eps}")
    x2 = _rows(x, C)
    L = x2.shape[0]
    # (new_empty and empty_like cost half of torch.empty(device=) on the host, a third of a short call)
    y = torch.empty_like(x, dtype=ydt) if x.is_contiguous() else x.new_empty(shape, dtype=ydt)
    mean = x.new_empty(L if len(shape) == 2 else shape[:-1], dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _lib.call_on(dev, "prfl_layer_norm_fwd", x2.data_ptr(), xt, x2.stride(0), L, C, pw, pb, wt, eps,
                 y.data_ptr(), yt, C, mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def _addr(t):
    return None if t is None else t.data_ptr()


def layer_norm_bwd(dy, x, mean, rstd, w=None, want_dx=True, want_dw=None, want_db=True):
    """Backward of layer_norm_fwd: (dx in x's type, dw, db fp32 [C]; None where not wanted).  dy has
    the forward's output type; dw is given by default where w is."""
    C = _last_axis(x.shape)
    dev = _one_device("layer_norm", x, dy, mean, rstd, w)
    if dy.shape != x.shape or mean.numel() * C != x.numel() or rstd.numel() != mean.numel():
        raise ValueError("layer_norm: dy has x's shape, mean and rstd one value a row")
    if mean.dtype != torch.float32 or rstd.dtype != torch.float32:
        raise ValueError("layer_norm: mean and rstd are the forward's fp32")
    if w is not None and w.shape != (C,):
        raise ValueError(f"layer_norm: w is [{C}]")
    xt, yt = _type(x.dtype, "layer_norm x"), _type(dy.dtype, "layer_norm dy")
    wt = 0 if w is None else _type(w.dtype, "layer_norm w")
    want_dw = w is not None if want_dw is None else want_dw
    x2, dy2 = _rows(x, C), _rows(dy, C)
    L = x2.shape[0]
    mean, rstd = mean.contiguous(), rstd.contiguous()
    w = None if w is None else w.contiguous()
    dx = None
    if want_dx:
        dx = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    dw = mean.new_empty(C) if want_dw else None
    db = mean.new_empty(C) if want_db else None
    part = None
    if want_dw or want_db:
        n = _lib.load().prfl_layer_norm_parts(L, C, xt)
        part = mean.new_empty(n * C * (int(want_dw) + int(want_db))) if n else None
    _lib.call_on(dev, "prfl_layer_norm_bwd", dy2.data_ptr(), yt, dy2.stride(0), x2.data_ptr(), xt,
                 x2.stride(0), mean.data_ptr(), rstd.data_ptr(), L, C, _addr(w), wt, _addr(dx), C,
                 _addr(dw), _addr(db), _addr(part))
    return dx, dw, db


# ------------------------------------------- gradient norm and clipping (csrc/grads.hip) --------
def _dense(t):
    """whether t's elements fill one run of memory (in any order of its axes)"""
    if t.is_contiguous():
        return True
    n = 1
    for size, stride in sorted(((a, b) for a, b in zip(t.shape, t.stride()) if a != 1),
                               key=lambda d: d[1]):
        if stride != n:
            return False
        n *= size
    return True


def _grad_list(grads, what, disjoint):
    """(addresses, sizes, type codes) of the tensors as host arrays; whether all are contiguous.  (A call
    over a few dozen small tensors is these lists' time: one pass of C calls per attribute.)"""
    if not grads:
        raise ValueError(f"{what}: no tensors")
    dev = grads[0].device
    if dev.type != "cuda":
        _lib.require_gpu(grads[0])
    plain = False
    try:
        plain = all([t.is_contiguous() for t in grads])
        at = array.array("Q", [t.data_ptr() for t in grads])
        types = array.array("i", [TYPES[t.dtype] for t in grads])
        ok = plain or all([_dense(t) for t in grads])
    except (KeyError, RuntimeError):             # another type; sparse tensors have no address
        ok = False
    if not ok:
        got = next((t for t in grads if t.dtype not in TYPES or t.layout is not torch.strided or not _dense(t)),
                   grads[0])
        raise ValueError(f"{what}: dense fp32, bf16 or fp16 tensors in memory, got {got.dtype} "
                         f"{tuple(got.shape)}, {got.layout}")
    for t in grads:
        if t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
    n = array.array("q", [t.numel() for t in grads])
    if disjoint and _lib.load().prfl_grads_overlap(_host(at), _host(n), _host(types), len(grads)):
        raise ValueError(f"{what}: two of the tensors share memory")
    return at, n, types, plain


def _host(a):
    return a.buffer_info()[0]


def grads_sumsq(grads):
    """Sum of the squares of all elements of a list of dense fp32 / bf16 / fp16 tensors: fp64 [1] on
    their device.  (Ranks that hold shards add theirs, then clip_grads(sumsq=...).)"""
    grads = list(grads)
    at, n, types, _ = _grad_list(grads, "grads_sumsq", False)
    dev, k = grads[0].device, len(grads)
    parts = _lib.load().prfl_grads_parts(_host(n), k)
    part = torch.empty(parts, dtype=torch.float64, device=dev)
    out = torch.empty(1, dtype=torch.float64, device=dev)
    _lib.call_on(dev, "prfl_grads_sumsq", _host(at), _host(n), _host(types), k, part.data_ptr(), parts, out.data_ptr())
    return out


def clip_grads(grads, max_norm, eps=1e-6, out=None, sumsq=None):
    """Scale the tensors by min(1, max_norm / (norm + eps)), norm their global L2 norm (or
    sqrt(sumsq) where that is given); in place, or into `out`, a list of tensors of the same shapes
    and one type.  Returns the norm before clipping, fp32 0-dim on the device (nothing waits; infinity
    where it is past fp32, which the clipped values do not suffer from)."""
    if not max_norm >= 0 or not eps >= 0:
        raise ValueError(f"clip_grads: max_norm and eps are not negative, got {max_norm}, {eps}")
    grads = list(grads)
    dst, otype, k = None, -1, len(grads)
    if out is None:
        at, n, types, _ = _grad_list(grads, "clip_grads", True)
    else:
        out = list(out)
        if len(out) != k or [o.shape for o in out] != [g.shape for g in grads]:
            raise ValueError("clip_grads: out has the gradients' shapes and strides, and one type")
        at, n, types, plain = _grad_list(grads + out, "clip_grads", True)      # first k: the gradients
        otype = types[k]
        if types[k:].count(otype) != k or not (plain or all(o.stride() == g.stride() for o, g in zip(out, grads))):
            raise ValueError("clip_grads: out has the gradients' shapes and strides, and one type")
        dst = _host(at) + 8 * k
    dev = grads[0].device
    part, parts = None, 0
    if sumsq is None:
        parts = _lib.load().prfl_grads_parts(_host(n), k)
        part = grads[0].new_empty(parts, dtype=torch.float64)
    elif sumsq.dtype != torch.float64 or sumsq.numel() != 1 or sumsq.device != dev:
        raise ValueError("clip_grads: sumsq is one fp64 value on the gradients' device")
    norm = grads[0].new_empty((), dtype=torch.float32)
    _lib.call_on(dev, "prfl_grads_clip", _host(at), dst, _host(n), _host(types), k, otype, _addr(sumsq), _addr(part), parts,
                 max_norm, eps, norm.data_ptr())
    if out is not None:
        # written: AdamW and autograd read it off the version counter.  (In place the counter stays, as it does
        # for scale_: a gradient that AdamW zeroed and that received nothing since is still none after it.)
        torch.autograd.graph.increment_version(out)
    return norm


# ------------------------------------------------------------ microscaled fp4 (csrc/mxfp4.hip) --
MX_MOST = 1 << 24              # columns of a tiled matrix, and rows of one that is multiplied by


def _mx_shape(rows, cols):
    return -(-rows // 64), -(-cols // 128)


def quant_mxfp4(x):
    """x [M, K] (fp32 / bf16 / fp16, row-strided) -> (q uint8 [M/64, K/128, 4, 64, 16], s uint8
    [M/64, K/128, 64, 4]): e2m1 codes and e8m0 scales in the tiled layout of include/prfl_hip.h."""
    if x.dim() != 2 or not 1 <= x.shape[1] <= MX_MOST:
        raise ValueError(f"quant_mxfp4: [M, K] with K of 1 to 2^24, got {tuple(x.shape)}")
    dev = _one_device("quant_mxfp4", x)
    xt = _type(x.dtype, "quant_mxfp4")
    M, K = x.shape
    x = _rows(x, K)
    G, S = _mx_shape(M, K)
    q = x.new_empty((G, S, 4, 64, 16), dtype=torch.uint8)
    s = q.new_empty((G, S, 64, 4))
    _lib.call_on(dev, "prfl_quant_mxfp4", x.data_ptr(), xt, x.stride(0), M, K, q.data_ptr(),
                 s.data_ptr())
    return q, s


def _mx_check(what, q, s, rows, cols):
    if not 1 <= cols <= MX_MOST or rows < 0:
        raise ValueError(f"{what}: a [{rows}, {cols}] matrix")
    G, S = _mx_shape(rows, cols)
    if (q.shape != (G, S, 4, 64, 16) or s.shape != (G, S, 64, 4) or q.dtype != torch.uint8
            or s.dtype != torch.uint8 or not q.is_contiguous() or not s.is_contiguous()):
        raise ValueError(f"{what}: a tiled [{rows}, {cols}] matrix has contiguous uint8 q "
                         f"{(G, S, 4, 64, 16)} and s {(G, S, 64, 4)}, got {tuple(q.shape)} and "
                         f"{tuple(s.shape)}")


def dequant_mxfp4(q, s, rows, cols, out_dtype=BF16):
    """The values of quant_mxfp4's (q, s), [rows, cols] in bf16 (exact) or fp32."""
    dev = _one_device("dequant_mxfp4", q, s)
    _mx_check("dequant_mxfp4", q, s, rows, cols)
    if out_dtype not in (BF16, torch.float32):
        raise ValueError(f"dequant_mxfp4: bf16 or fp32, got {out_dtype}")
    out = q.new_empty((rows, cols), dtype=out_dtype)
    _lib.call_on(dev, "prfl_dequant_mxfp4", q.data_ptr(), s.data_ptr(), rows, cols, out.data_ptr(),
                 int(out_dtype == torch.float32), cols)
    return out


def linear_mxfp4(x, wq, ws, out_features, bias=None):
    """y [..., N] bf16 = x W^T + bias on the block-scaled MFMA: x [..., K] (fp32 / bf16 / fp16) is
    quantised to microscaled fp4 in the call, (wq, ws) = quant_mxfp4(W [N, K]), bias bf16 [N]."""
    if x.dim() < 1 or x.shape[-1] < 1 or not 1 <= out_features <= MX_MOST:
        raise ValueError(f"linear_mxfp4: x is [..., K], got {tuple(x.shape)} to {out_features}")
    K, N = x.shape[-1], out_features
    dev = _one_device("linear_mxfp4", x, wq, ws, bias)
    _mx_check("linear_mxfp4", wq, ws, N, K)
    if bias is not None and (bias.dtype != BF16 or bias.shape != (N,) or not bias.is_contiguous()):
        raise ValueError(f"linear_mxfp4: a contiguous bf16 bias of [{N}]")
    xt = _type(x.dtype, "linear_mxfp4")
    x2 = _rows(x, K)
    M = x2.shape[0]
    y = x.new_empty((*x.shape[:-1], N), dtype=BF16)
    nb = _lib.load().prfl_linear_mxfp4_ws_bytes(M, K)
    work = wq.new_empty(nb) if nb else None
    _lib.call_on(dev, "prfl_linear_mxfp4", x2.data_ptr(), xt, x2.stride(0), wq.data_ptr(),
                 ws.data_ptr(), _addr(bias), y.data_ptr(), N, M, N, K, _addr(work), nb)
    return y


def linear_mxfp4_dx(dy, wq, ws, in_features):
    """dx [..., K] bf16 = dy W of linear_mxfp4, x's quantisation taken as the identity: W is read
    back to bf16 (exact) and multiplied on the bf16 MFMA, for small products in one launch.  dy [..., N] is
    taken in bf16."""
    if dy.dim() < 1 or not 1 <= dy.shape[-1] <= MX_MOST:
        raise ValueError(f"linear_mxfp4_dx: dy is [..., N], got {tuple(dy.shape)}")
    N, K = dy.shape[-1], in_features
    dev = _one_device("linear_mxfp4_dx", dy, wq, ws)
    _mx_check("linear_mxfp4_dx", wq, ws, N, K)
    yt = _type(dy.dtype, "linear_mxfp4_dx")
    d = _rows(dy, N)
    M, Np, Kp = d.shape[0], -(-N // 8) * 8, -(-K // 8) * 8
    if M == 0 or _lib.load().prfl_linear_mxfp4_dx_direct(M, N, K):
        dx = dy.new_empty((*dy.shape[:-1], K), dtype=BF16)
        _lib.call_on(dev, "prfl_linear_mxfp4_dx", d.data_ptr(), yt, d.stride(0), wq.data_ptr(),
                     ws.data_ptr(), dx.data_ptr(), K, M, N, K)
        return dx
    d = d.to(BF16)
    # the bf16 product takes extents in eights: padding rows and columns of W read back as zeros
    w = dequant_mxfp4(wq, ws, Np, Kp)
    if Np != N:
        d = torch.nn.functional.pad(d, (0, Np - N))
    elif d.stride(0) % 8 or d.data_ptr() % 16:
        d = d.clone(memory_format=torch.contiguous_format)
    with torch.cuda.device(dev):
        dx = linear_dx(d, w)
    if Kp != K:
        dx = dx[:, :K].contiguous()
    return dx.view(*dy.shape[:-1], K)


def prof_enable(on=True):
    call("prfl_prof_enable", I32(int(on)))


def prof_collect():
    import ctypes
    n = _lib.NKID
    counts = (ctypes.c_int64 * n)()
    ms = (ctypes.c_double * n)()
    work = (ctypes.c_double * n)()
    call("prfl_prof_collect", ctypes.cast(counts, ctypes.c_void_p), ctypes.cast(ms, ctypes.c_void_p),
         ctypes.cast(work, ctypes.c_void_p), I32(n))
    return {k: dict(count=counts[i], ms=ms[i], work=work[i]) for k, i in _lib.KID.items()}


def prof_clock():
    """Effective shader clock of the self-attention forwards since the last call (MHz)."""
    import ctypes
    v = (ctypes.c_double * 3)()
    n = ctypes.c_int64()
    base = ctypes.addressof(v)
    call("prfl_prof_clock", P(base), P(base + 8), P(base + 16), P(ctypes.addressof(n)))
    return dict(mean_mhz=v[0], min_mhz=v[1], max_mhz=v[2], launches=n.value)


def _coef_array(coef):
    import ctypes
    assert len(coef) == 11
    return (ctypes.c_float * 11)(*[float(c) for c in coef])


def unipc_step_fwd(sample, model_output, last_sample, hist1, hist2, coef, corr_order, pred_order):
    """Fused FlowUniPC update (csrc/unipc.hip).  Returns (m_t fp32, sample_c bf16, prev bf16)."""
    import ctypes
    _lib.require_gpu(sample, model_output)
    if sample.dtype != torch.bfloat16 or model_output.dtype != torch.float32:
        raise NotImplementedError("fused UniPC step: bf16 sample and fp32 model output "
                                  "(the PRFL chain's dtypes, train_prfl.py:687-734)")
    n = sample.numel()
    for t in (model_output, last_sample, hist1, hist2):
        if t is not None and (t.numel() != n or not t.is_contiguous()):
            raise ValueError("fused UniPC step: operands must be contiguous with the sample's shape")
    sample = sample.contiguous()
    m_t = torch.empty(sample.shape, dtype=torch.float32, device=sample.device)
    prev = torch.empty_like(sample)
    sample_c = torch.empty_like(sample) if corr_order else sample
    cf = _coef_array(coef)
    call("prfl_unipc_step", ptr(sample), ptr(model_output), ptr(last_sample), ptr(hist1),
         ptr(hist2), ptr(m_t), ptr(sample_c) if corr_order else P(0), ptr(prev), I64(n),
         ctypes.cast(cf, ctypes.c_void_p), I32(corr_order), I32(pred_order), stream_ptr())
    return m_t, sample_c, prev


def unipc_step_bwd(grad_prev, coef, corr_order, pred_order):
    import ctypes
    g = grad_prev.to(torch.bfloat16).contiguous()
    out = torch.empty(g.shape, dtype=torch.float32, device=g.device)
    cf = _coef_array(coef)
    call("prfl_unipc_step_bwd", ptr(g), ptr(out), I64(g.numel()), ctypes.cast(cf, ctypes.c_void_p),
         I32(corr_order), I32(pred_order), stream_ptr())
    return out
