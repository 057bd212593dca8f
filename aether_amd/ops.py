"""torch-tensor wrappers over the per-kernel C-ABI entry points (include/aether_hip.h).

These are the calls the parity tests exercise one by one; the production transformer goes through the single
`aether_dit_forward` entry instead.  Every function enqueues on torch's current stream and raises on error.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch

from . import _lib
from ._lib import AETHER_EPI_BIAS, AETHER_EPI_BIAS_GATE_RES, AETHER_EPI_BIAS_GELU  # noqa: F401


def _need_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("aether_amd ops need device tensors (no CPU fallback)")


def gemm_bf16(A, W, bias=None, epilogue=AETHER_EPI_BIAS, R=None, gate_vid=None, gate_txt=None, rows_per_batch=0, n_text=0,
              out=None, flags=0, splitk_ws=None):
    """out[M,N] = epi(A[M,K] @ W[N,K]^T); A,W,R bf16; bias/gates fp32. gate_*: [B, N] (row stride = stride(0)).
    splitk_ws: optional fp32 scratch (>= 64 MiB) enabling the split-K tail launch."""
    _need_cuda(A, W, bias, R, gate_vid, gate_txt)
    assert A.dtype == torch.bfloat16 and W.dtype == torch.bfloat16 and A.dim() == 2 and W.dim() == 2
    assert A.stride(1) == 1 and W.stride(1) == 1
    M, K = A.shape
    N = W.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=A.device)
    gstride = gate_vid.stride(0) if gate_vid is not None else 0
    lib = _lib.load()
    rc = lib.aether_gemm_bf16(_lib.ptr(A), A.stride(0), _lib.ptr(W), W.stride(0), _lib.ptr(out), out.stride(0), M, N, K,
                              _lib.ptr(bias), epilogue, _lib.ptr(R), R.stride(0) if R is not None else 0,
                              _lib.ptr(gate_vid), _lib.ptr(gate_txt), gstride, rows_per_batch, n_text, _lib.ptr(splitk_ws),
                              splitk_ws.numel() * 4 if splitk_ws is not None else 0, flags, _lib.current_stream())
    _lib.check(rc, "aether_gemm_bf16")
    return out


def layernorm_modulate(x, w=None, b=None, eps=1e-5, shift_vid=None, scale_vid=None, shift_txt=None, scale_txt=None,
                       rows_per_batch=0, n_text=0, out=None):
    _need_cuda(x, w, b, shift_vid)
    assert x.dtype == torch.bfloat16 and x.dim() == 2 and x.stride(1) == 1
    rows, D = x.shape
    if out is None:
        out = torch.empty_like(x)
    mstride = shift_vid.stride(0) if shift_vid is not None else 0
    lib = _lib.load()
    rc = lib.aether_layernorm_modulate(_lib.ptr(x), x.stride(0), _lib.ptr(out), out.stride(0), rows, D, float(eps), _lib.ptr(w),
                                       _lib.ptr(b), _lib.ptr(shift_vid), _lib.ptr(scale_vid), _lib.ptr(shift_txt),
                                       _lib.ptr(scale_txt), mstride, rows_per_batch, n_text, _lib.current_stream())
    _lib.check(rc, "aether_layernorm_modulate")
    return out


def gemv_rows(x, W, bias=None, act_in=0, act_out=0):
    """out[B,N] = act_out(bias + act_in(x[B,K]) @ W[N,K]^T); x fp32, W bf16, out fp32."""
    _need_cuda(x, W, bias)
    assert x.dtype == torch.float32 and W.dtype == torch.bfloat16 and x.is_contiguous() and W.is_contiguous()
    B, K = x.shape
    N = W.shape[0]
    out = torch.empty(B, N, dtype=torch.float32, device=x.device)
    lib = _lib.load()
    rc = lib.aether_gemv_rows(_lib.ptr(x), B, K, _lib.ptr(W), _lib.ptr(bias), _lib.ptr(out), N, act_in, act_out,
                              _lib.current_stream())
    _lib.check(rc, "aether_gemv_rows")
    return out


def timestep_sinusoid(t, dim):
    _need_cuda(t)
    t = t.to(torch.float32).contiguous()
    out = torch.empty(t.shape[0], dim, dtype=torch.float32, device=t.device)
    rc = _lib.load().aether_timestep_sinusoid(_lib.ptr(t), t.shape[0], dim, _lib.ptr(out), _lib.current_stream())
    _lib.check(rc, "aether_timestep_sinusoid")
    return out


def patchify(x, p):
    _need_cuda(x)
    assert x.dtype == torch.bfloat16 and x.is_contiguous() and x.dim() == 5
    B, F, Cc, H, W = x.shape
    out = torch.empty(B * F * (H // p) * (W // p), Cc * p * p, dtype=torch.bfloat16, device=x.device)
    rc = _lib.load().aether_patchify(_lib.ptr(x), _lib.ptr(out), B, F, Cc, H, W, p, _lib.current_stream())
    _lib.check(rc, "aether_patchify")
    return out


def unpatchify(Y, B, F, Cout, H, W, p):
    _need_cuda(Y)
    assert Y.dtype == torch.bfloat16 and Y.stride(1) == 1
    out = torch.empty(B, F, Cout, H, W, dtype=torch.bfloat16, device=Y.device)
    rc = _lib.load().aether_unpatchify(_lib.ptr(Y), Y.stride(0), _lib.ptr(out), B, F, Cout, H, W, p, _lib.current_stream())
    _lib.check(rc, "aether_unpatchify")
    return out


def qk_norm_rope(qkv, H, n_text, qn_w, qn_b, kn_w, kn_b, eps, cos, sin, q_scale):
    """qkv bf16 [B,S,3*H*64] -> (Qh [B,H,S,64], Kh [B,H,S,64], Vt [B,H,64,Spad])."""
    _need_cuda(qkv)
    assert qkv.dtype == torch.bfloat16 and qkv.is_contiguous()
    B, S, _ = qkv.shape
    Spad = (S + 63) // 64 * 64
    Qh = torch.empty(B, H, S, 64, dtype=torch.bfloat16, device=qkv.device)
    Kh = torch.empty_like(Qh)
    Vt = torch.empty(B, H, 64, Spad, dtype=torch.bfloat16, device=qkv.device)
    rc = _lib.load().aether_qk_norm_rope(_lib.ptr(qkv), B, S, H, n_text, _lib.ptr(qn_w), _lib.ptr(qn_b), _lib.ptr(kn_w),
                                         _lib.ptr(kn_b), float(eps), _lib.ptr(cos), _lib.ptr(sin), float(q_scale),
                                         _lib.ptr(Qh), _lib.ptr(Kh), _lib.ptr(Vt), Spad, _lib.current_stream())
    _lib.check(rc, "aether_qk_norm_rope")
    return Qh, Kh, Vt


def flash_attn_fwd(Qh, Kh, Vt, flags=0):
    """Qh,Kh [B,H,S,64] (softmax scale x log2(e) folded into Qh: _lib.ATTN_Q_SCALE), Vt [B,H,64,Spad] -> O [B,S,H*64].
    flags: AETHER_GEMM_WIDE_STORE | AETHER_ATTN_EXACT_MAX (the conservative path alone)."""
    _need_cuda(Qh, Kh, Vt)
    B, H, S, d = Qh.shape
    assert d == 64 and Qh.is_contiguous() and Kh.is_contiguous() and Vt.is_contiguous()
    Spad = Vt.shape[-1]
    O = torch.empty(B, S, H * 64, dtype=torch.bfloat16, device=Qh.device)
    rc = _lib.load().aether_flash_attn_fwd(_lib.ptr(Qh), _lib.ptr(Kh), _lib.ptr(Vt), _lib.ptr(O), B, H, S, Spad, flags, _lib.current_stream())
    _lib.check(rc, "aether_flash_attn_fwd")
    return O


# ---- the text encoder's operators ------------------------------------------------------------------------------------
# These take tensors of any leading shape, strides and device (another device than the current one included: the call runs on that
# device's current stream), and refuse what they do not compute with ValueError before anything is enqueued.


def _same_device(first, *others):
    """The device of the call.  Every operand lives there."""
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            _need_cuda(first, *others)
            raise ValueError(f"operands are on different devices: {dev} and {t.device}")
    if not first.is_cuda:
        _need_cuda(first)
    return dev


def _run(what, dev, fn, *args):
    """fn(*args, stream) on `dev` and its current stream."""
    if dev.index == torch._C._cuda_getDevice():
        rc = fn(*args, _lib.stream_of(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _lib.stream_of(dev.index))
    if rc:
        _lib.check(rc, what)


def _rows(t, width):
    """`t` as [rows, width] with unit stride, an aligned base and rows a multiple of 8 elements and of 16 bytes apart; copied only where it is not so."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    by, one = t.stride()
    if one != 1 or by % 8 or by * t.element_size() % 16 or by < width or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _vector(t):
    """A 1-d operand with unit stride and a 16-byte aligned base; copied only where it is not so."""
    return t if t.stride(0) == 1 and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _like(t, dtype):
    """An output of t's shape (half the time of torch.empty with a device)."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _workspace(t, nbytes):
    return t.new_empty((nbytes,), dtype=torch.uint8)


_STREAMS = {torch.bfloat16: _lib.AETHER_STREAM_BF16, torch.float32: _lib.AETHER_STREAM_FP32}


def _norm_operands(x, w, delta, name):
    if not (x.dtype in _STREAMS):
        raise ValueError(f"{name}: the stream is bfloat16 or float32, got {x.dtype}")
    if not (x.dim() >= 1 and x.shape[-1] > 0):
        raise ValueError(f"{name}: the stream has no last dimension")
    D = x.shape[-1]
    if w.dtype != torch.float32 or w.shape != (D,):
        raise ValueError(f"{name}: the weight is float32 [{D}], got {w.dtype} {list(w.shape)}")
    if delta is not None:
        if not (delta.dtype == torch.bfloat16 and delta.shape == x.shape):
            raise ValueError(f"{name}: delta is bfloat16 {list(x.shape)}, got {delta.dtype} {list(delta.shape)}")
    return D


def _rms_norm(x, w, eps, delta, e4m3):
    name = "rms_norm_e4m3" if e4m3 else "rms_norm"
    dev = _same_device(x, w, delta)
    D = _norm_operands(x, w, delta, name)
    x2, w = _rows(x, D), _vector(w)
    rows = x2.shape[0]
    y = _like(x, torch.float8_e4m3fn if e4m3 else torch.bfloat16)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if e4m3 else None
    if delta is None:
        d2, res = None, None
    else:
        d2, res = _rows(delta, D), _like(x, x.dtype)
    if rows:
        _run(name, dev, _lib.load().aether_rms_norm, x2.data_ptr(), _STREAMS[x.dtype], x2.stride(0), _lib.ptr(d2), d2.stride(0) if d2 is not None else 0,
             _lib.ptr(res), D, w.data_ptr(), float(eps), y.data_ptr(), D, _lib.ptr(scale), rows, D)
    return y, scale, x if res is None else res


def rms_norm(x, w, eps=1e-6, delta=None):
    """h = x + delta;  y = h (mean(h²) + eps)^-1/2 w over the last dimension.  x: the residual stream [..., D], bfloat16 or float32; delta: a block's
    output, bfloat16 [..., D], or None; w float32 [D]; D a multiple of 8 up to 16384.  -> (y bfloat16, h in the stream's type; x itself without
    delta).  Statistics in fp32 of the unrounded sum."""
    y, _, res = _rms_norm(x, w, eps, delta, False)
    return y, res


def rms_norm_e4m3(x, w, eps=1e-6, delta=None):
    """`rms_norm` with its output in 8 bits -> (q float8_e4m3fn, scale float32 [...], h):  y ≈ q · scale with one power of two per row, the smallest
    one that brings the row into ±448.  A row that holds an infinity or a NaN becomes NaN (scale and values)."""
    return _rms_norm(x, w, eps, delta, True)


def rms_norm_backward(dy, res, w, eps=1e-6, dres=None, need_ddelta=False, delta=None):
    """Gradients of `rms_norm` from its stored h (`res`): dy bfloat16 [..., D] for y, dres (the stream's type) for h or None.  With delta, `res` is the stream before
    the addition and the sum is taken again: a bfloat16 stream's h is rounded, the norm was of the unrounded sum.
    -> (dx in the stream's type, ddelta bfloat16 or None, dw float32 [D]).  Summed in an order that depends on the sizes alone."""
    dev = _same_device(res, dy, w, dres, delta)
    D = _norm_operands(res, w, dy, "rms_norm_backward")
    if delta is not None:
        _norm_operands(res, w, delta, "rms_norm_backward")
    if dres is not None:
        if not (dres.dtype == res.dtype and dres.shape == res.shape):
            raise ValueError(f"rms_norm_backward: dres is {res.dtype} {list(res.shape)}, got {dres.dtype} {list(dres.shape)}")
    r2, g2, w = _rows(res, D), _rows(dy, D), _vector(w)
    s2 = None if dres is None else _rows(dres, D)
    d2 = None if delta is None else _rows(delta, D)
    rows = r2.shape[0]
    dx = _like(res, res.dtype)
    ddelta = _like(res, torch.bfloat16) if need_ddelta else None      # (a bf16 stream's dx again, in memory of its own: either may be changed in place)
    dw = _like(w, torch.float32)
    lib = _lib.load()
    nbytes = lib.aether_rms_norm_bwd_workspace_bytes(rows, D)
    ws = _workspace(w, nbytes)
    _run("rms_norm_backward", dev, lib.aether_rms_norm_bwd, g2.data_ptr(), g2.stride(0), r2.data_ptr(), _STREAMS[res.dtype], r2.stride(0),
         _lib.ptr(d2), d2.stride(0) if d2 is not None else 0, _lib.ptr(s2), s2.stride(0) if s2 is not None else 0, w.data_ptr(), float(eps), dx.data_ptr(), D, _lib.ptr(ddelta), D, dw.data_ptr(), rows, D,
         ws.data_ptr(), nbytes)
    return dx, ddelta, dw


def quantize_rows_e4m3(x):
    """x bfloat16 [rows, K] (K a multiple of 8) -> (q float8_e4m3fn [rows, K], scale float32 [rows]), x ≈ q · scale: a weight matrix in the form
    `gated_ff_e4m3` takes (one power of two per row, as `rms_norm_e4m3`)."""
    dev = _same_device(x)
    if not (x.dtype == torch.bfloat16 and x.dim() == 2):
        raise ValueError(f"quantize_rows_e4m3: bfloat16 [rows, K], got {x.dtype} {list(x.shape)}")
    x2 = _rows(x, x.shape[1]) if x.numel() else x
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    scale = torch.empty(x.shape[0], dtype=torch.float32, device=dev)
    if x.shape[0]:
        _run("quantize_rows_e4m3", dev, _lib.load().aether_quantize_rows_e4m3, x2.data_ptr(), x2.stride(0), q.data_ptr(), x.shape[1], scale.data_ptr(), *x.shape)
    return q, scale


@functools.lru_cache(maxsize=None)
def relbias_borders(num_buckets, max_distance):
    """Where each bucket of one side behind the first logarithmic one begins.  One side has half = num_buckets / 2 buckets: the distances below
    near = half // 2 have one each, the others are spaced over the logarithm up to max_distance: bucket near + b begins at the smallest n with
    log(n / near) / log(max_distance / near) (half − near) >= b.  Compared as whole numbers, so that no rounding moves a border."""
    if num_buckets < 4 or num_buckets % 2 or num_buckets > 128:
        raise ValueError(f"num_buckets must be an even number in [4, 128], got {num_buckets}")
    half = num_buckets // 2
    near = half // 2
    if max_distance != int(max_distance) or max_distance <= near:
        raise ValueError(f"max_distance must be a whole number above num_buckets / 4 = {near}, got {max_distance}")
    found, n = [], near
    for b in range(1, half - near):
        # (n / near)^(half - near) >= (max_distance / near)^b
        while n ** (half - near) * near ** b < int(max_distance) ** b * near ** (half - near):
            n += 1
            if n > 1024:
                raise ValueError(f"max_distance {max_distance} with {num_buckets} buckets: the last bucket must begin at 1024 or before")
        found.append(n)
    return (C.c_int * len(found))(*found)


@functools.lru_cache(maxsize=None)
def _borders(num_buckets, max_distance):
    found = relbias_borders(num_buckets, max_distance)
    return found, C.addressof(found)


def _heads(t):
    """[B, S, H, 64] with a dense last dimension, whole 16-byte pieces between rows and an aligned base; copied only where it is not so."""
    sb, ss, sh, one = t.stride()
    if one != 1 or sb % 8 or ss % 8 or sh % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _relbias(name, q, k, v, table, max_distance, scale, key_mask):
    """(device, descriptor, what it points at) of a call."""
    dev = _same_device(q, k, v, table, key_mask)
    shape = q.shape
    for n, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != torch.bfloat16 or t.shape != shape or len(shape) != 4 or shape[3] != 64:
            raise ValueError(f"{name}: q, k, v are bfloat16 [B, S, H, 64] of one shape; {n} is {t.dtype} {list(t.shape)}")
    B, S, H, _ = shape
    if H < 1:
        raise ValueError(f"{name}: no heads")
    if table.dtype != torch.bfloat16 or table.dim() != 2 or table.shape[1] != H:
        raise ValueError(f"{name}: the table is bfloat16 [num_buckets, {H}], got {table.dtype} {list(table.shape)}")
    if not (scale == 0 or 1e-20 <= abs(scale) <= 1e20):
        raise ValueError(f"{name}: the scale is 0 or of a magnitude in [1e-20, 1e20], got {scale}")
    borders, borders_at = _borders(table.shape[0], max_distance)
    q, k, v, table = _heads(q), _heads(k), _heads(v), table.contiguous()
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != (B, S):
            raise ValueError(f"{name}: key_mask is bool [{B}, {S}], True where a key counts, got {key_mask.dtype} {list(key_mask.shape)}")
        if key_mask.stride(1) != 1 or key_mask.stride(0) < 0:
            key_mask = key_mask.contiguous()
    d = _lib.RELBIAS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], table.data_ptr(),
                          0 if key_mask is None else key_mask.data_ptr(), 0 if key_mask is None else key_mask.stride(0), B, S, H, scale,
                          table.shape[0], borders_at, len(borders))
    return dev, d, (q, k, v, table, key_mask)


def relbias_attn(q, k, v, table, max_distance=128, scale=1.0, key_mask=None, need_lse=False):
    """Self-attention with a learned bias by relative position: S_ij = scale q_i·k_j + table[bucket(j − i), h], O = softmax(S) V over the keys that count.
    q, k, v bfloat16 [B, S, H, 64] (views of a packed projection included), table bfloat16 [num_buckets, H] (buckets of both directions, exact up to
    num_buckets / 4, logarithmic up to max_distance), key_mask bool [B, S], True where a key counts.  A row without keys gives 0, also where buckets
    at -inf leave none; what stands at keys that do not count reaches nothing.  |v| up to 1e22: weighted sums are held in float32 before they are normalized.
    -> o bfloat16 [B, S, H, 64]; with need_lse (o, lse), where lse (float32, flat) is what
    `relbias_attn_backward` needs besides o: the rows' log-sums to base 2 [B, H, S], then, from the next 16 bytes on, o's rounding remainders
    (bfloat16 [B, S, H, 64]).  P then multiplies v in two parts, and o is a little more exact than without."""
    dev, d, keep = _relbias("relbias_attn", q, k, v, table, max_distance, scale, key_mask)
    o = _like(q, torch.bfloat16)
    n = o.numel() // 64
    lse = q.new_empty((_lse_pad(n) + 32 * n,), dtype=torch.float32) if need_lse else None
    at = lse.data_ptr() if need_lse else None
    _run("relbias_attn", dev, _lib.load().aether_relbias_attn, d, o.data_ptr(), at + 4 * _lse_pad(n) if need_lse else None, at)
    return (o, lse) if need_lse else o


def _lse_pad(n):
    return (n + 3) // 4 * 4         # the remainders behind the log-sums begin at whole 16 bytes


_strides = struct.Struct("@3l").pack


def relbias_attn_backward(do, q, k, v, o, lse, table, max_distance=128, scale=1.0, key_mask=None, need_dtable=True):
    """Gradients of `relbias_attn` from its inputs, its output o and its lse: -> (dq, dk, dv bfloat16 [B, S, H, 64], thirds of one packed
    [B, S, 3, H, 64] buffer; dtable bfloat16 [num_buckets, H] or None).  dk and dv are 0 at keys that do not count.  P comes from
    the log-sums again: a row whose largest score lies beyond ±7e5 has no gradient.  Summed in an order that
    depends on the sizes alone."""
    name = "relbias_attn_backward"
    dev, d, keep = _relbias(name, q, k, v, table, max_distance, scale, key_mask)
    _same_device(q, do, o, lse)
    B, S, H, _ = q.shape
    for n, t in (("do", do), ("o", o)):
        if t.dtype != torch.bfloat16 or t.shape != q.shape:
            raise ValueError(f"{name}: {n} is bfloat16 {list(q.shape)}, got {t.dtype} {list(t.shape)}")
    n = B * H * S
    if lse.dtype != torch.float32 or tuple(lse.shape) != (_lse_pad(n) + 32 * n,):
        raise ValueError(f"{name}: lse is what relbias_attn gave with need_lse, float32 [{_lse_pad(n) + 32 * n}], got {lse.dtype} {list(lse.shape)}")
    do, o, lse = _heads(do), _heads(o), _vector(lse)
    dqkv = q.new_empty(B, S, 3, H, 64)
    dq, dk, dv = dqkv.unbind(2)
    dtable = _like(table, torch.bfloat16) if need_dtable else None
    lib = _lib.load()
    nbytes = lib.aether_relbias_attn_bwd_workspace_bytes(d, need_dtable)
    ws = _workspace(q, nbytes)
    st = _strides(S * 3 * H * 64, 3 * H * 64, 64)
    _run(name, dev, lib.aether_relbias_attn_bwd, d, do.data_ptr(), _strides(*do.stride()[:3]), o.data_ptr(), _strides(*o.stride()[:3]), lse.data_ptr() + 4 * _lse_pad(n), lse.data_ptr(),
         dq.data_ptr(), st, dk.data_ptr(), st, dv.data_ptr(), st, _lib.ptr(dtable), ws.data_ptr(), nbytes)
    return dq, dk, dv, dtable


_ACTS = {"gelu_tanh": _lib.AETHER_ACT_GELU_TANH, "silu": _lib.AETHER_ACT_SILU}


def _ff_operands(name, x, wg, wu, act, dtype):
    if act not in _ACTS:
        raise ValueError(f"{name}: act is one of {list(_ACTS)}, got {act!r}")
    if x.dtype != dtype or wg.dtype != dtype or wu.dtype != dtype:
        raise ValueError(f"{name}: x, wg and wu are {dtype}, got {x.dtype}, {wg.dtype}, {wu.dtype}")
    if x.dim() < 1 or wg.dim() != 2 or wg.shape != wu.shape or wg.shape[1] != x.shape[-1]:
        raise ValueError(f"{name}: x [..., K], wg and wu [F, K], got {list(x.shape)}, {list(wg.shape)}, {list(wu.shape)}")
    F, K = wg.shape
    if F == 0 or F % 32 or K == 0 or K * x.element_size() % 128:
        raise ValueError(f"{name}: F must be a multiple of 32 and K of {128 // x.element_size()}, got F = {F}, K = {K}")
    wg, wu = _rows(wg, K), _rows(wu, K)
    if wg.stride(0) != wu.stride(0):
        wg, wu = wg.contiguous(), wu.contiguous()
    return _rows(x, K), wg, wu, F, K


def gated_ff(x, wg, wu, act="gelu_tanh", need_gu=False):
    """h = act(x wgᵀ) ⊙ (x wuᵀ): both projections, the activation and the product in one kernel.  x bfloat16 [..., K], wg and wu bfloat16 [F, K], K a multiple
    of 64, F of 32; act "gelu_tanh" or "silu".  -> h bfloat16 [..., F]; with need_gu (h, gu), where gu float32 [rows, 2F] holds both projections for
    `gated_ff_backward`; that takes rows · 2F (rows rounded up to 64) and 2F · K below 2^31, and need_gu is refused beyond."""
    dev = _same_device(x, wg, wu)
    x2, wg, wu, F, K = _ff_operands("gated_ff", x, wg, wu, act, torch.bfloat16)
    M = x2.shape[0]
    h = x.new_empty(*x.shape[:-1], F)
    gu = x.new_empty(M, 2 * F, dtype=torch.float32) if need_gu else None
    if M:
        _run("gated_ff", dev, _lib.load().aether_gated_ff, x2.data_ptr(), x2.stride(0), wg.data_ptr(), wu.data_ptr(), wg.stride(0), h.data_ptr(), F, _lib.ptr(gu),
             M, F, K, _ACTS[act])
    return (h, gu) if need_gu else h


def gated_ff_e4m3(x, x_scale, wg, wg_scale, wu, wu_scale, act="gelu_tanh"):
    """`gated_ff` on 8-bit operands: x float8_e4m3fn [..., K] with x_scale float32 [...] (`rms_norm_e4m3`), wg and wu float8_e4m3fn [F, K] with a scale float32 [F]
    each (`quantize_rows_e4m3`); K a multiple of 128, F of 32.  -> h bfloat16 [..., F]."""
    name = "gated_ff_e4m3"
    dev = _same_device(x, wg, wu, x_scale, wg_scale, wu_scale)
    x2, wg, wu, F, K = _ff_operands(name, x, wg, wu, act, torch.float8_e4m3fn)
    for n, t, shape in (("x_scale", x_scale, x.shape[:-1]), ("wg_scale", wg_scale, (F,)), ("wu_scale", wu_scale, (F,))):
        if t.dtype != torch.float32 or tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name}: {n} is float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    M = x2.shape[0]
    h = x.new_empty(*x.shape[:-1], F, dtype=torch.bfloat16)
    if M:
        x_scale, wg_scale, wu_scale = x_scale.contiguous(), _vector(wg_scale), _vector(wu_scale)
        _run(name, dev, _lib.load().aether_gated_ff_e4m3, x2.data_ptr(), x2.stride(0), x_scale.data_ptr(), wg.data_ptr(), wg_scale.data_ptr(), wu.data_ptr(),
             wu_scale.data_ptr(), wg.stride(0), h.data_ptr(), F, M, F, K, _ACTS[act])
    return h


def gated_ff_backward(dh, x, wg, wu, gu, act="gelu_tanh", need_dx=True, need_dw=True):
    """Gradients of `gated_ff` (bfloat16 operands) from its inputs and gu: dh bfloat16 [..., F] -> (dx bfloat16 like x, dwg, dwu bfloat16 [F, K], the halves of one
    [2F, K] buffer; None for what is not needed).  dh act'(g) u and dh act(g) are rounded to bf16 once, as operands of the products; sums are fp32, in an order that depends on the
    sizes alone."""
    name = "gated_ff_backward"
    dev = _same_device(x, dh, wg, wu, gu)
    x2, wg, wu, F, K = _ff_operands(name, x, wg, wu, act, torch.bfloat16)
    M = x2.shape[0]
    if dh.dtype != torch.bfloat16 or tuple(dh.shape) != (*x.shape[:-1], F):
        raise ValueError(f"{name}: dh is bfloat16 {[*x.shape[:-1], F]}, got {dh.dtype} {list(dh.shape)}")
    if gu.dtype != torch.float32 or tuple(gu.shape) != (M, 2 * F):
        raise ValueError(f"{name}: gu is float32 [{M}, {2 * F}], as gated_ff gave it, got {gu.dtype} {list(gu.shape)}")
    dx = _like(x, torch.bfloat16) if need_dx else None
    dw = (torch.empty if M else torch.zeros)(2 * F, K, dtype=torch.bfloat16, device=dev) if need_dw else None
    out = dx, dw[:F] if need_dw else None, dw[F:] if need_dw else None
    if M == 0 or not (need_dx or need_dw):
        return out
    d2, gu = _rows(dh, F), _rows(gu, 2 * F)
    if gu.stride(0) != 2 * F:
        gu = gu.contiguous()
    lib = _lib.load()
    nbytes = lib.aether_gated_ff_bwd_workspace_bytes(M, F, K)
    ws = _workspace(x, nbytes)
    _run(name, dev, lib.aether_gated_ff_bwd, d2.data_ptr(), d2.stride(0), x2.data_ptr(), x2.stride(0), wg.data_ptr(), wu.data_ptr(), wg.stride(0), gu.data_ptr(),
         _lib.ptr(dx), K, _lib.ptr(dw), M, F, K, _ACTS[act], ws.data_ptr(), nbytes)
    return out
