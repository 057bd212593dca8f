"""The text encoder's operators on the host: what they refuse (before anything reaches a device) and what they compute there."""
import pytest
import torch


# ---- C entries: argument checks come before any launch, so they run without a device -------------------------------------------------
def _norm(lib, x=4096, xt=1, ldx=64, delta=None, ldd=64, res=None, ldr=64, w=4096, y=4096, ldy=64, scale=None, rows=4, D=64):
    return lib.aether_rms_norm(x, xt, ldx, delta, ldd, res, ldr, w, 1e-6, y, ldy, scale, rows, D, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(xt=2), -1, b"bf16 or fp32"),
    (dict(rows=-1), -2, b"rows"),
    (dict(D=0), -2, b"multiple of 8"),
    (dict(D=60), -2, b"multiple of 8"),
    (dict(D=16392), -2, b"16384"),
    (dict(x=None), -1, b"null"),
    (dict(w=None), -1, b"null"),
    (dict(y=None), -1, b"null"),
    (dict(delta=4096), -1, b"res"),
    (dict(ldx=60), -3, b"leading"),
    (dict(ldy=60), -3, b"leading"),
    (dict(delta=4096, res=4096, ldd=63), -3, b"leading"),
    (dict(x=4100), -3, b"aligned"),
    (dict(w=4100), -3, b"aligned"),
    (dict(y=4104), -3, b"aligned"),
    (dict(y=4100, scale=4096), -3, b"aligned"),
])
def test_rms_norm_entry_refuses(hip_lib, kw, code, text):
    assert _norm(hip_lib, **kw) == code and text in hip_lib.aether_last_error()


def test_rms_norm_entry_without_rows(hip_lib):
    assert _norm(hip_lib, rows=0, x=None, y=None) == 0


def _norm_bwd(lib, dy=4096, ldy=64, res=4096, xt=1, ldr=64, dres=None, lds=64, w=4096, dx=4096, ldx=64, dd=None, ldd=64, dw=4096, rows=4, D=64, ws=4096, n=1 << 20):
    return lib.aether_rms_norm_bwd(dy, ldy, res, xt, ldr, dres, lds, w, 1e-6, dx, ldx, dd, ldd, dw, rows, D, ws, n, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(xt=7), -1, b"bf16 or fp32"),
    (dict(D=12), -2, b"multiple of 8"),
    (dict(dw=None), -1, b"null"),
    (dict(dy=None), -1, b"null"),
    (dict(res=None), -1, b"null"),
    (dict(ldy=4), -3, b"leading"),
    (dict(dres=4096, lds=4), -3, b"leading"),
    (dict(dx=4104), -3, b"aligned"),
    (dict(ws=None), -1, b"workspace"),
    (dict(n=4 * 64 * 4 - 1), -1, b"workspace"),
])
def test_rms_norm_backward_entry_refuses(hip_lib, kw, code, text):
    assert _norm_bwd(hip_lib, **kw) == code and text in hip_lib.aether_last_error()


@pytest.mark.parametrize("args,code", [
    ((4096, 64, 4096, 64, 4096, 4, 60, None), -2), ((4096, 64, 4096, 64, 4096, -1, 64, None), -2), ((None, 64, 4096, 64, 4096, 4, 64, None), -1),
    ((4096, 64, 4096, 64, None, 4, 64, None), -1), ((4100, 64, 4096, 64, 4096, 4, 64, None), -3), ((4096, 64, 4096, 4, 4096, 4, 64, None), -3),
    ((None, 64, None, 64, None, 0, 64, None), 0)])
def test_quantize_rows_entry_refuses(hip_lib, args, code):
    assert hip_lib.aether_quantize_rows_e4m3(*args) == code


# ---- Python wrappers: no CPU fallback ---------------------------------------------------------------------------------------------------
def test_wrappers_refuse_host_tensors(hip_lib):
    from aether_amd import ops
    x, w = torch.zeros(2, 64), torch.ones(64)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_e4m3(x, w), lambda: ops.rms_norm_backward(x.bfloat16(), x, w),
                 lambda: ops.quantize_rows_e4m3(x.bfloat16())):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()
