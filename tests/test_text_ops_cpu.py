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


def _norm_bwd(lib, dy=4096, ldy=64, res=4096, xt=1, ldr=64, delta=None, ldl=64, dres=None, lds=64, w=4096, dx=4096, ldx=64, dd=None, ldd=64, dw=4096, rows=4, D=64, ws=4096, n=1 << 20):
    return lib.aether_rms_norm_bwd(dy, ldy, res, xt, ldr, delta, ldl, dres, lds, w, 1e-6, dx, ldx, dd, ldd, dw, rows, D, ws, n, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(xt=7), -1, b"bf16 or fp32"),
    (dict(D=12), -2, b"multiple of 8"),
    (dict(dw=None), -1, b"null"),
    (dict(dy=None), -1, b"null"),
    (dict(res=None), -1, b"null"),
    (dict(ldy=4), -3, b"leading"),
    (dict(dres=4096, lds=4), -3, b"leading"),
    (dict(delta=4096, ldl=4), -3, b"leading"),
    (dict(delta=4104), -3, b"aligned"),
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


# ---- attention with a relative position bias --------------------------------------------------------------------------------------------
def _relbias(lib, o=4096, **kw):
    import ctypes as C
    from aether_amd import _lib
    a = dict(low=None, lse=None, q=4096, k=4096, v=4096, st=(64 * 64, 64, 64 * 32), table=4096, mask=None, B=1, S=32, H=2, num_buckets=32, borders=(12, 16, 23, 32, 46, 64, 91))
    a.update(kw)
    b = a["borders"]
    arr = (C.c_int * len(b))(*b) if b is not None else None
    d = _lib.AetherRelbias(a["q"], a["k"], a["v"], a["st"], a["st"], a["st"], a["table"], a["mask"], 0, a["B"], a["S"], a["H"], a.get("scale", 1.0), a["num_buckets"], arr, len(b or ()))
    return lib.aether_relbias_attn(C.byref(d), o, a["low"], a["lse"], None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(B=-1), -2, b"negative"), (dict(S=-1), -2, b"negative"), (dict(H=0), -2, b"negative"), (dict(S=65537), -2, b"65536"),
    (dict(num_buckets=3, borders=()), -2, b"num_buckets"), (dict(num_buckets=2, borders=()), -2, b"num_buckets"), (dict(num_buckets=130), -2, b"num_buckets"),
    (dict(borders=(12, 16)), -1, b"borders"), (dict(borders=None), -1, b"borders"), (dict(borders=(7, 16, 23, 32, 46, 64, 91)), -1, b"borders"),
    (dict(borders=(12, 11, 23, 32, 46, 64, 91)), -1, b"borders"), (dict(borders=(12, 16, 23, 32, 46, 64, 1025)), -2, b"1024"),
    (dict(table=None), -1, b"table"), (dict(q=None), -1, b"operand"), (dict(v=None), -1, b"operand"), (dict(k=4104), -3, b"aligned"),
    (dict(st=(4096, 60, 64)), -3, b"aligned"), (dict(st=(4096, -64, 64)), -2, b"stride"), (dict(st=(-4096, 64, 64)), -2, b"stride"),
    (dict(st=(0, 1 << 15, 64), S=65536), -2, b"4 GiB"), (dict(o=None), -1, b"output"), (dict(low=4096), -1, b"together"), (dict(lse=4096), -1, b"together"), (dict(low=4104, lse=4096), -3, b"aligned"), (dict(o=4104), -3, b"aligned"),
    (dict(B=1 << 20, H=1 << 10, S=65536), -2, b"blocks"), (dict(scale=float("nan")), -1, b"scale"), (dict(scale=float("inf")), -1, b"scale"), (dict(scale=1e-30), -1, b"scale"),
])
def test_relbias_entry_refuses(hip_lib, kw, code, text):
    assert _relbias(hip_lib, **kw) == code and text in hip_lib.aether_last_error()


def test_relbias_entry_without_rows(hip_lib):
    assert _relbias(hip_lib, S=0, q=None, table=None, o=None) == 0 and _relbias(hip_lib, B=0, q=None, table=None, o=None) == 0
    assert hip_lib.aether_relbias_attn(None, 4096, None, None, None) == -1


def test_relbias_descriptor_bytes():
    """The packed descriptor has the bytes of the declared structure."""
    import ctypes as C
    from aether_amd import _lib
    arr = (C.c_int * 7)(*range(7))
    st = (2 ** 40 + 1, 2 ** 33, 64), (5, 6, 7), (8, 9, 10)
    d = _lib.AetherRelbias(2 ** 47 + 4096, 4112, 4128, *st, 8192, None, 2 ** 35, 3, 65536, 64, -0.125, 32, arr, 7)
    assert _lib.RELBIAS.size == C.sizeof(d)
    assert _lib.RELBIAS.pack(2 ** 47 + 4096, 4112, 4128, *st[0], *st[1], *st[2], 8192, 0, 2 ** 35, 3, 65536, 64, -0.125, 32, C.addressof(arr), 7) == bytes(d)


def test_bucket_borders():
    """The borders against the published definition evaluated in float64 (away from its own roundings) and by counting."""
    import math
    from aether_amd.ops import relbias_borders
    from relbias_reference import bucket
    assert list(relbias_borders(32, 128)) == [12, 16, 23, 32, 46, 64, 91]
    for nb, md in ((4, 2), (6, 3), (8, 20), (10, 9), (32, 128), (64, 256), (128, 1000), (32, 32), (12, 1024), (32, 1024)):
        half = nb // 2
        near = half // 2
        borders = list(relbias_borders(nb, md))
        assert len(borders) == half - near - 1 and borders == sorted(borders)
        for n in range(1, 1400):
            ours = n if n < near else near + sum(b <= n for b in borders)
            assert ours == bucket(-n, nb, md) == bucket(n, nb, md) - half
            if n >= near:
                x = math.log(n / near) / math.log(md / near) * (half - near)
                if abs(x - round(x)) > 1e-9:
                    assert ours == min(half - 1, near + math.floor(x))
    for nb, md in ((2, 10), (5, 10), (130, 1000), (32, 8), (32, 7), (32, 128.5), (32, 100000)):
        with pytest.raises(ValueError):
            relbias_borders(nb, md)


@pytest.mark.parametrize("kw,code,text", [
    (dict(lse=None), -1, b"lse"), (dict(low=None), -1, b"o_low"), (dict(low=4104), -3, b"aligned"), (dict(go=None), -1, b"operand"), (dict(o=4100), -3, b"aligned"), (dict(dq=None), -1, b"operand"),
    (dict(st=(4096, 4, 64)), -3, b"aligned"), (dict(ws=None), -1, b"workspace"), (dict(ws=4104), -1, b"workspace"), (dict(n=32 * 2 * 4 + 255), -1, b"workspace"),
])
def test_relbias_backward_entry_refuses(hip_lib, kw, code, text):
    import ctypes as C
    from aether_amd import _lib
    a = dict(go=4096, o=4096, low=4096, lse=4096, dq=4096, dk=4096, dv=4096, dt=4096, ws=4096, n=1 << 20, st=(64 * 64, 64, 64 * 32))
    a.update(kw)
    b = (C.c_int * 7)(12, 16, 23, 32, 46, 64, 91)
    ok = (64 * 64, 64, 64 * 32)
    d = _lib.AetherRelbias(4096, 4096, 4096, ok, ok, ok, 4096, None, 0, 1, 32, 2, 1.0, 32, b, 7)
    assert hip_lib.aether_relbias_attn_bwd_workspace_bytes(C.byref(d), 1) == 32 * 2 * 4 + 2 * 32 * 4
    assert hip_lib.aether_relbias_attn_bwd_workspace_bytes(C.byref(d), 0) == 32 * 2 * 4
    st = (C.c_long * 3)(*a["st"])
    rc = hip_lib.aether_relbias_attn_bwd(C.byref(d), a["go"], st, a["o"], st, a["low"], a["lse"], a["dq"], st, a["dk"], st, a["dv"], st, a["dt"], a["ws"], a["n"], None)
    assert rc == code and text in hip_lib.aether_last_error()


# ---- gated feed-forward -----------------------------------------------------------------------------------------------------------------
_FF = dict(x=4096, ldx=128, wg=4096, wu=4096, ldw=128, h=4096, ldh=64, M=4, F=64, K=128, act=0)


@pytest.mark.parametrize("kw,code,text", [
    (dict(act=2), -1, b"activation"), (dict(M=-1), -2, b"negative"), (dict(F=0), -2, b"positive"), (dict(K=0), -2, b"positive"), (dict(F=48), -2, b"multiple of 32"),
    (dict(K=96), -2, b"64"), (dict(x=None), -1, b"null"), (dict(wu=None), -1, b"null"), (dict(ldx=64), -2, b"shorter"), (dict(ldw=64), -2, b"shorter"),
    (dict(ldx=132), -3, b"aligned"), (dict(x=4104), -3, b"aligned"), (dict(F=1 << 20, K=4096, ldw=4096, ldx=4096, ldh=1 << 20), -2, b"4 GiB"),
    (dict(ldx=1 << 23), -2, b"too far"), (dict(h=None), -1, b"output"), (dict(ldh=32), -3, b"aligned"), (dict(h=4104), -3, b"aligned"), (dict(M=(1 << 30) + 1), -2, b"rows"),
])
def test_gated_ff_entry_refuses(hip_lib, kw, code, text):
    a = {**_FF, **kw}
    rc = hip_lib.aether_gated_ff(a["x"], a["ldx"], a["wg"], a["wu"], a["ldw"], a["h"], a["ldh"], None, a["M"], a["F"], a["K"], a["act"], None)
    assert rc == code and text in hip_lib.aether_last_error()


@pytest.mark.parametrize("kw,code", [(dict(K=64), -2), (dict(sx=None), -1), (dict(sg=None), -1), (dict(su=4100), -3), (dict(h=None), -1), (dict(ldh=60), -3), (dict(ldw=136), -3)])
def test_gated_ff_e4m3_entry_refuses(hip_lib, kw, code):
    a = {**_FF, **dict(sx=4096, sg=4096, su=4096), **kw}
    assert hip_lib.aether_gated_ff_e4m3(a["x"], a["ldx"], a["sx"], a["wg"], a["sg"], a["wu"], a["su"], a["ldw"], a["h"], a["ldh"], a["M"], a["F"], a["K"], a["act"], None) == code


@pytest.mark.parametrize("kw,code,text", [
    (dict(dw=None, dx=None), -1, b"null"), (dict(dh=None), -1, b"null"), (dict(gu=None), -1, b"null"), (dict(M=0), -2, b"rows"), (dict(lddh=32), -3, b"aligned"),
    (dict(lddx=64), -3, b"aligned"), (dict(dw=4104), -3, b"aligned"), (dict(ws=None), -1, b"workspace"), (dict(n=1000), -1, b"workspace"), (dict(act=5), -1, b"activation"),
    (dict(M=1 << 26), -2, b"4 GiB"),
])
def test_gated_ff_backward_entry_refuses(hip_lib, kw, code, text):
    a = {**_FF, **dict(dh=4096, lddh=64, gu=4096, dx=4096, lddx=128, dw=4096, ws=4096, n=1 << 30), **kw}
    rc = hip_lib.aether_gated_ff_bwd(a["dh"], a["lddh"], a["x"], a["ldx"], a["wg"], a["wu"], a["ldw"], a["gu"], a["dx"], a["lddx"], a["dw"], a["M"], a["F"], a["K"], a["act"],
                                     a["ws"], a["n"], None)
    assert rc == code and text in hip_lib.aether_last_error()


def test_gated_ff_entries_without_rows(hip_lib):
    assert hip_lib.aether_gated_ff(None, 128, None, None, 128, None, 64, None, 0, 64, 128, 0, None) == 0
    assert hip_lib.aether_gated_ff_e4m3(None, 128, None, None, None, None, None, 128, None, 64, 0, 64, 128, 0, None) == 0


@pytest.mark.parametrize("kw,refused", [(dict(B=1 << 20, H=64, S=1), True), (dict(B=(1 << 20) - 1, H=64, S=1), False), (dict(B=1 << 18, H=128, S=40), True),
                                        (dict(B=1 << 14, H=64, S=2000), True), (dict(B=1 << 26, H=1, S=32), True), (dict(B=(1 << 25), H=1, S=64), True),
                                        (dict(B=(1 << 25) - 1, H=1, S=64), False)])
def test_relbias_grids_beyond_a_launch(hip_lib, kw, refused):
    """A grid of 2^32 threads or more would be cut short: such calls are refused, forward and backward.  (The others come as far as the missing output.)"""
    import ctypes as C
    from aether_amd import _lib
    text = b"blocks" if refused else b"output"
    assert _relbias(hip_lib, o=None, st=(0, 64, 0), **kw) == (-2 if refused else -1) and text in hip_lib.aether_last_error()
    st = (0, 64, 0)
    b = (C.c_int * 7)(12, 16, 23, 32, 46, 64, 91)
    d = _lib.AetherRelbias(4096, 4096, 4096, st, st, st, 4096, None, 0, kw["B"], kw["S"], kw["H"], 1.0, 32, b, 7)
    assert (hip_lib.aether_relbias_attn_bwd_workspace_bytes(C.byref(d), 1) == 0) == refused


def test_gated_ff_backward_refuses_a_row_stride_beyond_32_bits(hip_lib):
    """The product behind dx takes its row stride as 32 bits: one that would be cut is refused before anything is enqueued."""
    a = {**_FF, **dict(M=70000, F=64)}
    lddx = (1 << 32) + 128
    rc = hip_lib.aether_gated_ff_bwd(4096, 64, a["x"], a["ldx"], a["wg"], a["wu"], a["ldw"], 4096, 4096, lddx, None, a["M"], a["F"], a["K"], 0, 4096, 1 << 40, None)
    assert rc == -2 and b"too far" in hip_lib.aether_last_error()


@pytest.mark.parametrize("kw", [dict(M=1 << 25, F=32, K=64), dict(M=104896, F=10240, K=4096, ldx=4096, ldw=4096, ldh=10240), dict(F=8192, K=131072, ldx=131072, ldw=131072, ldh=8192)])
def test_gated_ff_refuses_projections_that_have_no_backward_pass(hip_lib, kw):
    """What the backward pass does not take is refused where its projections are asked for, not after the forward pass has run."""
    a = {**_FF, **kw}
    text = b"4 GiB"
    rc = hip_lib.aether_gated_ff_bwd(4096, a["F"], a["x"], a["ldx"], a["wg"], a["wu"], a["ldw"], 4096, 4096, a["ldx"], 4096, a["M"], a["F"], a["K"], 0, 4096, 1 << 60, None)
    assert rc == -2 and text in hip_lib.aether_last_error()
    rc = hip_lib.aether_gated_ff(a["x"], a["ldx"], a["wg"], a["wu"], a["ldw"], a["h"], a["ldh"], 4096, a["M"], a["F"], a["K"], 0, None)
    assert rc == -2 and text in hip_lib.aether_last_error()


@pytest.mark.parametrize("K,code", [(0x7ffffff8, -2), ((1 << 30) + 8, -2), (1 << 30, -1)])
def test_quantize_rows_refuses_what_its_counter_does_not_hold(hip_lib, K, code):
    """The kernel counts a row's elements in 32 bits, 2048 at a time: K ends at 2^30.  (-1: as far as the missing operand.)"""
    assert hip_lib.aether_quantize_rows_e4m3(None, K, 4096, K, 4096, 4, K, None) == code
