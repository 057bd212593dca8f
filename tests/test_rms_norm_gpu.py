"""rms_norm and its backward pass against the formulas in float64 on the same inputs.

Tolerances.  One rounding to bf16 is off by at most 2^-8 relative (half a step), so |got − exact| <= 2^-8 |exact| + what fp32 arithmetic
adds: a row sum of D squares in fp32 is off by at most D · 2^-24 relative in the worst order, in the tree order used here by (8 NCH + 8) · 2^-24 < 2^-17;
r carries half of that and one rounding of its own.  F32 = 2^-16 relative covers norm, product and sum.  Gradients are sums of terms of either sign:
their error is relative to the sum of magnitudes, not to the result."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32 = 2.0 ** -8, 2.0 ** -16


def _inputs(rows, D, stream, seed=0, cuda=None):
    g = torch.Generator().manual_seed(seed + 1000 * rows + D)
    x = (torch.randn(rows, D, generator=g) * torch.exp(torch.randn(D, generator=g))).to(stream)
    return (t.to(cuda) for t in (x, torch.randn(rows, D, generator=g).to(torch.bfloat16), 0.5 + torch.rand(D, generator=g),
                                 torch.randn(rows, D, generator=g).to(torch.bfloat16), torch.randn(rows, D, generator=g).to(stream)))


def _exact(x, delta, w, eps=1e-6):
    h = x.double() + (delta.double() if delta is not None else 0)
    return h, h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()


def _near(got, want, rel, floor=0.0):
    err = (got.double() - want).abs()
    lim = rel * want.abs() + floor
    assert got.shape == want.shape and bool((err <= lim).all()), f"worst excess {(err - lim).max().item():.3e} at limit {lim.max().item():.3e}"


SIZES = [(1, 8), (3, 64), (5, 504), (226, 512), (7, 520), (9, 1024), (33, 1032), (2, 2048), (17, 2056), (226, 4096), (5, 4104), (3, 8192), (2, 16384),
         (2500, 128), (4099, 1040)]     # the last two: more rows than one pass of the grid


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D", SIZES)
def test_forward(cuda, hip_lib, rows, D, stream):
    from aether_amd import ops
    x, delta, w, _, _ = _inputs(rows, D, stream, cuda=cuda)
    h, want = _exact(x, delta, w)
    y, res = ops.rms_norm(x, w, delta=delta)
    assert y.dtype == torch.bfloat16 and res.dtype == stream
    _near(y, want, BF16 + F32)
    assert torch.equal(res, (x.float() + delta.float()).to(stream))
    h, want = _exact(x, None, w)
    y, res = ops.rms_norm(x, w)
    assert res is x
    _near(y, want, BF16 + F32)


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D", SIZES)
def test_e4m3(cuda, hip_lib, rows, D, stream):
    from aether_amd import ops
    x, delta, w, _, _ = _inputs(rows, D, stream, seed=1, cuda=cuda)
    _, want = _exact(x, delta, w)
    q, scale, res = ops.rms_norm_e4m3(x, w, delta=delta)
    assert q.dtype == torch.float8_e4m3fn and scale.shape == (rows,)
    assert torch.equal(res, (x.float() + delta.float()).to(stream))
    m, e = torch.frexp(scale)
    assert bool((m == 0.5).all()), "scales are powers of two"
    top = want.abs().amax(-1) / scale.double()
    assert bool((top <= 448 * (1 + F32)).all()) and bool((top > 224 * (1 - F32)).all()), "the smallest power of two that fits"
    # half a step of e4m3: 2^-4 relative, 2^-10 among the subnormals (steps of 2^-9)
    _near(q.float(), want / scale.double()[:, None], 2.0 ** -4 + F32, 2.0 ** -10 + 448 * F32)


def test_e4m3_borders(cuda, hip_lib):
    """Rows whose largest value is at 448 · 2^k and next to it, a row of zeros, and rows that hold an infinity or a NaN."""
    from aether_amd import ops
    x = torch.zeros(8, 64)
    for i, v in enumerate((448.0, 448.0 * 2 ** 10, 449.0, 1.75, 1.7578125)):
        x[i, 3], x[i, 5] = v, -v / 2
    x[5] = 0.0
    x[6, 0], x[7, 1] = math.inf, math.nan
    q, s = ops.quantize_rows_e4m3(x.to(torch.bfloat16).to(cuda))
    xb = x.to(torch.bfloat16).float()
    assert s[:6].tolist() == [1.0, 1024.0, 2.0 if xb[2, 3] > 448 else 1.0, 2.0 ** -8, 2.0 ** -7, 2.0 ** -126]
    assert bool(torch.isnan(s[6:]).all()) and bool(torch.isnan(q[6:].float()).all())
    got = q[:6].float().cpu() * s[:6].cpu()[:, None]
    assert bool(((got - xb[:6]).abs() <= 2.0 ** -4 * xb[:6].abs()).all())
    # the norm keeps that: one such value makes its row NaN, and no other row
    w = torch.ones(64, device=cuda)
    q, s, _ = ops.rms_norm_e4m3(x.to(cuda), w)
    assert bool(torch.isnan(s[6:]).all()) and bool(torch.isnan(q[6:].float()).all()) and bool(torch.isfinite(s[:6]).all()) and bool(torch.isfinite(q[:6].float()).all())
    y, _ = ops.rms_norm(x.to(cuda), w)
    assert bool(torch.isfinite(y[:6].float()).all()) and bool(torch.isnan(y[7].float()).all()) and bool(torch.isnan(y[6, 0].float()))


@pytest.mark.parametrize("rows,K", [(1, 8), (3, 64), (5, 2048), (7, 2056), (2, 10240)])
def test_quantize_rows(cuda, hip_lib, rows, K):
    from aether_amd import ops
    g = torch.Generator().manual_seed(K)
    wide = torch.randn(rows, K + 24, generator=g).to(torch.bfloat16).to(cuda)
    x = wide[:, 8:8 + K]                                     # rows with a stride, not at the base
    q, s = ops.quantize_rows_e4m3(x)
    amax = x.float().abs().amax(-1)
    assert torch.equal(s, torch.exp2(torch.ceil(torch.log2(amax.double() / 448))).float())
    assert torch.equal(q.float(), (x.float() / s[:, None]).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("with_dres", [True, False])
@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D", SIZES)
def test_backward(cuda, hip_lib, rows, D, stream, with_dres):
    from aether_amd import ops
    x, _, w, dy, dres = _inputs(rows, D, stream, seed=2, cuda=cuda)
    dres = dres if with_dres else None
    h, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * wd
    dx, dw = torch.autograd.grad((y * dy.double()).sum() + ((h * dres.double()).sum() if with_dres else 0), (h, wd))
    gx, gd, gw = ops.rms_norm_backward(dy, x, w, dres=dres, need_ddelta=True)
    assert gx.dtype == stream and gd.dtype == torch.bfloat16 and gw.dtype == torch.float32
    with torch.no_grad():
        r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
        n = (dy.double() * wd).abs()
        terms = r * (n + (h * r).abs() * (n * (h * r).abs()).mean(-1, keepdim=True)) + (dres.double().abs() if with_dres else 0)
        wterms = (dy.double() * h * r).abs().sum(0)
    err = (gx.double() - dx).abs()
    assert bool((err <= F32 * terms + (BF16 if stream == torch.bfloat16 else 0.0) * dx.abs()).all())
    assert torch.equal(gd, gx.to(torch.bfloat16))
    # a sum of `rows` terms in fp32: at most (terms in a row slot + 32 + 2) roundings each, of the sum of magnitudes
    assert bool(((gw.double() - dw).abs() <= (F32 + (rows / 512 + 64) * 2.0 ** -24) * wterms).all())
    assert ops.rms_norm_backward(dy, x, w, dres=dres)[1] is None
    again = ops.rms_norm_backward(dy, x, w, dres=dres)
    assert torch.equal(again[0], gx) and torch.equal(again[2], gw), "the same order of sums every time"


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D", [(1, 8), (11, 2224), (300, 520), (700, 4096), (5, 8200), (3, 16384)])
def test_backward_from_both_terms(cuda, hip_lib, rows, D, stream):
    """With delta the sum is taken again: the gradients of the norm of the unrounded sum, dw to fp32's accuracy with a bfloat16 stream too."""
    from aether_amd import functional, ops
    x, delta, w, dy, dres = _inputs(rows, D, stream, seed=5, cuda=cuda)
    h, wd = (x.double() + delta.double()).requires_grad_(True), w.double().requires_grad_(True)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * wd
    dx, dw = torch.autograd.grad((y * dy.double()).sum() + (h * dres.double()).sum(), (h, wd))
    gx, gd, gw = ops.rms_norm_backward(dy, x, w, dres=dres, need_ddelta=True, delta=delta)
    with torch.no_grad():
        r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6)
        n = (dy.double() * wd).abs()
        hm = (x.double().abs() + delta.double().abs()) * 2.0 ** -24 * r              # the sum's own rounding in fp32
        terms = r * (n + (h * r).abs() * (n * (h * r).abs()).mean(-1, keepdim=True)) + dres.double().abs()
        moved = r * (hm * (n * (h * r).abs()).mean(-1, keepdim=True) + (h * r).abs() * (n * hm).mean(-1, keepdim=True))
        wterms = (dy.double() * h * r).abs().sum(0)
        wmoved = (dy.double().abs() * hm).sum(0)
    assert bool(((gx.double() - dx).abs() <= F32 * terms + 2 * moved + (BF16 if stream == torch.bfloat16 else 0.0) * dx.abs()).all())
    assert torch.equal(gd, gx.to(torch.bfloat16))
    assert bool(((gw.double() - dw).abs() <= (F32 + (rows / 512 + 64) * 2.0 ** -24) * wterms + 2 * wmoved).all())
    leaves = [t.clone().requires_grad_(True) for t in (x, delta, w)]
    got = torch.autograd.grad(functional.rms_norm(leaves[0], leaves[2], delta=leaves[1]), leaves, [dy, dres])
    if stream == torch.bfloat16:
        assert all(torch.equal(a, b) for a, b in zip(got, (gx, gd, gw)))
    with pytest.raises(ValueError):
        ops.rms_norm_backward(dy, x, w, delta=delta[:, :-1])


def test_backward_against_differences(cuda, hip_lib):
    """(f(h + e d) − f(h − e d)) / 2e of the float64 formula along random directions equals the kernel's gradient · d."""
    from aether_amd import ops
    x, _, w, dy, _ = _inputs(6, 64, torch.float32, seed=3, cuda=cuda)
    gx, _, gw = ops.rms_norm_backward(dy, x, w)
    f = lambda h, w: (_exact(h, None, w)[1] * dy.double()).sum()  # noqa: E731
    g = torch.Generator().manual_seed(4)
    for _ in range(4):
        d, dwd = torch.randn(6, 64, generator=g).double().to(cuda), torch.randn(64, generator=g).double().to(cuda)
        e = 1e-5
        num = (f(x.double() + e * d, w.double()) - f(x.double() - e * d, w.double())) / (2 * e)
        assert abs((gx.double() * d).sum() - num) <= 1e-5 * (gx.double() * d).abs().sum() + 1e-8
        num = (f(x.double(), w.double() + e * dwd) - f(x.double(), w.double() - e * dwd)) / (2 * e)
        assert abs((gw.double() * dwd).sum() - num) <= 1e-5 * (gw.double() * dwd).abs().sum() + 1e-8


def test_layouts(cuda, hip_lib):
    """Leading shapes, strided rows, transposed and misaligned inputs, no rows; what lies around a view stays as it was."""
    from aether_amd import ops
    x, delta, w, dy, dres = _inputs(24, 64, torch.float32, seed=5, cuda=cuda)
    y0, r0 = ops.rms_norm(x, w, delta=delta)
    y, r = ops.rms_norm(x.view(2, 3, 4, 64), w, delta=delta.view(2, 3, 4, 64))
    assert y.shape == (2, 3, 4, 64) and torch.equal(y.view(24, 64), y0) and torch.equal(r.view(24, 64), r0)
    wide = torch.full((24, 96), 7.0, device=cuda)
    wide[:, 16:80] = x
    keep = wide.clone()
    y, r = ops.rms_norm(wide[:, 16:80], w, delta=delta)
    assert torch.equal(y, y0) and torch.equal(r, r0) and torch.equal(wide, keep)
    y, r = ops.rms_norm(x.t().contiguous().t(), w, delta=delta.t().contiguous().t())
    assert torch.equal(y, y0) and torch.equal(r, r0)
    off = torch.empty(24 * 64 + 1, device=cuda)[1:].view(24, 64).copy_(x)
    w_off = torch.empty(65, device=cuda)[1:].copy_(w)
    y, r = ops.rms_norm(off, w_off, delta=delta)
    assert torch.equal(y, y0) and torch.equal(r, r0)
    y, r = ops.rms_norm(x[:1].expand(24, 64), w)
    assert torch.equal(y[5], ops.rms_norm(x[:1], w)[0][0])
    y, r = ops.rms_norm(x[:0], w, delta=delta[:0])
    assert y.shape == (0, 64) and r.shape == (0, 64)
    q, s, r = ops.rms_norm_e4m3(x[:0], w)
    assert q.shape == (0, 64) and s.shape == (0,)
    gx, gd, gw = ops.rms_norm_backward(dy[:0], x[:0], w, need_ddelta=True)
    assert gx.shape == (0, 64) and torch.equal(gw, torch.zeros_like(w))
    b0 = ops.rms_norm_backward(dy, x, w, dres=dres, need_ddelta=True)
    wide[:, 16:80] = x
    b1 = ops.rms_norm_backward(dy.t().contiguous().t(), wide[:, 16:80], w_off, dres=dres.view(4, 6, 64).reshape(24, 64), need_ddelta=True)
    assert all(torch.equal(p, q) for p, q in zip(b0, b1))


def test_in_place_entry(cuda, hip_lib):
    """The C entry may write the sum over the stream it reads."""
    from aether_amd import _lib, ops
    x, delta, w, _, _ = _inputs(300, 1032, torch.float32, seed=6, cuda=cuda)
    y0, r0 = ops.rms_norm(x, w, delta=delta)
    y = torch.empty_like(y0)
    _lib.check(hip_lib.aether_rms_norm(x.data_ptr(), 1, 1032, delta.data_ptr(), 1032, x.data_ptr(), 1032, w.data_ptr(), 1e-6, y.data_ptr(), 1032, None, 300, 1032,
                                       _lib.current_stream()))
    assert torch.equal(x, r0) and torch.equal(y, y0)


def test_refusals(cuda, hip_lib):
    from aether_amd import ops
    x, w = torch.zeros(4, 64, device=cuda), torch.ones(64, device=cuda)
    for bad in (lambda: ops.rms_norm(x.half(), w), lambda: ops.rms_norm(x, w.half()), lambda: ops.rms_norm(x, w[:32]),
                lambda: ops.rms_norm(x, w, delta=x), lambda: ops.rms_norm(x, w, delta=x[:3].bfloat16()), lambda: ops.rms_norm(x[:, :60], w[:60]),
                lambda: ops.rms_norm(torch.zeros(1, 16392, device=cuda), torch.ones(16392, device=cuda)),
                lambda: ops.rms_norm_backward(x, x, w), lambda: ops.rms_norm_backward(x.bfloat16(), x, w, dres=x.bfloat16()),
                lambda: ops.quantize_rows_e4m3(x), lambda: ops.quantize_rows_e4m3(x.bfloat16()[:, :60])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.rms_norm(x, w.cpu())


def test_stream_and_graph(cuda, hip_lib):
    """On another stream than the default one, and captured: replays on new values equal the eager call."""
    from aether_amd import ops
    x, delta, w, dy, dres = _inputs(37, 1040, torch.float32, seed=7, cuda=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            y, r = ops.rms_norm(x, w, delta=delta)
            b = ops.rms_norm_backward(dy, r, w, dres=dres, need_ddelta=True)
    torch.cuda.current_stream().wait_stream(side)
    want = (*ops.rms_norm(x, w, delta=delta), *ops.rms_norm_backward(dy, r, w, dres=dres, need_ddelta=True))
    assert all(torch.equal(p, q) for p, q in zip((y, r, *b), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, r = ops.rms_norm(x, w, delta=delta)
        b = ops.rms_norm_backward(dy, r, w, dres=dres, need_ddelta=True)
    for k in range(3):
        x.mul_(0.5).add_(k)
        graph.replay()
        y1, r1 = ops.rms_norm(x, w, delta=delta)
        want = (y1, r1, *ops.rms_norm_backward(dy, r1, w, dres=dres, need_ddelta=True))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip((y, r, *b), want))


@pytest.mark.parametrize("rows", [2 ** 24 - 1, 2 ** 24 + 3])
def test_quantize_many_rows(cuda, hip_lib, rows):
    """More rows than a launch of one workgroup each can hold."""
    from aether_amd import ops
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn(rows, 8, generator=g, device=cuda, dtype=torch.bfloat16)
    q, s = ops.quantize_rows_e4m3(x)
    assert torch.equal(s, torch.exp2(torch.ceil(torch.log2(x.float().abs().amax(-1).double() / 448))).float())
    assert torch.equal(q.float(), (x.float() / s[:, None]).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
def test_gradients_do_not_share_memory(cuda, hip_lib, stream):
    """dx and ddelta are tensors of their own: scaling one in place leaves the other as it was."""
    from aether_amd import functional, ops
    x, delta, w, dy, dres = _inputs(19, 520, stream, seed=8, cuda=cuda)
    dx, ddelta, _ = ops.rms_norm_backward(dy, x, w, dres=dres, need_ddelta=True, delta=delta)
    keep = ddelta.clone()
    dx.mul_(0.5)
    assert torch.equal(ddelta, keep)
    leaves = [t.clone().requires_grad_(True) for t in (x, delta)]
    y, h = functional.rms_norm(leaves[0], w, delta=leaves[1])
    a, b = torch.autograd.grad([y, h], leaves, [dy, dres])
    a.mul_(0.5)
    assert torch.equal(b, keep)
    # only the sum is used
    y, h = functional.rms_norm(leaves[0], w, delta=leaves[1])
    keep = dres.bfloat16().clone()
    a, b = torch.autograd.grad(h, leaves, dres)
    assert torch.equal(a, dres) and torch.equal(b, keep)
    a.mul_(0.5)
    assert torch.equal(b, keep)
