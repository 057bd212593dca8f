"""relbias_attn_backward against float64 autograd of the definition, and against differences of it.

Tolerances (elementwise; all sums over the float64 tensors of the reference).  P carries 2^-10 from the scores (see test_relbias_attn_gpu.py) and is
rounded to bf16 as an operand: dv is off by (2^-8 + 2^-10) Σ P |dO| + 2^-8 |dv|.  δ_i is taken from O in two parts, off by (2^-16 + 2^-10) T
together, so δ by D_i = Σ_d |dO| of that; dP is a sum of 64 products in fp32 (66 · 2^-24 of its magnitudes).  dS = P (dP − δ) is off by
E = P (2^-10 (|dP| + |δ|) + D + 66 · 2^-24 Σ|dO||v|) + 2^-8 |dS| with its own rounding to bf16; dq, dk and dtable by E summed over what they are summed
of, and 2^-8 of themselves."""
import math

import pytest
import torch

from relbias_reference import attention, bucket, inputs
from test_relbias_attn_gpu import LENGTHS, _masks

pytestmark = pytest.mark.gpu
BF16, S32 = 2.0 ** -8, 2.0 ** -10


def _run(q, k, v, table, do, **kw):
    from aether_amd import ops
    o, lse = ops.relbias_attn(q, k, v, table, need_lse=True, **kw)
    return ops.relbias_attn_backward(do, q, k, v, o, lse, table, **kw)


def _check(got, q, k, v, table, do, scale=1.0, S32=S32, **kw):
    leaf = [t.double().requires_grad_(True) for t in (q, k, v, table)]
    o, p = attention(*leaf, scale=scale, **kw)
    want = torch.autograd.grad((o * do.double()).sum(), leaf)
    mask, S = kw.get("key_mask"), q.shape[1]
    with torch.no_grad():
        zero = torch.zeros((), dtype=torch.float64, device=q.device)
        keep = (lambda t: t) if mask is None else (lambda t: torch.where(mask[:, :, None, None], t, zero))  # noqa: E731
        heads = lambda t: t.permute(0, 2, 1, 3).contiguous()  # noqa: E731
        g, va, ka, qa = heads(do.double()), heads(keep(leaf[2].abs())), heads(keep(leaf[1].abs())), heads(leaf[0].abs())
        vv = heads(keep(leaf[2]))
        T = torch.matmul(p, va)
        D = (g.abs() * (2.0 ** -16 + S32) * T).sum(-1, keepdim=True)
        dP, dPa = torch.matmul(g, vv.transpose(2, 3).contiguous()), torch.matmul(g.abs(), va.transpose(2, 3).contiguous())
        delta = (g * heads(o)).sum(-1, keepdim=True)
        E = p * (S32 * (dP.abs() + delta.abs()) + D + 66 * 2.0 ** -24 * dPa) + BF16 * (p * (dP - delta)).abs()
        back = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
        Et = E.transpose(2, 3).contiguous()
        lim = [abs(scale) * back(torch.matmul(E, ka)), abs(scale) * back(torch.matmul(Et, qa)),
               (BF16 + S32) * back(torch.matmul(p.transpose(2, 3).contiguous(), g.abs()))]
        bk = torch.tensor([bucket(d, table.shape[0], kw.get("max_distance", 128)) for d in range(1 - S, S)], device=q.device)
        at = torch.arange(S, device=q.device)
        lim.append(torch.zeros_like(want[3]).index_add_(0, bk[at[None, :] - at[:, None] + S - 1].reshape(-1), E.sum(0).permute(1, 2, 0).reshape(S * S, -1)))
        for n, x, y, l in zip(("dq", "dk", "dv", "dtable"), got, want, lim):
            assert x.shape == y.shape and x.dtype == torch.bfloat16
            err = (x.double() - y).abs()
            excess = err - l - BF16 * y.abs()
            assert bool(torch.isfinite(x.float()).all()) and bool((excess <= 1e-30).all()), f"{n}: worst excess {excess.max().item():.3e}, rel {(err.norm() / y.norm()).item():.3e}"
            print(n, (err.norm() / y.norm()).item())


def _do(q, seed=0):
    return torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(q.device)


@pytest.mark.parametrize("S", LENGTHS)
@pytest.mark.parametrize("B,H", [(1, 1), (2, 3)])
def test_lengths(cuda, hip_lib, S, B, H):
    qkv, table = inputs(B, S, H, device=cuda, seed=20)
    q, k, v = qkv.unbind(2)
    do = _do(q)
    got = _run(q, k, v, table, do)
    _check(got, q, k, v, table, do)
    again = _run(q, k, v, table, do)
    assert all(torch.equal(x, y) for x, y in zip(got, again)), "the same order of sums every time"
    if S == 1:      # one key: P is 1 whatever the scores
        assert not any(x.float().abs().max() for x in (got[0], got[1], got[3])) and torch.equal(got[2], do)


@pytest.mark.parametrize("B,S,H", [(1, 226, 64), (6, 226, 64), (8, 64, 64), (1, 1290, 16), (40, 33, 8), (300, 5, 2)])
def test_many_blocks(cuda, hip_lib, B, S, H):
    qkv, table = inputs(B, S, H, device=cuda, seed=21)
    q, k, v = qkv.unbind(2)
    do = _do(q)
    _check(_run(q, k, v, table, do), q, k, v, table, do)


@pytest.mark.parametrize("num_buckets,max_distance", [(4, 2), (4, 100), (6, 3), (8, 20), (10, 9), (32, 32), (64, 256), (128, 1000), (12, 1024)])
@pytest.mark.parametrize("S", [65, 700])
def test_buckets(cuda, hip_lib, num_buckets, max_distance, S):
    qkv, table = inputs(1, S, 2, num_buckets, device=cuda, seed=22)
    q, k, v = qkv.unbind(2)
    do = _do(q)
    _check(_run(q, k, v, table, do, max_distance=max_distance), q, k, v, table, do, max_distance=max_distance)


def test_largest_tables(cuda, hip_lib):
    """The farthest reach, long sequences with a mask and every workgroup size: the most LDS a call can need."""
    from aether_amd import ops
    for B, S, H in ((1, 30, 1), (1, 60, 1), (2, 300, 64)):
        qkv, table = inputs(B, S, H, 32, device=cuda, seed=23)
        q, k, v = qkv.unbind(2)
        do, mask = _do(q), torch.ones(B, S, dtype=torch.bool, device=cuda)
        table = inputs(1, 1, H, 4 + 8, device=cuda)[1]
        _check(_run(q, k, v, table, do, max_distance=2000, key_mask=mask), q, k, v, table, do, max_distance=2000, key_mask=mask)
    assert ops.relbias_borders(12, 2000)[1] > 200


@pytest.mark.parametrize("kind", ["right", "left", "holes", "one", "none", "blocks"])
@pytest.mark.parametrize("S", [1, 33, 64, 226, 515])
def test_masks(cuda, hip_lib, kind, S):
    B, H = 3, 2
    qkv, table = inputs(B, S, H, device=cuda, seed=24)
    mask = _masks(B, S, cuda)[kind]
    q, k, v = qkv.unbind(2)
    do = _do(q)
    got = _run(q, k, v, table, do, key_mask=mask)
    _check(got, q, k, v, table, do, key_mask=mask)
    assert bool((got[1][~mask] == 0).all()) and bool((got[2][~mask] == 0).all()) and bool((got[0][~mask.any(1)] == 0).all())
    if kind == "one":
        assert not any(x.float().abs().max() for x in (got[0], got[1], got[3]))
    bad = qkv.clone()
    for i, val in enumerate((math.nan, math.inf, -math.inf, 3e38)):
        at = ~mask & ((torch.arange(S, device=cuda) % 4) == i)[None, :]
        bad[:, :, 1:][at] = val
    again = _run(q, bad[:, :, 1], bad[:, :, 2], table, do, key_mask=mask)
    assert all(torch.equal(x, y) for x, y in zip(got, again)), "what stands behind the mask reaches nothing"


@pytest.mark.parametrize("kind", ["right", "left", "holes", "blocks"])
def test_masks_long(cuda, hip_lib, kind):
    B, S, H = 2, 1030, 2
    qkv, table = inputs(B, S, H, device=cuda, seed=34)
    mask = _masks(B, S, cuda)[kind]
    q, k, v = qkv.unbind(2)
    do = _do(q)
    got = _run(q, k, v, table, do, key_mask=mask)
    _check(got, q, k, v, table, do, key_mask=mask)
    bad = qkv.clone()
    bad[:, :, 1:][~mask] = math.nan
    assert all(torch.equal(x, y) for x, y in zip(got, _run(q, bad[:, :, 1], bad[:, :, 2], table, do, key_mask=mask)))


@pytest.mark.parametrize("scale", [0.0, -0.1, 0.02])
@pytest.mark.parametrize("S", [70, 500])
def test_scales(cuda, hip_lib, scale, S):
    qkv, table = inputs(2, S, 2, device=cuda, seed=35, qk=4.0)
    q, k, v = qkv.unbind(2)
    do = _do(q)
    got = _run(q, k, v, table, do, scale=scale)
    _check(got, q, k, v, table, do, scale=scale)
    if scale == 0:
        assert not got[0].any() and not got[1].any()


@pytest.mark.parametrize("order", ["early", "late", "rising", "far_below"])
@pytest.mark.parametrize("S", [200, 700])
def test_score_ranges(cuda, hip_lib, order, S):
    """Scores of several hundred: they and the log-sum carry 66 · 2^-24 · 800 < 2^-8 each."""
    qkv, table = inputs(1, S, 2, device=cuda, seed=36)
    at = torch.arange(S, device=cuda, dtype=torch.float32)
    level = dict(early=400 * (at < 5), late=400 * (at > S - 9), rising=at * (400 / S), far_below=at * 0 - 400)[order]
    q, k, v = (t.clone() for t in qkv.unbind(2))
    q[..., 0], k[..., 0] = 4.0, (level / 4).to(torch.bfloat16)[None, :, None]
    do = _do(q)
    _check(_run(q, k, v, table, do), q, k, v, table, do, S32=2.0 ** -6)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.bfloat16).min, -1e9])
@pytest.mark.parametrize("S", [70, 500])
@pytest.mark.parametrize("scale", [1.0, 0.1])
def test_one_side_switched_off(cuda, hip_lib, low, S, scale):
    """Buckets at −inf or the type's lowest value: rows see the keys up to their own.  Rows of the padding in front, which see the lowest value alone, have no
    gradient and bring none."""
    qkv, table = inputs(2, S, 2, device=cuda, seed=37)
    table[table.shape[0] // 2:] = low
    q, k, v = qkv.unbind(2)
    do = _do(q)
    got = _run(q, k, v, table, do, scale=scale)
    want = table.clone()
    want[table.shape[0] // 2:] = -2000.0         # exp of it is 0 in float64 too, and its gradient a number
    _check(got, q, k, v, want, do, scale=scale)
    if low != -math.inf:
        mask = torch.ones(2, S, dtype=torch.bool, device=cuda)
        mask[1, :25] = False
        do[1, :25] = 0
        got = _run(q, k, v, table, do, scale=scale, key_mask=mask)
        assert all(bool(torch.isfinite(x.float()).all()) for x in got) and not got[0][1, :25].any()
        part = _run(q[1:, 25:], k[1:, 25:], v[1:, 25:], table, do[1:, 25:], scale=scale)
        for x, y in zip(got[:3], part[:3]):
            assert bool(((x[1, 25:].double() - y[0].double()).norm() <= 4 * BF16 * y.double().norm()))


def test_far_buckets_of_long_rows(cuda, hip_lib):
    """A row's dS add up to 0, so the far buckets' sums are what the near ones are, over ten times as many terms: their relative error (in the norm) is that of
    sums in fp32 and one rounding to bf16 (2^-8 / sqrt(12) · 1.2 in the mean), not of terms rounded before they are summed."""
    qkv, table = inputs(1, 2039, 4, device=cuda, seed=38, qk=0.3)
    q, k, v = qkv.unbind(2)
    do = _do(q)
    got = _run(q, k, v, table, do)[3].double()
    leaf = [t.double().requires_grad_(True) for t in (q, k, v, table)]
    want, = torch.autograd.grad((attention(*leaf)[0] * do.double()).sum(), leaf[3:])
    assert (got - want).norm() <= 2.0 ** -9 * want.norm()


def test_empty_row_with_non_finite_gradient(cuda, hip_lib):
    """A NaN in the gradient of one row reaches that row and the keys it attends to, not the keys that do not count."""
    qkv, table = inputs(2, 100, 2, device=cuda, seed=25)
    q, k, v = qkv.unbind(2)
    mask = torch.arange(100, device=cuda)[None, :] < torch.tensor([[70], [0]], device=cuda)
    do = _do(q)
    do[0, 3, 1, 7] = math.nan
    dq, dk, dv, _ = _run(q, k, v, table, do, key_mask=mask)
    assert bool((dk[~mask] == 0).all()) and bool((dv[~mask] == 0).all()) and bool((dq[1] == 0).all())
    rows = torch.ones(100, 2, dtype=torch.bool, device=cuda)
    rows[3, 1] = False
    assert bool(torch.isfinite(dq[0][rows].float()).all()) and bool(torch.isnan(dq[0, 3, 1].float()).all())
    assert bool(torch.isfinite(dk[0, :, 0].float()).all()) and bool(torch.isfinite(dv[0, :, 0].float()).all())


def test_against_differences(cuda, hip_lib):
    """(f(x + e d) − f(x − e d)) / 2e of the float64 definition along directions in q, k, v and the table; the gradients' own rounding is 2^-8."""
    qkv, table = inputs(2, 40, 2, device=cuda, seed=26)
    q, k, v = qkv.unbind(2)
    mask = _masks(2, 40, cuda)["right"]
    do = _do(q)
    got = _run(q, k, v, table, do, key_mask=mask)
    x = [t.double() for t in (q, k, v, table)]
    f = lambda a: (attention(*a, key_mask=mask)[0] * do.double()).sum()  # noqa: E731
    for i, g in enumerate(got):
        d = g.double().sign()
        up, dn = list(x), list(x)
        up[i], dn[i] = x[i] + 1e-5 * d, x[i] - 1e-5 * d
        num = (f(up) - f(dn)) / 2e-5
        assert abs((g.double() * d).sum() - num) <= 4 * BF16 * g.double().abs().sum()


def test_scale_and_layouts(cuda, hip_lib):
    from aether_amd import ops
    qkv, table = inputs(2, 130, 3, device=cuda, seed=27, qk=4.0)
    q, k, v = qkv.unbind(2)
    do = _do(q)
    _check(_run(q, k, v, table, do, scale=0.125), q, k, v, table, do, scale=0.125)
    base = _run(q, k, v, table, do, scale=0.125)
    assert base[0].data_ptr() + 3 * 64 * 2 == base[1].data_ptr() and base[0].stride() == (130 * 9 * 64, 9 * 64, 64, 1)
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    dh = do.transpose(1, 2).contiguous().transpose(1, 2)
    assert all(torch.equal(x, y) for x, y in zip(base, _run(*heads, table, dh, scale=0.125)))
    wide = torch.full((2, 140, 3, 80), math.nan, dtype=torch.bfloat16, device=cuda)
    wide[:, 5:135, :, 8:72] = do
    assert all(torch.equal(x, y) for x, y in zip(base, _run(q, k, v, table, wide[:, 5:135, :, 8:72], scale=0.125)))
    one = do[:, :1].expand(2, 130, 3, 64)
    assert all(torch.equal(x, y) for x, y in zip(_run(q, k, v, table, one), _run(q, k, v, table, one.contiguous())))
    o, lse = ops.relbias_attn(q, k, v, table, need_lse=True)
    got = ops.relbias_attn_backward(do, q, k, v, o.transpose(2, 3).contiguous().transpose(2, 3), torch.stack([lse, lse], 1)[:, 0], table, need_dtable=False)
    want = ops.relbias_attn_backward(do, q, k, v, o, lse, table)
    assert got[3] is None and all(torch.equal(x, y) for x, y in zip(got[:3], want[:3]))


def test_without_rows(cuda, hip_lib):
    qkv, table = inputs(2, 16, 2, device=cuda)
    for cut in (qkv[:0], qkv[:, :0]):
        q, k, v = cut.unbind(2)
        dq, dk, dv, dt = _run(q, k, v, table, torch.empty_like(q))
        assert dq.shape == dk.shape == dv.shape == q.shape and torch.equal(dt, torch.zeros_like(table))


def test_refusals(cuda, hip_lib):
    from aether_amd import ops
    qkv, table = inputs(2, 16, 2, device=cuda)
    q, k, v = qkv.unbind(2)
    o, lse = ops.relbias_attn(q, k, v, table, need_lse=True)
    for bad in (lambda: ops.relbias_attn_backward(o.float(), q, k, v, o, lse, table), lambda: ops.relbias_attn_backward(o[:1], q, k, v, o, lse, table),
                lambda: ops.relbias_attn_backward(o, q, k, v, o[:, :8], lse, table), lambda: ops.relbias_attn_backward(o, q, k, v, o, lse[:8], table),
                lambda: ops.relbias_attn_backward(o, q, k, v, o, lse.half(), table), lambda: ops.relbias_attn_backward(o, q, k, v, o, lse, table.float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.relbias_attn_backward(o, q, k, v, o, lse.cpu(), table)


def test_graph(cuda, hip_lib):
    """Forward and backward captured together, replayed on new values with eager work in between."""
    qkv, table = inputs(2, 226, 4, device=cuda, seed=28)
    mask = _masks(2, 226, cuda)["right"]
    q, k, v = qkv.unbind(2)
    do = _do(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(q, k, v, table, do, key_mask=mask)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(q, k, v, table, do, key_mask=mask)
    for n in (226, 100, 3):
        qkv.mul_(-0.9)
        mask[1] = torch.arange(226, device=cuda) < n
        graph.replay()
        want = _run(q, k, v, table, do, key_mask=mask)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
