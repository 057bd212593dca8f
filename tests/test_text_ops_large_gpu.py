"""The text encoder's operators at the largest lengths and with offsets beyond 32 bits, against float64 (rows and keys that are picked out)."""
import math

import pytest
import torch

from relbias_reference import bucket

pytestmark = pytest.mark.gpu
BF16, S32 = 2.0 ** -8, 2.0 ** -10


def test_attention_at_its_longest(cuda, hip_lib):
    """S = 65536.  Bounds as in test_relbias_attn_gpu.py and test_relbias_attn_backward_gpu.py: o of every row, dq, dk and dv of some."""
    from aether_amd import ops
    S = 65536
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(1, S, 3, 1, 64, generator=g)
    qkv[:, :, :2] *= math.sqrt(0.5)
    qkv = qkv.to(torch.bfloat16).to(cuda)
    table = (torch.randn(32, 1, generator=g) * 2).to(torch.bfloat16).to(cuda)
    do = torch.randn(1, S, 1, 64, generator=g).to(torch.bfloat16).to(cuda)
    mask = torch.ones(1, S, dtype=torch.bool, device=cuda)
    mask[0, 30000:41000] = False
    mask[0, -3:] = False
    q, k, v = qkv.unbind(2)
    o, lse = ops.relbias_attn(q, k, v, table, key_mask=mask, need_lse=True)
    dq, dk, dv, dtable = ops.relbias_attn_backward(do, q, k, v, o, lse, table, key_mask=mask)
    assert not dk[0, 30000:41000].any() and not dv[0, 30000:41000].any()

    qd, kd, vd, gd = (t[0, :, 0].double() for t in (q, k, v, do))
    of = torch.tensor([bucket(d, 32, 128) for d in range(-200, 201)], device=cuda)
    td = table[:, 0].double()
    at = torch.arange(S, device=cuda)
    rows = torch.tensor([0, 1, 63, 64, 8191, 29999, 30000, 40999, 65532, 65535], device=cuda)
    keys = torch.tensor([0, 1, 127, 128, 16384, 29999, 41000, 65472, 65532], device=cuda)
    want = {n: torch.zeros(len(keys), 64, dtype=torch.float64, device=cuda) for n in ("dk", "dv", "lk", "lv")}
    for at0 in range(0, S, 1024):
        i = at[at0:at0 + 1024]
        s = (qd[i] @ kd.t().contiguous()) + td[of[(at[None, :] - i[:, None]).clamp(-200, 200) + 200]]
        s.masked_fill_(~mask, -math.inf)
        p = torch.softmax(s, -1)
        T = p @ vd.abs()
        oo = p @ vd
        err = (o[0, i, 0].double() - oo).abs()
        assert bool((err <= (BF16 + S32) * T + BF16 * oo.abs()).all()), at0
        delta = (gd[i] * oo).sum(-1, keepdim=True)
        D = (gd[i].abs() * (2.0 ** -16 + S32) * T).sum(-1, keepdim=True)

        def ds_of(p, j):
            dP, dPa = gd[i] @ vd[j].t().contiguous(), gd[i].abs() @ vd[j].abs().t().contiguous()
            ds = p * (dP - delta)
            return ds, p * (S32 * (dP.abs() + delta.abs()) + D + 66 * 2.0 ** -24 * dPa) + BF16 * ds.abs()

        pj = p[:, keys]
        ds, E = ds_of(pj, keys)
        want["dk"] += ds.t().contiguous() @ qd[i]
        want["lk"] += E.t().contiguous() @ qd[i].abs()
        want["dv"] += pj.t().contiguous() @ gd[i]
        want["lv"] += (BF16 + S32) * (pj.t().contiguous() @ gd[i].abs())
        for r in rows[(rows >= at0) & (rows < at0 + 1024)].tolist():
            ds, E = ds_of(p, at)
            x, lim = ds[r - at0] @ kd, E[r - at0] @ kd.abs()
            assert bool(((dq[0, r, 0].double() - x).abs() <= lim + BF16 * x.abs()).all()), r
    for n, got in (("k", dk), ("v", dv)):
        x = want["d" + n]
        assert bool(((got[0, keys, 0].double() - x).abs() <= want["l" + n] + BF16 * x.abs()).all()), n
    assert bool(torch.isfinite(dtable.float()).all())


def test_batch_items_far_apart(cuda, hip_lib):
    """The second item begins more than 4 GiB behind the first: the same bits as from packed operands."""
    from aether_amd import ops
    S, H, far = 130, 2, (2 ** 32 + 4096) // 2 + 8 * 1000
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(2, S, 3, H, 64, generator=g).to(torch.bfloat16).to(cuda)
    table = torch.randn(32, H, generator=g).to(torch.bfloat16).to(cuda)
    store = torch.empty(far + S * 3 * H * 64, dtype=torch.bfloat16, device=cuda)
    wide = store.as_strided(qkv.shape, (far, *qkv.stride()[1:]))
    wide.copy_(qkv)
    do = torch.randn(2, S, H, 64, generator=g).to(torch.bfloat16).to(cuda)
    out = []
    for t in (qkv, wide):
        q, k, v = t.unbind(2)
        o, lse = ops.relbias_attn(q, k, v, table, need_lse=True)
        out.append([o, *ops.relbias_attn_backward(do, q, k, v, o, lse, table)])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_rows_far_apart(cuda, hip_lib):
    """Rows of one tensor over more than 4 GiB: the norm and its gradients, and the feed-forward, which goes through them in several launches."""
    from aether_amd import ops
    g = torch.Generator().manual_seed(3)
    M, D, F = 600, 128, 96
    step = 4 * 2 ** 20                                       # 8 MiB between rows: 600 rows over 4.7 GiB
    x = torch.randn(M, D, generator=g).to(torch.bfloat16).to(cuda)
    wide = torch.empty(M * step, dtype=torch.bfloat16, device=cuda).as_strided((M, D), (step, 1))
    wide.copy_(x)
    w = torch.randn(D, generator=g).to(cuda)
    assert all(torch.equal(a, b) for a, b in zip(ops.rms_norm(wide, w, delta=x), ops.rms_norm(x, w, delta=x)))
    dy = torch.randn(M, D, generator=g).to(torch.bfloat16).to(cuda)
    assert all(torch.equal(a, b) for a, b in zip(ops.rms_norm_backward(dy, wide, w, need_ddelta=True), ops.rms_norm_backward(dy, x, w, need_ddelta=True)))
    wg, wu = (torch.randn(F, D, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
    h, gu = ops.gated_ff(wide, wg, wu, need_gu=True)
    parts = [ops.gated_ff(x[m:m + 256], wg, wu, need_gu=True) for m in range(0, M, 256)]
    want = torch.cat([p[0] for p in parts])
    # a launch of other sizes may take another tile, and K in another order: fp32 sums of 128 products on both sides (|act'| < 1.2), one rounding to bf16 each
    A = [(x.float().abs() @ t.float().abs().t().contiguous()) for t in (wg, wu)]
    lim = 2 * BF16 * want.float().abs() + 2 * 128 * 2.0 ** -24 * (1.2 * A[0] * gu[:, F:].abs() + A[1] * gu[:, :F].abs())
    assert bool(((h.float() - want.float()).abs() <= lim).all())
    assert all(torch.equal(a, b) for a, b in zip(ops.gated_ff_backward(h, wide, wg, wu, gu), ops.gated_ff_backward(h, x, wg, wu, gu)))


def test_the_most_batch_items_of_a_launch(cuda, hip_lib):
    """2^26 - 64 heads of one token each: every one gets its only value.  One batch item more is refused."""
    from aether_amd import ops
    B, H = 2 ** 20 - 1, 64
    g = torch.Generator(device=cuda).manual_seed(5)
    v = torch.randn(B + 1, 1, H, 64, generator=g, device=cuda, dtype=torch.bfloat16)
    one = torch.ones(1, 1, 1, 64, dtype=torch.bfloat16, device=cuda).expand(B + 1, 1, H, 64)
    table = torch.zeros(32, H, dtype=torch.bfloat16, device=cuda)
    assert torch.equal(ops.relbias_attn(one[:B], one[:B], v[:B], table), v[:B])
    with pytest.raises(ValueError, match="blocks"):
        ops.relbias_attn(one, one, v, table)


def _check_ff_gradients(dh, x, wg, wu, gu, got, rows, cols):
    """dx of some rows and the weights' gradients of some columns, bounds as in test_gated_ff_gpu.py; g and u are the stored projections."""
    M, F = dh.shape
    dx, dwg, dwu = got
    cat = torch.cat([wg, wu]).double()
    F64 = torch.float64
    sum_g, sum_u, lim_g, lim_u = (torch.zeros(F, len(cols), dtype=F64, device=x.device) for _ in range(4))
    for m in range(0, M, 1 << 18):
        g = gu[m:m + (1 << 18), :F].double().requires_grad_(True)
        u, d = gu[m:m + (1 << 18), F:].double(), dh[m:m + (1 << 18)].double()
        a = torch.nn.functional.gelu(g, approximate="tanh")
        dg = torch.autograd.grad((a * u * d).sum(), g)[0]
        du, xc = (d * a).detach(), x[m:m + (1 << 18)][:, cols].double()
        eg, eu = (2.0 ** -14 * (d * u).abs() + BF16 * dg.abs()), 2.0 ** -14 * (d * g.detach()).abs() + BF16 * du.abs()
        t = lambda z: z.t().contiguous()  # noqa: E731
        sum_g += t(dg) @ xc
        sum_u += t(du) @ xc
        lim_g += t(eg + M * 2.0 ** -24 * dg.abs()) @ xc.abs()
        lim_u += t(eu + M * 2.0 ** -24 * du.abs()) @ xc.abs()
        here = [r for r in rows if m <= r < m + (1 << 18)]
        if here and dx is not None:
            i = torch.tensor(here, device=x.device) - m
            both, e = torch.cat([dg[i], du[i]], 1), torch.cat([eg[i], eu[i]], 1)
            want = both @ cat
            assert bool(((dx[i + m].double() - want).abs() <= (e + 2 * F * 2.0 ** -24 * both.abs()) @ cat.abs() + BF16 * want.abs()).all())
    for grad, want, lim in ((dwg, sum_g, lim_g), (dwu, sum_u, lim_u)):
        assert bool(((grad[:, cols].double() - want).abs() <= lim + BF16 * want.abs()).all())


@pytest.mark.parametrize("M,K,F", [(131072 + 40, 16384, 256), (4200001, 64, 32)])
def test_feed_forward_gradients_of_many_rows(cuda, hip_lib, M, K, F):
    """x of more than 4 GiB, whose turned copy is an operand of the weights' gradients; and more than 65535 blocks of 64 rows."""
    from aether_amd import ops
    g = torch.Generator(device=cuda).manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda, dtype=torch.bfloat16)  # noqa: E731
    x, wg, wu, dh = r(M, K), r(F, K) * K ** -0.5, r(F, K) * K ** -0.5, r(M, F)
    _, gu = ops.gated_ff(x, wg, wu, need_gu=True)
    got = ops.gated_ff_backward(dh, x, wg, wu, gu)
    assert all(bool(torch.isfinite(t).all()) for t in got)
    cols = torch.tensor([0, 1, 31, K // 2, K - 65 if K > 64 else 40, K - 64, K - 1], device=cuda)
    _check_ff_gradients(dh, x, wg, wu, gu, got, [0, 63, 64, 65536, 131071, M - 65, M - 64, M - 1], cols)
    frozen = ops.gated_ff_backward(dh, x, wg, wu, gu, need_dw=False)
    assert torch.equal(frozen[0], got[0]) and frozen[1] is None


def test_largest_tables_at_the_longest(cuda, hip_lib):
    """S = 65536 with a mask and a bias that reaches 1020 positions: ring, table and mask words together are more than 64 KiB of LDS.  Rows that are picked out,
    bound as in test_relbias_attn_gpu.py."""
    from aether_amd import ops
    S, nb, far = 65536, 128, 1140
    assert ops.relbias_borders(nb, far)[-1] == 1020
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(1, S, 3, 1, 64, generator=g)
    qkv[:, :, :2] *= math.sqrt(0.5)
    q, k, v = qkv.to(torch.bfloat16).to(cuda).unbind(2)
    table = (torch.randn(nb, 1, generator=g) * 2).to(torch.bfloat16).to(cuda)
    mask = torch.ones(1, S, dtype=torch.bool, device=cuda)
    mask[0, 20000:50000], mask[0, -70:] = False, False
    of = torch.tensor([bucket(d, nb, far) for d in range(-1100, 1101)], device=cuda)
    at = torch.arange(S, device=cuda)
    i = torch.tensor([0, 1, 1000, 19990, 20000, 35000, 49999, 51000, 65400, S - 1], device=cuda)
    s = q[0, i, 0].double() @ k[0, :, 0].double().t().contiguous() + table[:, 0].double()[of[(at[None, :] - i[:, None]).clamp(-1100, 1100) + 1100]]
    p = torch.softmax(s.masked_fill(~mask, -math.inf), -1)
    want, T = p @ v[0, :, 0].double(), p @ v[0, :, 0].double().abs()
    plain = ops.relbias_attn(q, k, v, table, far, key_mask=mask)
    train, lse = ops.relbias_attn(q, k, v, table, far, key_mask=mask, need_lse=True)
    for o in (plain, train):
        assert bool(((o[0, i, 0].double() - want).abs() <= (BF16 + S32) * T + BF16 * want.abs()).all())
    got = ops.relbias_attn_backward(o, q, k, v, train, lse, table, far, key_mask=mask)
    assert all(bool(torch.isfinite(t.float()).all()) for t in got) and not got[1][0, 20000:50000].any()


def test_table_gradient_at_the_longest(cuda, hip_lib):
    """S = 65536, masked tiles in between: the table's gradient.  Near buckets, entry by entry: dS is off by E of test_relbias_attn_backward_gpu.py without its rounding
    (near dS are summed in fp32), the entry by 2^-8.  Of the far ones, two sums over half a million keys each whose terms nearly cancel, the sum of all E says nothing:
    their errors are independent from row to row, and what remains is the rounding of the result, 2^-9 in the norm as in test_far_buckets_of_long_rows."""
    from aether_amd import ops
    S, near = 65536, 91
    g = torch.Generator().manual_seed(12)
    qkv = torch.randn(1, S, 3, 1, 64, generator=g)
    qkv[:, :, :2] *= math.sqrt(0.5)
    q, k, v = qkv.to(torch.bfloat16).to(cuda).unbind(2)
    table = (torch.randn(32, 1, generator=g) * 2).to(torch.bfloat16).to(cuda)
    do = torch.randn(1, S, 1, 64, generator=g).to(torch.bfloat16).to(cuda)
    mask = torch.ones(1, S, dtype=torch.bool, device=cuda)
    mask[0, 30000:41000], mask[0, 50010:50100], mask[0, -3:] = False, False, False
    o, lse = ops.relbias_attn(q, k, v, table, key_mask=mask, need_lse=True)
    got = ops.relbias_attn_backward(do, q, k, v, o, lse, table, key_mask=mask)[3][:, 0].double()

    qd, kd, vd, gd = (t[0, :, 0].double() for t in (q, k, v, do))
    kt, vt, va = kd.t().contiguous(), vd.t().contiguous(), vd.abs()
    of = torch.tensor([bucket(d, 32, 128) for d in range(-200, 201)], device=cuda)
    td, at = table[:, 0].double(), torch.arange(S, device=cuda)
    assert int(of[200 - near]) == 15 and int(of[200 + near]) == 31 and int(of[200 - near + 1]) == 14 and int(of[200 + near - 1]) == 30
    want, lim = torch.zeros(32, dtype=torch.float64, device=cuda), torch.zeros(32, dtype=torch.float64, device=cuda)
    band = torch.arange(1 - near, near, device=cuda)
    for at0 in range(0, S, 1024):
        i = at[at0:at0 + 1024]
        d = at[None, :] - i[:, None]
        s = (qd[i] @ kt) + td[of[d.clamp(-200, 200) + 200]]
        p = torch.softmax(s.masked_fill_(~mask, -math.inf), -1)
        dP = gd[i] @ vt
        delta = (p * dP).sum(-1, keepdim=True)
        ds = p * (dP - delta)
        want[15] += (ds * (d <= -near)).sum()
        want[31] += (ds * (d >= near)).sum()
        j = i[:, None] + band[None, :]
        ok, jc = (j >= 0) & (j < S), j.clamp(0, S - 1)
        D = (gd[i].abs() * (2.0 ** -16 + S32) * (p @ va)).sum(-1, keepdim=True)
        pick = lambda t: torch.gather(t, 1, jc) * ok  # noqa: E731
        pj, dj = pick(p), pick(dP)
        dPa = (gd[i].abs()[:, None, :] * va[jc]).sum(-1)
        E = pj * (S32 * (dj.abs() + delta.abs()) + D + 66 * 2.0 ** -24 * dPa)
        b = of[band + 200].expand(len(i), -1).reshape(-1)
        want.index_add_(0, b, pick(ds).reshape(-1))
        lim.index_add_(0, b, E.reshape(-1))
    few = torch.ones(32, dtype=torch.bool, device=cuda)
    few[15] = few[31] = False
    few[16] = False                                           # no pair has it: distance 0 is of the other side
    err = (got - want).abs()
    print("near", err[few].max().item(), lim[few].min().item(), want[few].abs().median().item(), "far", err[~few].tolist(), want[~few].tolist())
    assert bool((err[few] <= lim[few] + BF16 * want[few].abs()).all()) and got[16] == 0
    assert bool((lim[few] < 0.5 * want[few].abs().max()).all()), "a gradient of zeros does not pass"
    assert (got - want).norm() <= 2.0 ** -9 * want.norm()
