"""relbias_attn against the definition in float64 on the same bf16 inputs.

Tolerance of an output element o = Σ_j p_j v_j, with T = Σ_j p_j |v_j|: every p_j is rounded to bf16 (2^-8 p_j) before its product; a score is a sum
of 64 exact products in fp32, scaled and exponentiated: its absolute error is at most 66 · 2^-24 · (Σ|q k| scale + |bias|) and moves p_j by as much,
numerator and denominator each; the output is rounded once (2^-8 |o|).  Scores of the tests below have Σ|q k| · scale < 60 where nothing else is said:
2 · 66 · 2^-24 · 66 < 2^-10.  Bound: (2^-8 + 2^-10) T + 2^-8 |o|."""
import math

import pytest
import torch

from relbias_reference import attention, bucket, inputs

pytestmark = pytest.mark.gpu
BF16 = 2.0 ** -8


def _check_o(got, q, k, v, table, extra=2.0 ** -10, **kw):
    d = [t.double() for t in (q, k, v, table)]
    want, p = attention(*d, **kw)
    mask = kw.get("key_mask")
    va = d[2].abs() if mask is None else torch.where(mask[:, :, None, None], d[2].abs(), 0.0)
    T = torch.matmul(p, va.permute(0, 2, 1, 3).contiguous()).permute(0, 2, 1, 3)
    err = (got.double() - want).abs()
    lim = (BF16 + extra) * T + BF16 * want.abs()
    assert got.shape == want.shape and got.dtype == torch.bfloat16
    assert bool(torch.isfinite(got.float()).all()) and bool((err <= lim).all()), f"worst {(err - lim).max().item():.3e}, rel {(err.norm() / want.norm()).item():.3e}"
    return want, p


LENGTHS = [1, 2, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 191, 226, 300, 513, 1030]


@pytest.mark.parametrize("S", LENGTHS)
@pytest.mark.parametrize("B,H", [(1, 1), (2, 3)])
def test_lengths(cuda, hip_lib, S, B, H):
    from aether_amd import ops
    qkv, table = inputs(B, S, H, device=cuda)
    q, k, v = qkv.unbind(2)
    _check_o(ops.relbias_attn(q, k, v, table), q, k, v, table)
    o, lse = ops.relbias_attn(q, k, v, table, need_lse=True)
    want, p = _check_o(o, q, k, v, table)
    # with the remainder the output is good to 2^-16 of Σ P |v|, besides what the scores' rounding moves P by
    lse, low = lse[:B * S * H].view(B, H, S), lse[(B * S * H + 3) // 4 * 4:].view(torch.bfloat16).view(B, S, H, 64)
    T = torch.matmul(p, v.double().abs().permute(0, 2, 1, 3).contiguous()).permute(0, 2, 1, 3)
    assert bool(((o.double() + low.double() - want).abs() <= (2.0 ** -16 + 2.0 ** -10) * T).all())
    assert ((o.double() + low.double() - want).norm() <= 2.0 ** -14 * T.norm()), "far below one rounding to bf16"
    # lse is the base-2 logarithm of the rows' sums of exp(score)
    s = torch.matmul(q.double().permute(0, 2, 1, 3).contiguous(), k.double().permute(0, 2, 3, 1).contiguous())
    bias = torch.tensor([[bucket(j - i, 32, 128) for j in range(S)] for i in range(S)], device=cuda)
    s = s + table.double()[bias].permute(2, 0, 1)
    assert bool(((torch.logsumexp(s, -1) / math.log(2) - lse.double()).abs() < 1e-4).all())


@pytest.mark.parametrize("B,S,H", [(1, 226, 64), (16, 226, 64), (8, 64, 64), (1, 2050, 16), (40, 33, 8), (300, 5, 2)])
def test_many_blocks(cuda, hip_lib, B, S, H):
    """Grids beyond one workgroup per CU, every block size."""
    from aether_amd import ops
    qkv, table = inputs(B, S, H, device=cuda, seed=1)
    q, k, v = qkv.unbind(2)
    _check_o(ops.relbias_attn(q, k, v, table), q, k, v, table)


@pytest.mark.parametrize("num_buckets,max_distance", [(4, 2), (4, 100), (6, 3), (8, 20), (10, 9), (32, 32), (32, 128), (64, 256), (128, 1000), (12, 1024)])
@pytest.mark.parametrize("S", [65, 700])
def test_buckets(cuda, hip_lib, num_buckets, max_distance, S):
    """Every way the buckets are laid out: reach 1 ... 930, few and many borders.  A wrong bucket shows: the table's entries are far apart."""
    from aether_amd import ops
    qkv, table = inputs(1, S, 2, num_buckets, device=cuda, seed=2)
    table = torch.randperm(num_buckets * 2, generator=torch.Generator().manual_seed(3)).view(num_buckets, 2).to(torch.bfloat16).to(cuda) / 4
    q, k, v = qkv.unbind(2)
    _check_o(ops.relbias_attn(q, k, v, table, max_distance), q, k, v, table, max_distance=max_distance)


def _masks(B, S, cuda):
    g = torch.Generator().manual_seed(S)
    right = torch.arange(S)[None, :] < torch.tensor([S] + [max(1, (S * (b + 1)) // (B + 1)) for b in range(B - 1)])[:, None]
    left = right.flip(1)
    holes = torch.rand(B, S, generator=g) < 0.5
    holes[:, S // 2] = True
    one = torch.zeros(B, S, dtype=torch.bool)
    one[torch.arange(B), torch.randint(0, S, (B,), generator=g)] = True
    none = right.clone()
    none[-1] = False
    blocks = (torch.arange(S) // 64 % 2 == 1)[None, :].repeat(B, 1) | one
    return {k: m.to(cuda) for k, m in dict(right=right, left=left, holes=holes, one=one, none=none, blocks=blocks).items()}


@pytest.mark.parametrize("kind", ["right", "left", "holes", "one", "none", "blocks"])
@pytest.mark.parametrize("S", [1, 33, 64, 226, 515])
def test_masks(cuda, hip_lib, kind, S):
    """Padding on either side, holes, one key alone, no key, whole tiles left out; NaN and infinities behind the mask reach nothing."""
    from aether_amd import ops
    B, H = 3, 2
    qkv, table = inputs(B, S, H, device=cuda, seed=4)
    mask = _masks(B, S, cuda)[kind]
    q, k, v = qkv.unbind(2)
    o = ops.relbias_attn(q, k, v, table, key_mask=mask)
    _check_o(o, q, k, v, table, key_mask=mask)
    o2, lse = ops.relbias_attn(q, k, v, table, key_mask=mask, need_lse=True)
    _check_o(o2, q, k, v, table, key_mask=mask)
    lse = lse[:B * S * H].view(B, H, S)
    empty = ~mask.any(1)
    assert bool((o[empty] == 0).all()) and bool(torch.isposinf(lse[empty]).all()) and bool(torch.isfinite(lse[~empty]).all())
    bad = qkv.clone()
    for i, val in enumerate((math.nan, math.inf, -math.inf, 3e38)):
        at = ~mask & ((torch.arange(S, device=cuda) % 4) == i)[None, :]
        bad[:, :, 1:][at] = val
    assert torch.equal(ops.relbias_attn(q, bad[:, :, 1], bad[:, :, 2], table, key_mask=mask), o)
    if kind == "right":     # an unpadded call on the shorter prompt gives the same rows
        n = int(mask[1].sum())
        alone = ops.relbias_attn(q[1:2, :n], k[1:2, :n], v[1:2, :n], table)
        assert bool(((alone.float() - o[1:2, :n].float()).abs() <= 2 * BF16 * o[1:2, :n].float().abs() + 1e-2).all())


def test_mask_layouts(cuda, hip_lib):
    from aether_amd import ops
    qkv, table = inputs(3, 100, 2, device=cuda, seed=5)
    q, k, v = qkv.unbind(2)
    mask = _masks(3, 100, cuda)["holes"]
    o = ops.relbias_attn(q, k, v, table, key_mask=mask)
    assert torch.equal(ops.relbias_attn(q, k, v, table, key_mask=mask.t().contiguous().t()), o)
    wide = torch.zeros(3, 137, dtype=torch.bool, device=cuda)
    wide[:, 11:111] = mask
    assert torch.equal(ops.relbias_attn(q, k, v, table, key_mask=wide[:, 11:111]), o)
    one = mask[:1]
    assert torch.equal(ops.relbias_attn(q, k, v, table, key_mask=one.expand(3, 100)), ops.relbias_attn(q, k, v, table, key_mask=one.repeat(3, 1)))
    every = torch.ones(3, 100, dtype=torch.bool, device=cuda)
    assert torch.equal(ops.relbias_attn(q, k, v, table, key_mask=every), ops.relbias_attn(q, k, v, table))


def test_layouts(cuda, hip_lib):
    """Packed, head-major, padded, broadcast, reversed-stride and misaligned operands; what lies around a view stays as it was."""
    from aether_amd import ops
    qkv, table = inputs(2, 70, 3, device=cuda, seed=6)
    q, k, v = qkv.unbind(2)
    o = ops.relbias_attn(q, k, v, table)
    dense = [t.contiguous() for t in (q, k, v)]
    assert torch.equal(ops.relbias_attn(*dense, table), o)
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(ops.relbias_attn(*heads, table), o)
    wide = torch.full((2, 75, 3, 96), math.nan, dtype=torch.bfloat16, device=cuda)
    wide[:, 2:72, :, 8:72] = k
    assert torch.equal(ops.relbias_attn(q, wide[:, 2:72, :, 8:72], v, table), o)
    off = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device=cuda)[1:].view(q.shape).copy_(q)
    assert torch.equal(ops.relbias_attn(off, k, v, table), o)
    last = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(ops.relbias_attn(last, k, v, table), o)
    assert torch.equal(ops.relbias_attn(q, k, v, table.t().contiguous().t()), o)
    shared = ops.relbias_attn(q, k[:, :, :1].expand(-1, -1, 3, -1), v[:1].expand(2, -1, -1, -1), table)
    assert torch.equal(shared, ops.relbias_attn(q, k[:, :, :1].repeat(1, 1, 3, 1), v[:1].repeat(2, 1, 1, 1), table))
    assert ops.relbias_attn(q[:0], k[:0], v[:0], table).shape == (0, 70, 3, 64)
    o0, lse0 = ops.relbias_attn(q[:, :0], k[:, :0], v[:, :0], table, need_lse=True)
    assert o0.shape == (2, 0, 3, 64) and lse0.numel() == 0


@pytest.mark.parametrize("order", ["early", "late", "rising", "falling", "far_below"])
def test_score_ranges(cuda, hip_lib, order):
    """Scores of several hundred, their peak in the first tile, the last one, rising or falling over the tiles, and all of them far below zero.
    A score of 400 carries 66 · 2^-24 · 800 < 2^-8 of absolute error, numerator and denominator each."""
    from aether_amd import ops
    B, S, H = 1, 400, 2
    qkv, table = inputs(B, S, H, device=cuda, seed=7)
    at = torch.arange(S, device=cuda, dtype=torch.float32)
    level = dict(early=400 * (at < 5), late=400 * (at > 390), rising=at, falling=400 - at, far_below=at * 0 - 400)[order]
    q = qkv[:, :, 0].clone()
    k = qkv[:, :, 1].clone()
    q[..., 0], k[..., 0] = 4.0, (level / 4).to(torch.bfloat16)[None, :, None]
    v = qkv[:, :, 2]
    _check_o(ops.relbias_attn(q, k, v, table), q, k, v, table, extra=2.0 ** -6)


@pytest.mark.parametrize("order", ["early", "late", "middle", "rising", "falling", "far_below"])
@pytest.mark.parametrize("masked", [False, True])
def test_score_ranges_long(cuda, hip_lib, order, masked):
    """The same over many tiles, with and without what a backward pass needs; the mask takes keys at the end and a few in between."""
    from aether_amd import ops
    B, S, H = 2, 1100, 2
    qkv, table = inputs(B, S, H, device=cuda, seed=17)
    at = torch.arange(S, device=cuda, dtype=torch.float32)
    level = dict(early=400 * (at < 5), late=400 * (at > S - 60), middle=400 * ((at > 500) & (at < 510)), rising=at * (400 / S), falling=(S - at) * (400 / S), far_below=at * 0 - 400)[order]
    q = qkv[:, :, 0].clone()
    k = qkv[:, :, 1].clone()
    q[..., 0], k[..., 0] = 4.0, (level / 4).to(torch.bfloat16)[None, :, None]
    q[1, ::2, :, 0] = 0.25                    # every other row of the second item has ordinary scores
    v = qkv[:, :, 2]
    mask = None
    if masked:
        mask = torch.ones(B, S, dtype=torch.bool, device=cuda)
        mask[0, 1070:], mask[1, 700:720], mask[1, 1099:] = False, False, False
    o = ops.relbias_attn(q, k, v, table, key_mask=mask)
    _check_o(o, q, k, v, table, extra=2.0 ** -6, key_mask=mask)
    o2, _ = ops.relbias_attn(q, k, v, table, key_mask=mask, need_lse=True)
    _check_o(o2, q, k, v, table, extra=2.0 ** -6, key_mask=mask)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.bfloat16).min, -1e9, -300.0])
@pytest.mark.parametrize("which", ["right", "left", "far", "near"])
@pytest.mark.parametrize("S", [70, 600])
def test_buckets_that_are_switched_off(cuda, hip_lib, low, which, S):
    """A table that holds the lowest value, −inf or a very negative number for one side, for the far buckets or for the near ones; scores of −200 where the
    others are.  Every row has a key with an ordinary bucket."""
    from aether_amd import ops
    qkv, table = inputs(2, S, 2, device=cuda, seed=18)
    half = table.shape[0] // 2
    if which == "right":
        table[half:] = low
    elif which == "left":
        table[1:half] = low
    elif which == "far":
        table[12:half], table[half + 12:] = low, low
    else:
        table[1:5], table[half:half + 5] = low, low
    q, k, v = (t.clone() for t in qkv.unbind(2))
    q[..., 0], k[..., 0] = 4.0, -50.0
    for train in (False, True):
        o = ops.relbias_attn(q, k, v, table, need_lse=train)
        _check_o(o[0] if train else o, q, k, v, table, extra=2.0 ** -7)     # 66 · 2^-24 · 2 · (200 + 60 + 300) < 2^-7


@pytest.mark.parametrize("S", [40, 500])
def test_rows_of_the_lowest_value_are_uniform(cuda, hip_lib, S):
    """Every key of a row at the type's lowest value: all scores are the same number, as they are in a sum with it in float32."""
    from aether_amd import ops
    qkv, table = inputs(1, S, 2, device=cuda, seed=19)
    q, k, v = qkv.unbind(2)
    o = ops.relbias_attn(q, k, v, torch.full_like(table, torch.finfo(torch.bfloat16).min))
    want, T = v.double().mean(1, keepdim=True), v.double().abs().mean(1, keepdim=True)
    assert bool(((o.double() - want).abs() <= (BF16 + 2.0 ** -10) * T + BF16 * want.abs()).all())


@pytest.mark.parametrize("S", [64, 700])
def test_large_values(cuda, hip_lib, S):
    """v at the documented limit, scores that rise over the sequence."""
    from aether_amd import ops
    qkv, table = inputs(1, S, 2, device=cuda, seed=20)
    q, k, v = (t.clone() for t in qkv.unbind(2))
    q[..., 0], k[..., 0] = 4.0, (torch.arange(S, device=cuda) * (80 / S)).to(torch.bfloat16)[None, :, None]
    v = (v.clamp(-4, 4) * 2.5e21).contiguous()
    for train in (False, True):
        o = ops.relbias_attn(q, k, v, table, need_lse=train)
        _check_o(o[0] if train else o, q, k, v, table, extra=2.0 ** -6)


@pytest.mark.parametrize("where", [0, 77, 599])
def test_non_finite_inputs_long(cuda, hip_lib, where):
    """A NaN in one query of a long sequence makes that row NaN and no other; one in a key makes its head's rows NaN and no other head's."""
    from aether_amd import ops
    qkv, table = inputs(1, 600, 2, device=cuda, seed=21)
    q, k, v = qkv.unbind(2)
    o = ops.relbias_attn(q, k, v, table)
    bad = q.clone()
    bad[0, where, 1, 5] = math.nan
    got = ops.relbias_attn(bad, k, v, table)
    assert bool(torch.isnan(got[0, where, 1].float()).all())
    keep = torch.ones(600, 2, dtype=torch.bool, device=cuda)
    keep[where, 1] = False
    assert bool(((got[0][keep].float() - o[0][keep].float()).abs() <= 2 * BF16 * o[0][keep].float().abs() + 1e-2).all())
    bad = k.clone()
    bad[0, where, 1, 5] = math.nan
    got = ops.relbias_attn(q, bad, v, table)
    assert torch.equal(got[:, :, 0], o[:, :, 0]) and bool(torch.isnan(got[:, :, 1].float()).all())


def test_scale(cuda, hip_lib):
    from aether_amd import ops
    qkv, table = inputs(2, 150, 2, device=cuda, seed=8, qk=8.0)
    q, k, v = qkv.unbind(2)
    for scale in (0.125, 0.0, -0.1):
        _check_o(ops.relbias_attn(q, k, v, table, scale=scale), q, k, v, table, scale=scale)


def test_non_finite_inputs_stay_where_they_are(cuda, hip_lib):
    """A NaN in one query makes that row NaN and no other."""
    from aether_amd import ops
    qkv, table = inputs(1, 200, 2, device=cuda, seed=9)
    q, k, v = qkv.unbind(2)
    o = ops.relbias_attn(q, k, v, table)
    bad = q.clone()
    bad[0, 77, 1, 5] = math.nan
    got = ops.relbias_attn(bad, k, v, table)
    assert bool(torch.isnan(got[0, 77, 1].float()).all())
    keep = torch.ones(200, 2, dtype=torch.bool, device=cuda)
    keep[77, 1] = False
    assert bool(((got[0][keep].float() - o[0][keep].float()).abs() <= 2 * BF16 * o[0][keep].float().abs() + 1e-2).all())


def test_long(cuda, hip_lib):
    """A long sequence with a mask: only the last rows and the first are compared (the reference is quadratic)."""
    from aether_amd import ops
    S = 20000
    qkv, table = inputs(1, S, 1, device=cuda, seed=10)
    q, k, v = qkv.unbind(2)
    mask = torch.arange(S, device=cuda)[None, :] < S - 1234
    mask[0, 5000:9000] = False
    o = ops.relbias_attn(q, k, v, table, key_mask=mask)
    rows = torch.tensor([0, 1, 63, 64, 4999, 5000, 9000, 10007, S - 1235, S - 1234, S - 1], device=cuda)
    s = torch.matmul(q[0, rows, 0].double(), k[0, :, 0].double().t().contiguous())
    b = torch.tensor([[bucket(j - i, 32, 128) for j in range(S)] for i in rows.tolist()], device=cuda)
    s = (s + table.double()[b][..., 0]).masked_fill(~mask, -math.inf)
    p = torch.softmax(s, -1)
    want, T = p @ v[0, :, 0].double(), p @ v[0, :, 0].double().abs()
    err = (o[0, rows, 0].double() - want).abs()
    assert bool((err <= (BF16 + 2.0 ** -10) * T + BF16 * want.abs()).all())


def test_refusals(cuda, hip_lib):
    from aether_amd import ops
    qkv, table = inputs(2, 16, 2, device=cuda)
    q, k, v = qkv.unbind(2)
    mask = torch.ones(2, 16, dtype=torch.bool, device=cuda)
    for bad in (lambda: ops.relbias_attn(q.half(), k, v, table), lambda: ops.relbias_attn(q, k[:, :8], v, table), lambda: ops.relbias_attn(q[..., :32], k[..., :32], v[..., :32], table),
                lambda: ops.relbias_attn(q, k, v, table.float()), lambda: ops.relbias_attn(q, k, v, table[:, :1]), lambda: ops.relbias_attn(q, k, v, table[:31]),
                lambda: ops.relbias_attn(q, k, v, table[:2]), lambda: ops.relbias_attn(q, k, v, table, max_distance=8), lambda: ops.relbias_attn(q, k, v, table, max_distance=5000),
                lambda: ops.relbias_attn(q, k, v, table, key_mask=mask.float()), lambda: ops.relbias_attn(q, k, v, table, key_mask=mask[:, :8]),
                lambda: ops.relbias_attn(q[0], k[0], v[0], table), lambda: ops.relbias_attn(q, k, v, table, scale=math.nan), lambda: ops.relbias_attn(q, k, v, table, scale=1e-25)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="device tensors"):
        ops.relbias_attn(q, k, v, table, key_mask=mask.cpu())


def test_graph(cuda, hip_lib):
    """Captured and replayed on new values, eager work in between."""
    from aether_amd import ops
    qkv, table = inputs(2, 226, 4, device=cuda, seed=11)
    mask = _masks(2, 226, cuda)["right"]
    q, k, v = qkv.unbind(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.relbias_attn(q, k, v, table, key_mask=mask)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.relbias_attn(q, k, v, table, key_mask=mask)
    for n in (226, 100, 3):
        qkv.mul_(-0.9)
        mask[1] = torch.arange(226, device=cuda) < n
        graph.replay()
        want = ops.relbias_attn(q, k, v, table, key_mask=mask)
        torch.cuda.synchronize()
        assert torch.equal(o, want)


@pytest.mark.parametrize("S", [600, 1030])
@pytest.mark.parametrize("apart", [8, 16, 64])
def test_row_sums_next_to_the_largest_float(cuda, hip_lib, S, apart):
    """Two keys far above all others, 2^126 ... 2^129 times the row's first scores each: a row's sum lies next to fp32's largest number on either side, with the two keys'
    shares in one lane or in two (8 keys apart).  Scores are sums of two exact products: 66 · 2^-24 · 90, numerator and denominator each, is below 2^-10."""
    from aether_amd import ops
    levels = torch.arange(126.0, 129.01, 0.125, dtype=torch.float64) * math.log(2)
    B, H, at = len(levels), 1, 200
    g = torch.Generator().manual_seed(S + apart)
    q, k = torch.zeros(B, S, H, 64), torch.zeros(B, S, H, 64)
    q[..., 0], q[..., 1] = 4.0, 1.0
    coarse = (levels / 4).float().bfloat16()
    rest = (levels - 4 * coarse.double()).float().bfloat16()
    for j in (at, at + apart):
        k[:, j, 0, 0], k[:, j, 0, 1] = coarse.float(), rest.float()
    v = (torch.rand(B, S, H, 64, generator=g) - 0.5) / 2
    q, k, v = (t.to(torch.bfloat16).to(cuda) for t in (q, k, v))
    table = torch.zeros(32, H, dtype=torch.bfloat16, device=cuda)
    _check_o(ops.relbias_attn(q, k, v, table), q, k, v, table)
    o, lse = ops.relbias_attn(q, k, v, table, need_lse=True)
    _, p = _check_o(o, q, k, v, table)
    level = 4 * coarse.double() + rest.double()
    want = level / math.log(2) + 1
    assert bool(((lse[:B * S].view(B, S).double().cpu() - want[:, None]).abs() <= 66 * 2.0 ** -24 * 130).all())
    do = torch.randn(B, S, H, 64, generator=g).to(torch.bfloat16).to(cuda)
    dv = ops.relbias_attn_backward(do, q, k, v, o, lse, table)[2]
    pt, gd = p.transpose(2, 3).contiguous(), do.double().permute(0, 2, 1, 3).contiguous()
    want, lim = torch.matmul(pt, gd).permute(0, 2, 1, 3), (BF16 + 2.0 ** -10) * torch.matmul(pt, gd.abs()).permute(0, 2, 1, 3)
    assert bool(((dv.double() - want).abs() <= lim + BF16 * want.abs() + 1e-30).all())


@pytest.mark.parametrize("S", [1, 40, 70, 500, 1030])
def test_rows_whose_buckets_are_all_switched_off(cuda, hip_lib, S):
    """A row is without keys too where the mask and buckets at −inf leave none together: 0, and no gradient through it.  Here rows see no key to their right, and the
    second item is padded in front."""
    from aether_amd import ops
    n = min(25, S - 1)
    qkv, table = inputs(2, S, 2, device=cuda, seed=23)
    table[table.shape[0] // 2:] = -math.inf
    q, k, v = qkv.unbind(2)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(S)).to(torch.bfloat16).to(cuda)
    mask = torch.ones(2, S, dtype=torch.bool, device=cuda)
    mask[1, :n] = False
    o = ops.relbias_attn(q, k, v, table, key_mask=mask)
    o2, lse = ops.relbias_attn(q, k, v, table, key_mask=mask, need_lse=True)
    assert not o[1, :n].any() and not o2[1, :n].any() and bool(torch.isposinf(lse[:2 * S * 2].view(2, 2, S)[1, :, :n]).all())
    for got in (o, o2):
        assert bool(torch.isfinite(got.float()).all())
        alone = ops.relbias_attn(q[1:, n:], k[1:, n:], v[1:, n:], table)
        assert bool(((got[1, n:].double() - alone[0].double()).norm() <= 2 * BF16 * alone.double().norm()))
    grads = ops.relbias_attn_backward(do, q, k, v, o2, lse, table, key_mask=mask)
    assert all(bool(torch.isfinite(t.float()).all()) for t in grads) and not any(t[1, :n].any() for t in grads[:3])
    a, l = ops.relbias_attn(q[1:, n:], k[1:, n:], v[1:, n:], table, need_lse=True)
    for x, y in zip(grads[:3], ops.relbias_attn_backward(do[1:, n:], q[1:, n:], k[1:, n:], v[1:, n:], a, l, table)):
        assert bool((x[1, n:].double() - y[0].double()).norm() <= 4 * BF16 * y.double().norm())
    # every bucket off: nothing anywhere
    off = torch.full_like(table, -math.inf)
    o, lse = ops.relbias_attn(q, k, v, off, need_lse=True)
    assert not o.any() and not any(t.any() for t in ops.relbias_attn_backward(do, q, k, v, o, lse, off))
