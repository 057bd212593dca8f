"""Attention with a relative position bias in float64, written from the definition."""
import math

import torch


def bucket(d, num_buckets, max_distance):
    """One distance's bucket, from the definition: exact below num_buckets / 4, then floor of a logarithm, found by whole-number comparison."""
    half = num_buckets // 2
    near = half // 2
    n, base = abs(d), half if d > 0 else 0
    if n < near:
        return base + n
    b = 0
    while b + 1 < half - near and n ** (half - near) * near ** (b + 1) >= max_distance ** (b + 1) * near ** (half - near):
        b += 1
    return base + near + b


def attention(q, k, v, table, max_distance=128, scale=1.0, key_mask=None):
    """-> (o [B, S, H, 64], p [B, H, S, S]), float64 and differentiable; inputs float64."""
    B, S, H, _ = q.shape
    one_side = torch.tensor([bucket(d, table.shape[0], max_distance) for d in range(1 - S, S)], device=q.device)
    at = torch.arange(S, device=q.device)
    bias = table[one_side[at[None, :] - at[:, None] + S - 1]].permute(2, 0, 1)
    if key_mask is not None:                  # what stands behind the mask does not take part
        k = torch.where(key_mask[:, :, None, None], k, torch.zeros((), dtype=k.dtype, device=k.device))
        v = torch.where(key_mask[:, :, None, None], v, torch.zeros((), dtype=v.dtype, device=v.device))
    q, k, v = (t.permute(0, 2, 1, 3).contiguous() for t in (q, k, v))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale + bias
    if key_mask is None:
        p = torch.softmax(s, -1)
    else:
        keep = key_mask[:, None, None, :]
        p = torch.softmax(s.masked_fill(~keep, -1e30), -1) * keep
    return torch.matmul(p, v).permute(0, 2, 1, 3), p


def inputs(B, S, H, num_buckets=32, seed=0, device="cpu", qk=0.5):
    g = torch.Generator().manual_seed(seed + 7 * S + 1000 * B + H)
    qkv = torch.randn(B, S, 3, H, 64, generator=g)
    qkv[:, :, :2] *= math.sqrt(qk)
    table = torch.randn(num_buckets, H, generator=g) * 2
    return qkv.to(torch.bfloat16).to(device), table.to(torch.bfloat16).to(device)
