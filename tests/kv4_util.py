"""64-bit definitions of the 4-bit cache's operators, for its tests."""
import math

import torch

BF16, F64 = torch.bfloat16, torch.float64


def coded(y):
    """Rows [..., D] (bf16 values) -> (low, scale, codes) per 64 dims, fp64 [..., D / 64, 1 | 1 | 64], from the definition."""
    y = y.to(BF16).to(F64).unflatten(-1, (y.shape[-1] // 64, 64))
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    scale = ((high - low) / 15).to(torch.float32).to(BF16).to(F64)
    q = (y - low) / torch.where(scale == 0, 1.0, scale)
    return low, scale, torch.where(scale == 0, 0.0, torch.round(q).clamp(max=15))


def values(y):
    low, scale, codes = coded(y)
    return (low + scale * codes).flatten(-2)


def turned(x, w, cos, sin, rot, neox, eps):
    """Norm (rounded to bf16) and rotation of [T, heads, D]; cos, sin [T, rot / 2]; fp64, unrounded."""
    x = x.to(F64)
    if w is not None:
        x = (x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(F64)).to(torch.float32).to(BF16).to(F64)
    half = rot // 2
    y = x.clone()
    if half:
        a = torch.arange(half, device=x.device) * (1 if neox else 2)
        b = a + (half if neox else 1)
        c, s = cos[:, None].to(F64), sin[:, None].to(F64)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def attention(q, rows, lens, news, scale, hkv, rounded):
    """q [T, Hq, D]; rows: per sequence the bf16 (keys, values) [len, Hkv, D] that were coded; -> (result, tolerance) [T, Hq, D] fp64.

    The tolerance counts roundings: half a step of bf16 is 2^-8 of a value, of fp16 2^-11. Results are rounded once (2^-8 |o|) and
    probabilities once: in the form on codes, times their scales, to fp16 (2^-11 of sum p s c; the low ends are added in fp32), over expanded
    tiles to bf16 (2^-8 of sum p |v|). Scores are fp32 sums of at most 128 products, good to 2^-22 of the sum of their magnitudes, some
    2^-17 at the sizes here; with expanded tiles (`rounded`) every key and value is rounded too: six standard deviations of 64 or
    128 independent roundings (uniform within half a step: 2^-8 / sqrt 3) in a score, 2^-8 sum p |v| for the values. The form on codes rounds half of its factors of
    queries to fp16: likewise, with 2^-11, in the codes' part of a score. A product of it that is below fp16's normal numbers is good to 2^-25 where the largest that can stand beside it is 2^6 and more: 2^-31
    of it a key."""
    out, tol = [], []
    at = 0
    for (k, v), n, new in zip(rows, lens, news):
        hq, d = q.shape[1], q.shape[2]
        g = hq // hkv
        qq = q[at:at + new].to(F64).unflatten(1, (hkv, g))
        at += new
        if n == 0:
            out.append(torch.zeros(new, hq, d, dtype=F64, device=q.device))
            tol.append(torch.zeros_like(out[-1]))
            continue
        kk, vv = values(k[:n]), values(v[:n])
        low, s, c = coded(v[:n])
        z = torch.einsum("qhgd,khd->hgqk", qq, kk) * scale
        z = z + torch.full((new, n), -math.inf, dtype=F64, device=q.device).triu(n - new + 1)
        p = z.softmax(-1)
        o = torch.einsum("hgqk,khd->qhgd", p, vv)
        size = torch.einsum("hgqk,khd->qhgd", p, vv.abs())
        if rounded:
            spread = torch.einsum("qhgd,khd->hgqk", qq.square(), kk.square()).sqrt() * scale
            dz = (6 * 2 ** -8 / math.sqrt(3) * spread).amax(-1).permute(2, 0, 1)[..., None]
            slack = (2 * 2 ** -8 + 2 * dz + 2 ** -16) * size
        else:
            steps = torch.einsum("hgqk,khd->qhgd", p, (s * c).flatten(-2))
            spread = torch.einsum("qhgd,khd->hgqk", qq.square(), c.flatten(-2).square() * s.expand(-1, -1, -1, 64).flatten(-2).square()).sqrt()
            dz = (6 * 2 ** -11 / math.sqrt(3) * spread * scale).amax(-1).permute(2, 0, 1)[..., None]
            least = 2 ** -31 * 15 * n * s.amax((0, 2, 3))[None, :, None, None] * p.amax(-1).permute(2, 0, 1)[..., None]
            slack = 2 ** -11 * steps + least + (2 ** -16 + 2 * dz) * (size + steps)
        out.append(o.flatten(1, 2))
        tol.append((slack + 2 ** -8 * o.abs()).flatten(1, 2) * 1.01)
    return torch.cat(out), torch.cat(tol)
