"""Inputs, the 64-bit oracle and the tolerances of the cross-attention tests.

The oracle is written apart from the operator: dense scores over the whole batch, a mask that says
which pairs meet, and the gradients by their formulas.
"""
import math

import torch

U32 = 2.0 ** -24  # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ptr(lens, dev="cpu"):
    return torch.tensor([0] + list(torch.tensor(lens, dtype=torch.long).cumsum(0)) if lens else [0],
                        dtype=torch.int32, device=dev)


def bucket_by_formula(q_pos, k_pos, num, far, two_sided, unit):
    """Bucket numbers [Nq, Nk] straight from the rule, in Python's whole numbers."""
    side = num // 2 if two_sided else num
    near = side // 2
    steps = side - near

    def of(n):
        n = min(n, far)
        if n < near:
            return n
        b = near
        while b + 1 < side and n ** steps * near ** (b + 1 - near) >= far ** (b + 1 - near) * near ** steps:
            b += 1
        return b

    table = [of(n) for n in range(far + 1)]
    out = torch.zeros(q_pos.shape[0], k_pos.shape[0], dtype=torch.long)
    for i in range(q_pos.shape[0]):
        for j in range(k_pos.shape[0]):
            if unit is not None:
                d = math.sqrt(sum((float(k_pos[j, c]) - float(q_pos[i, c])) ** 2 for c in range(3))) / unit
                out[i, j] = table[far if not d < far else int(d)]
            else:
                rel = int(k_pos[j]) - int(q_pos[i])
                n = abs(rel) if two_sided else max(-rel, 0)
                out[i, j] = table[min(n, far)] + (side if two_sided and rel > 0 else 0)
    return out


def oracle(q, k, v, ql, kl, scale=None, key_mask=None, table=None, bucket=None, d_out=None):
    """Dense, in 64 bits, on the CPU.  Returns a dict: out, and with d_out dq, dk, dv, dtable and what
    the table's tolerance goes by."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    H, D, g = q.shape[1], q.shape[2], q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    qs, ks = (torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n, dtype=torch.long)) for n in (ql, kl))
    qs = torch.cat([qs, torch.full((q.shape[0] - len(qs),), -1)])
    ks = torch.cat([ks, torch.full((k.shape[0] - len(ks),), -2)])
    pair = qs.view(-1, 1) == ks.view(1, -1)
    if key_mask is not None:
        pair = pair & key_mask.cpu().view(1, -1)
    used = pair.any(0).view(-1, 1, 1)
    k, v = (torch.where(used, t, torch.zeros_like(t)).repeat_interleave(g, 1).transpose(0, 1) for t in (k, v))
    q = torch.where(pair.any(1).view(-1, 1, 1), q, torch.zeros_like(q)).transpose(0, 1)
    s = q @ k.transpose(1, 2) * scale
    if table is not None:
        s = s + table.detach().double().cpu()[:, bucket]
    s = s.masked_fill(~pair, -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:2] + (1,))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    res = {"out": (p @ v).transpose(0, 1)}
    if d_out is None:
        return res
    do = d_out.detach().double().cpu().transpose(0, 1)
    do = torch.where(pair.any(1).view(1, -1, 1), do, torch.zeros_like(do))
    dp = do @ v.transpose(1, 2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)

    def shared(t):  # [H, Nk, D] -> [Nk, Hk, D]
        return t.view(H // g, g, t.shape[1], D).sum(1).transpose(0, 1)

    res.update(dq=(ds @ k).transpose(0, 1) * scale, dk=shared(ds.transpose(1, 2) @ q) * scale,
               dv=shared(p.transpose(1, 2) @ do))
    if table is not None:
        B = table.shape[1]
        size = p * (dp.abs() + delta.abs())
        res["dtable"] = torch.stack([ds[:, bucket == b].sum(-1) for b in range(B)], -1)
        res["dtable_size"] = torch.stack([size[:, bucket == b].sum(-1) for b in range(B)], -1)
    return res


def norm_tol(dtype, width, length, grad, saved):
    """Bound of |got - ref|_2 / |ref|_2.

    float32: rounding errors of sums grow like the root of their terms: a score has `width` of them
    and a row's sums `length`; 4 standard steps each, and 8 for the exponential and the scalings;
    a gradient chains two such products.
    16 bits: the output is rounded once (half a step at most), and one factor of its last product as
    well (p without gradients; dS; p of dv), whose errors are independent from key to key: half a
    step again.  Gradients: twice that, because dS cancels against its row."""
    f32 = 4 * U32 * (math.sqrt(width) + math.sqrt(max(length, 1)) + 8) * (2 if grad else 1)
    if dtype == torch.float32:
        return f32
    h = HALF[dtype]
    return (4 * h if grad else h if saved else 2 * h) + f32


def check_norm(got, ref, tol, what, floor=0.0):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off, size = (got - ref).norm().item(), ref.norm().item()
    assert off <= tol * size + floor, f"{what}: off by {off:.3e} of {size:.3e} (tol {tol:.1e})"


def score_error(q, k, scale):
    """Bound of a score's absolute error, where scores are not of the order of 1: a score is a sum of D
    products, rounded D times by half a step of a partial sum, which is at most S = |scale| sum |q k|;
    the errors are independent, so they add up to the root of D of them, and 4 more cover the scale's,
    the bias' and the logarithm's.  p = exp(score - lse) is off by that much, relatively, once for the
    score and once for the lse."""
    g = q.shape[1] // k.shape[1]
    kk = k.double().abs().repeat_interleave(g, 1).transpose(0, 1)
    size = (q.double().abs().transpose(0, 1) @ kk.transpose(1, 2)).max().item() * abs(scale)
    return 2 * (math.sqrt(q.shape[2]) + 4) * size * U32


def check_table(got, res, dtype, what, p_error=0.0):
    """Every dS is off by its factors' roundings, (|dP| + |delta|) p times a few 2^-24, and in 16 bits
    by delta's: `out` and what its rounding leaves give 2 half steps squared, p in two parts as much."""
    h = HALF[dtype]
    rel = 128 * U32 + p_error + (0 if dtype == torch.float32 else 4 * h * h)
    off = (got.detach().double().cpu() - res["dtable"]).abs()
    bound = rel * res["dtable_size"] + 1e-30
    assert (off <= bound).all(), f"{what}: off by {(off / bound).max().item():.2f} of the bound"
