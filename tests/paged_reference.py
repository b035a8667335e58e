"""Plain 64-bit forms of the causal and paged operators, and the tolerances
that follow from the roundings the kernels make."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows_attention(q, k, v, scale):
    """One request in 64 bits: q [n, H, D] (its newest tokens), k/v [m, Hk, D].
    Returns o [n, H, D], lse [H, n], and sum_j p_j |v_j| [n, H, D]."""
    q, k, v = q.double(), k.double(), v.double()
    n, h, d = q.shape
    m, hk, _ = k.shape
    if m == 0:
        z = torch.zeros((n, h, d), dtype=torch.float64, device=q.device)
        return z, torch.full((h, n), -math.inf, dtype=torch.float64, device=q.device), z
    k = k.repeat_interleave(h // hk, 1)
    v = v.repeat_interleave(h // hk, 1)
    x = torch.einsum("nhd,mhd->hnm", q, k) * scale
    last = m - n + torch.arange(n, device=q.device)
    hidden = torch.arange(m, device=q.device)[None] > last[:, None]
    x = x.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.where(lse[..., None] == -math.inf, 0.0, (x - lse[..., None]).exp())
    return torch.einsum("hnm,mhd->nhd", p, v), lse, torch.einsum("hnm,mhd->nhd", p, v.abs())


def attention_bound(o, weight, in_dtype, out_dtype, dim, keys, vmax, smax):
    """How far a kernel's o may be from the 64-bit one, element by element.

    weight = sum_j p_j |v_j|. The softmax numerators are rounded to the inputs'
    type (half a step each, relative), the scores are fp32 sums of `dim`
    products of size smax / dim or so each (error dim * 2^-24 * smax, entering
    through exp once in the numerator and once in the sum), the exponential
    itself is good to 4e-6, the sums over keys are fp32. fp16 numerators below
    2^-14 lose 2^-25 each beside a sum of at least 1. The result is rounded to
    the output's type."""
    rel = half_step(in_dtype) + 2 * (dim * 2.0 ** -24 * smax + 4e-6) + keys * 2.0 ** -24
    low = keys * 2.0 ** -25 * vmax if in_dtype == torch.float16 else 0.0
    return weight * rel + low + o.abs() * half_step(out_dtype) + 1e-30


def check_attention(got, lse, want, want_lse, weight, in_dtype, dim, keys, vmax, smax, what=""):
    bound = attention_bound(want, weight, in_dtype, got.dtype, dim, keys, vmax, smax)
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= bound).all(), (what, (err / bound).max().item(), err.max().item())
    if lse is not None:
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty), what
        dl = (lse.double() - want_lse)[~empty].abs()
        tol = dim * 2.0 ** -24 * smax + 4e-6 + keys * 2.0 ** -24 + 2.0 ** -23 * want_lse[~empty].abs()
        assert (dl <= tol).all(), (what, (dl / tol).max().item() if dl.numel() else 0)


def score_size(q, k, scale):
    """An upper bound of sum_d |q_d k_d| * scale over all pairs."""
    if q.numel() == 0 or k.numel() == 0:
        return 0.0
    return float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max() * scale)


def rotate(x, cos, sin, half):
    x = x.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    if half:
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def norm(x, gain, eps):
    x = x.double()
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gain.double()


def plan(ctx_lens, new_lens, free, table, page, room):
    """One step planned with Python integers; None if the pages do not suffice."""
    free = list(free)
    table = [list(r) for r in table]
    cu, kv, pos, slots = [0], [], [], []
    for i, (c, n) in enumerate(zip(ctx_lens, new_lens)):
        for col in range(-(-c // page), -(-(c + n) // page)):
            if not free:
                return None
            table[i][col] = free.pop()
        cu.append(cu[-1] + n)
        kv.append(c + n)
        for x in range(c, c + n):
            pos.append(x)
            slots.append(table[i][x // page] * page + x % page)
    pad = room - len(pos)
    return table, cu, kv, pos + [0] * pad, slots + [-1] * pad, len(free)
