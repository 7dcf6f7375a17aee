"""Plain 64-bit implementations of the paged-cache operators, and the bounds
that the kernels' results are held to.

Bounds. With u half a step of the output type (bf16 2^-8, fp16 2^-11):
  a rotated value   u |y| + 2^-20 (|x1| + |x2|): the angle's 32-bit turn is off
                    by at most pi 2^-24, sine and cosine by 2 ulp, two 32-bit
                    products and their scale: below 12 * 2^-24 in all
  a score           d = (dim + 4) 2^-24 scale sum |q| |k|, the 32-bit sum of
                    dim products and the scaling
  an output         u |o| + (uP + 2 d + 2^-19) A, A = sum p |v| / sum p: a
                    weight p is off by the score's error in numerator and
                    denominator and by exp2 (2^-22), is rounded to uP, and the
                    32-bit sums add below 2^-20 A more (blocks of products,
                    then one addition per tile). uP is u where P is rounded
                    once, u^2 where it is kept as two numbers
  log-sum-exp       d + 2^-20 (1 + |lse|)
FP16's smallest step adds 2^-25 to a result, and 2^-25 sum |v| / sum p to a
weighted sum.
"""
import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
SMALLEST = {torch.bfloat16: 0.0, torch.float16: 2.0**-25}


def rotate(x, pos, freq, axis=None, interleaved=False, scale=1.0, inverse=False):
    """x [T, H, D] (any float tensor), pos [A, T] integers, in 64 bits; and sum |x1| + |x2| of each value's pair."""
    x = x.double().cpu()
    f, n = freq.double().cpu(), freq.numel()
    ax = torch.zeros(n, dtype=torch.long) if axis is None else axis.long().cpu()
    a = (pos.cpu().double()[ax] * f[:, None]).T[:, None]
    c, s = torch.cos(a) * scale, torch.sin(a) * scale * (-1 if inverse else 1)
    i1 = torch.arange(n) * 2 if interleaved else torch.arange(n)
    i2 = i1 + 1 if interleaved else i1 + n
    y, size = x.clone(), torch.zeros_like(x)
    x1, x2 = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = x1 * c - x2 * s, x2 * c + x1 * s
    size[..., i1] = size[..., i2] = x1.abs() + x2.abs()
    return y, size


def check_rotated(got, want, size, scale=1.0):
    u = HALF_STEP[got.dtype]
    got = got.detach().double().cpu()
    err = (got - want).abs()
    tol = u * want.abs() + abs(scale) * 2.0**-20 * size + 2.0**-25
    assert bool((err <= tol).all()), float((err - tol).max())
    same = size == 0  # copied channels
    assert torch.equal(got[same], want[same])


def tokens_of(pages, table, n):
    """The first n tokens [n, H, D] that a list of pages holds, in 64 bits."""
    pt = pages.shape[2]
    rows = [pages[int(table[t // pt]), :, t % pt] for t in range(0, n)] if n < 4 * pt else None
    if rows is None:
        idx = torch.as_tensor([int(p) for p in table[: (n + pt - 1) // pt]], device=pages.device)
        return pages[idx].permute(0, 2, 1, 3).reshape(-1, *pages.shape[1:2], pages.shape[3])[:n].double().cpu()
    return torch.stack(rows).double().cpu() if rows else torch.zeros(0, pages.shape[1], pages.shape[3], dtype=torch.double)


def attention(q, ks, vs, seen, scale):
    """One sequence: q [n, Hq, D], K and V [L, H, D] (64 bits), row i sees its first seen[i] tokens.
    Returns out, lse, A (sum p |v| / sum p), d (score error), w (sum |v| / sum p) per row and head."""
    n, hq, dim = q.shape
    L, H, _ = ks.shape
    g = hq // H
    out = torch.zeros(n, hq, dim, dtype=torch.double)
    lse = torch.full((n, hq), -math.inf, dtype=torch.double)
    A, W = torch.zeros(n, hq, dim, dtype=torch.double), torch.zeros(n, hq, dim, dtype=torch.double)
    d = torch.zeros(n, hq, dtype=torch.double)
    for h in range(hq):
        k, v = ks[:, h // g], vs[:, h // g]
        for i in range(n):
            m = int(seen[i])
            if m <= 0:
                continue
            s = (k[:m] @ q[i, h]) * scale
            z = torch.logsumexp(s, 0)
            p = torch.exp(s - z)
            out[i, h], lse[i, h] = p @ v[:m], z
            A[i, h] = p @ v[:m].abs()
            W[i, h] = v[:m].abs().sum(0) * math.exp(min(700.0, float(s.max() - z)))
            d[i, h] = (dim + 4) * 2.0**-24 * abs(scale) * float((k[:m].abs() @ q[i, h].abs()).max())
    return out, lse, A, d, W


def check_attention(got, got_lse, want, dtype, split_p):
    out, lse, A, d, W = want
    u = HALF_STEP[dtype]
    up = u * u if split_p else u
    got = got.double().cpu()
    tol = u * out.abs() + (up + 2 * d[..., None] + 2.0**-19) * A + SMALLEST[dtype] * (1 + W) + 1e-30
    err = (got - out).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()))
    empty = lse == -math.inf
    assert bool((got[empty] == 0).all())
    if got_lse is not None:
        gl = got_lse.double().cpu()
        assert torch.equal(gl == -math.inf, empty)
        f = ~empty
        assert bool(((gl - lse).abs()[f] <= d[f] + 2.0**-20 * (1 + lse[f].abs())).all())


def make_batch(g, lens, new, page, n_kv, dim, dtype, device="cuda:0", spare=3, unused=math.nan, kscale=1.0):
    """Pools with random pages, a table in random order (-1 past each sequence), places past the lengths holding `unused`."""
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + spare
    k = (torch.randn(total, n_kv, page, dim, generator=g) * kscale).to(dtype)
    v = torch.randn(total, n_kv, page, dim, generator=g).to(dtype)
    order = torch.randperm(total, generator=g)
    width = max(max(need), 1) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
        if lens[b] % page:
            k[table[b, n - 1].long(), :, lens[b] % page:] = unused
            v[table[b, n - 1].long(), :, lens[b] % page:] = unused
    starts = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
    return dict(k=k.to(device), v=v.to(device), table=table.to(device), starts=starts.to(device),
                lens=torch.tensor(lens, dtype=torch.int32, device=device), spare=order[at:])


def batch_reference(c, lens, new, q, scale, prefix=None):
    """The whole batch's attention in 64 bits; prefix: (K, V) [P, H, D] seen by every row."""
    parts = []
    t = 0
    qd = q.double().cpu()
    for b, n in enumerate(lens):
        ks, vs = tokens_of(c["k"], c["table"][b].tolist(), n), tokens_of(c["v"], c["table"][b].tolist(), n)
        seen = [n - new[b] + i + 1 for i in range(new[b])]
        if prefix is not None:
            p = prefix[0].shape[0]
            ks, vs = torch.cat([prefix[0], ks]), torch.cat([prefix[1], vs])
            seen = [p + max(x, 0) for x in seen]
        parts.append(attention(qd[t:t + new[b]], ks, vs, seen, scale))
        t += new[b]
    return [torch.cat([p[i] for p in parts]) for i in range(5)]
