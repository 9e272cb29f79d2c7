"""The definitions of the drafted-token operators in 64 bits, written for reading, not for speed."""
import math

import numpy as np
import torch

MOST = {"int8": 127.0, "e4m3": 448.0}


def rotate(x, positions, frequencies, factor, interleaved, inverse=False):
    """x [..., heads, hd] (any dtype), positions x.shape[:-2] -> fp64."""
    w = torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    n = w.numel()
    a = positions.double()[..., None, None] * w
    c, s = factor * a.cos(), (-factor if inverse else factor) * a.sin()
    x = x.double()
    y = x.clone()
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def rotate_slack(x, n, factor, interleaved):
    """|x0| + |x1| of the pair that each value belongs to, times factor: what the errors of its angle are relative to."""
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    m = torch.zeros_like(x, dtype=torch.float64)
    m[..., first] = m[..., second] = factor * (x[..., first].double().abs() + x[..., second].double().abs())
    return m


def attention(q, k, v, length, counts, masks, max_len, scale=None):
    """q [B,T,nh,hd], k, v [B,kv,max_len,hd] fp64 -> fp64 [B,T,nh,hd]; masks: numpy uint64 [B,T] or None (a chain)."""
    B, T, nh, hd = q.shape
    kv = k.shape[1]
    out = torch.zeros(B, T, nh, hd, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = T if counts is None else max(0, min(T, int(counts[b])))
        l = min(max_len, max(0, int(length[b])))
        for i in range(n):
            see = list(range(l)) + [l + j for j in range(n) if l + j < max_len and ((j <= i) if masks is None else (int(masks[b][i]) >> j) & 1)]
            if not see:
                continue
            see = torch.tensor(see, device=q.device)
            kk, vv = k[b][:, see].repeat_interleave(nh // kv, 0), v[b][:, see].repeat_interleave(nh // kv, 0)
            s = torch.einsum("hd,hnd->hn", q[b, i].double(), kk) * (hd ** -0.5 if scale is None else scale)
            out[b, i] = torch.einsum("hn,hnd->hd", torch.softmax(s, -1), vv)
    return out


def attention_slack(q, k, v, dtype, scale=None):
    """Largest error that fp32 sums and weights held in dtype allow, without the result's own rounding: a score's sum of hd products
    is off by (hd + 4) 2^-24 sum |q k| scale at most (twice that where the unit truncates), a weight by twice its score's error (its own and that of the largest
    score) and by eps / 2 where it is held in dtype, the running sums by the number of keys times 2^-24 (random signs: its root, times 4)."""
    hd, n = q.shape[-1], k.shape[2]
    top = float(q.double().abs().amax() * k.double().abs().amax()) * hd * abs(hd ** -0.5 if scale is None else scale)
    rms = float(q.double().square().sum(-1).amax().sqrt() * torch.nan_to_num(k.double()).square().sum(-1).amax().sqrt()) * abs(hd ** -0.5 if scale is None else scale)
    score = 2 * (hd + 4) ** 0.5 * 2.0 ** -23 * min(top, rms)
    weight = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 2.0 ** -22
    return (2 * score + weight + 4 * math.sqrt(n) * 2.0 ** -24) * float(v.double().abs().amax())


def draw(mass, u):
    run = np.cumsum(mass)
    if not (run[-1] > 0) or not np.isfinite(run[-1]):
        return -1
    over = np.nonzero(run > u * run[-1])[0]
    return int(over[0]) if len(over) else int(np.nonzero(mass > 0)[0][-1])


def verify(tokens, target, uniform, parents, draft, n):
    """One sequence, numpy: -> (path, next)."""
    if n <= 0:
        return [], -1
    if draft is not None:
        v = 0
        while v + 1 < n:
            x = int(tokens[v + 1])
            if 0 <= x < target.shape[1] and float(uniform[v + 1]) * float(draft[v, x]) < float(target[v, x]):
                v += 1
                continue
            rest = np.maximum(target[v].astype(np.float64) - draft[v].astype(np.float64), 0)
            return list(range(v + 1)), draw(rest if rest.sum() != 0 else target[v].astype(np.float64), float(uniform[0]))
        return list(range(v + 1)), draw(target[v].astype(np.float64), float(uniform[0]))
    path, v = [0], 0
    while True:
        x = int(target[v]) if target.ndim == 1 else draw(target[v].astype(np.float64), float(uniform[v]))
        hit = [c for c in range(v + 1, n) if (c - 1 if parents is None else int(parents[c])) == v and int(tokens[c]) == x]
        if not hit:
            return path, x
        v = hit[0]
        path.append(v)


def random_tree(r, T, near=6):
    """parents (numpy int64, node 0 the root) and what each node sees (uint64)."""
    par = np.full(T, -1, np.int64)
    see = np.zeros(T, np.uint64)
    for i in range(T):
        if i:
            par[i] = r.randint(max(0, i - near), i)
        see[i] = np.uint64(1 << i) | (see[par[i]] if i else np.uint64(0))
    return par, see
