"""The drafted-token operators from their definitions in 64 bits (NumPy), for their tests."""
import math

import numpy as np


def rope_freqs(n_rot, theta, scaling=0, factor=1.0, low=0.0, high=0.0, orig_ctx=0, factors=None):
    """Radians per position of each pair, by the formulas of the header."""
    out = []
    for i in range(n_rot // 2):
        f = theta ** (-2.0 * i / n_rot) / (1.0 if factors is None else float(factors[i]))
        if scaling == 0:
            keep = 1.0
        elif scaling == 1:
            keep = 0.0
        elif scaling == 2:
            keep = (orig_ctx * f / (2 * math.pi) - low) / (high - low)
        else:
            def pair_of(turns):
                return n_rot * math.log(orig_ctx / (turns * 2 * math.pi)) / (2 * math.log(theta))
            first, last = max(math.floor(pair_of(high)), 0), min(math.ceil(pair_of(low)), n_rot - 1)
            keep = 1 - (i - first) / max(last - first, 0.001)
        keep = min(max(keep, 0.0), 1.0)
        out.append(f * keep + f / factor * (1 - keep) if scaling else f)
    return np.array(out)


def rope(x, pos, freq, interleaved, mscale):
    """Rotated x [tok][head][dim] (float64) and the magnitude that its rounding errors scale with."""
    x = x.astype(np.float64)
    y, size = x.copy(), np.zeros_like(x)
    n = len(freq)
    ang = pos.astype(np.float64)[:, None, None] * freq
    c, s = np.cos(ang) * mscale, np.sin(ang) * mscale
    one, two = ((slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n)))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one] = size[..., two] = abs(mscale) * (abs(a) + abs(b))
    return y, size


def paths(parent):
    """The nodes each node sees among the drafted ones: its path to a root, or none (padding)."""
    out = []
    for i in range(len(parent)):
        path, j = [], i
        while j >= 0:
            path.append(j)
            up = int(parent[j])
            j = up if up == -1 or 0 <= up < j else -2
        out.append(sorted(path) if j == -1 else [])
    return out


def tree_attention(q, k, v, n_past, parent, scale, half_step):
    """(out, tolerance) for q [seq][node][head][dim] over k, v [seq][kv][rows][dim], all float64.
    half_step: half the relative step of the type, 0 where probabilities and outputs stay in 32 bits.

    The tolerance: with u = 2^-23 (a 32-bit sum on the tensor cores may truncate), a score of dim
    products is off by at most e = dim u scale sum|q k| + 4 u |score|, a probability by the factor
    exp(2 e) (its own score and the sum's) with 2^-22 for the exponential, a sum of n terms by n u
    of the sum of magnitudes, and the rounded probability by half a step."""
    S, N, H, D = q.shape
    KV, L = k.shape[1], k.shape[2]
    out, tol = np.zeros((S, N, H, D)), np.zeros((S, N, H, D))
    u = 2.0 ** -23
    for s in range(S):
        seen = paths(parent[s] if parent is not None else np.arange(N) - 1)
        past = max(int(n_past[s]), 0)
        for i in range(N):
            if not seen[i]:
                continue
            rows = [j for j in list(range(min(past, L))) + [past + j for j in seen[i]] if j < L]
            if not rows:
                continue
            for h in range(H):
                kk, vv = k[s, h // (H // KV), rows], v[s, h // (H // KV), rows]
                x = kk @ q[s, i, h] * scale
                e = D * u * abs(scale) * (abs(kk) @ abs(q[s, i, h])) + 4 * u * abs(x) + 4 * u * abs(x - x.max())
                p = np.exp(x - x.max())
                p /= p.sum()
                out[s, i, h] = p @ vv
                rel = math.expm1(2 * e.max()) + 2.0 ** -21 + 2 * len(rows) * u + half_step
                tol[s, i, h] = rel * (p @ abs(vv)) + half_step * abs(out[s, i, h]) + 1e-30
    return out, tol


def sample(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, prob) of one row of float64 logits."""
    ok = np.flatnonzero(row > -np.inf)
    if not ok.size:
        return -1, 0.0
    order = ok[np.argsort(-row[ok], kind="stable")]
    if not temperature > 0:
        return int(order[0]), 1.0
    top = row[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        # (an infinite logit takes all the weight, whatever the temperature)
        far = -np.inf if np.isinf(top) else 0.0
        w = np.where(row[order] == top, 1.0, np.exp(far if far else (row[order] - top) / temperature))
    n = len(order)
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        c = np.cumsum(w[:n])
        n = min(n, int((c < max(top_p, 0.0) * c[-1]).sum()) + 1)
    if min_p > 0:
        n = max(1, min(n, int((w >= min(min_p, 1.0)).sum())))
    kept = np.argsort(order[:n])
    ids, wk = order[:n][kept], w[:n][kept]
    wk = np.where(wk * 2.0 ** 44 > 0.5, wk, 0.0)  # what rounds to no multiple of 2^-44 has no share
    c = np.cumsum(wk)
    u = 0.0 if not u > 0 else u
    i = int((c <= u * c[-1]).sum())
    if i >= n:
        i = int(np.flatnonzero(wk > 0)[-1])
    return int(ids[i]), wk[i] / c[-1]
