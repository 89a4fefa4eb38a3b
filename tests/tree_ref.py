"""Drafted trees and sampling in 64 bits on the CPU, row by row."""
import math
import random

import torch

import paged_ref as ref


def random_tree(n, seed, wide=False):
    """Parents of n rows: any earlier row, or (wide) the first ones more often."""
    rng = random.Random(seed)
    return [-1] + [rng.randint(0, (i - 1) // 4 if wide else i - 1) for i in range(1, n)] if n else []


def lines(parents, window=0):
    """(depths, the rows each row sees) of one sequence's tree."""
    depth, see = [], []
    for i, p in enumerate(parents):
        ok = 0 <= p < i
        depth.append(depth[p] + 1 if ok else 0)
        see.append((see[p] if ok else []) + [i])
    if window:
        see = [s[-window:] for s in see]
    return depth, see


def masks(rows, words):
    """Lists of rows as words of 64 bits (int64, as torch holds them)."""
    out = torch.zeros(len(rows), words, dtype=torch.int64)
    for i, s in enumerate(rows):
        for j in s:
            bit = 1 << (j & 63)
            out[i, j >> 6] |= bit - (1 << 64) if bit >> 63 else bit
    return out


def attend(b, q, heads, depth, see, scale=None, window=0, k_step=ref.STEP, v_step=ref.STEP):
    """paged_ref.attend over trees: depth and see (lists of rows) by row of the batch."""
    grp, hd = heads // b.kvh, b.hd
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(b.ntok, heads, hd, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((b.ntok, heads), -math.inf, dtype=torch.float64)
    err = torch.zeros(b.ntok, heads, dtype=torch.float64)
    for s, (n, m) in enumerate(zip(b.nq, b.kv)):
        base = m - n
        for r in range(n):
            t = int(b.qs[s]) + r
            lo = max(0, base + depth[t] - window + 1) if window else 0
            at = list(range(lo, max(base, 0))) + [base + j for j in sorted(set(see[t])) if 0 <= j < n and base + j >= 0]
            if not at:
                continue
            at = torch.tensor(at)
            for h in range(b.kvh):
                k = ref.value(b.rows(s, b.k, h, m)[at], k_step)
                v = ref.value(b.rows(s, b.v, h, m)[at], v_step)
                qh = q[t, h * grp:(h + 1) * grp].double()
                x = qh @ k.T * scale
                p = torch.softmax(x, 1)
                sl = slice(h * grp, (h + 1) * grp)
                out[t, sl], mag[t, sl], lse[t, sl] = p @ v, p @ v.abs(), torch.logsumexp(x, 1)
                err[t, sl] = (qh.abs() @ k.abs().T * scale).amax(1)
    return out, lse, mag, err


def accept(parents, tokens, chosen):
    """(path, next) of one sequence."""
    if not parents:
        return [], -1
    at, path = 0, [0]
    while True:
        fit = [j for j in range(at + 1, len(parents)) if parents[j] == at and tokens[j] == chosen[at]]
        if not fit:
            return path, chosen[at]
        at = fit[0]
        path.append(at)


FLT_MAX = torch.finfo(torch.float32).max


def sample(x, u, temp=None, top_k=None, top_p=None, min_p=None):
    """(token, kept, prob) of one row."""
    x = x.double() / (256.0 if x.dtype == torch.int16 else 1.0)
    x = torch.where(x.isnan(), -math.inf, x.clamp(max=FLT_MAX))
    m = float(x.max())
    if m == -math.inf:
        return -1, 0, 0.0
    if temp is not None and not temp > 0:
        return int((x == m).nonzero()[0]), 1, 1.0
    t = 1.0 if temp is None else max(float(temp), 1e-30)
    order = torch.sort(x, descending=True, stable=True)[1]
    order = order[x[order] > -math.inf]
    w = torch.exp((x[order] - m) / t)
    n = len(order)
    if top_k is not None and top_k > 0:
        n = min(n, top_k)
    if top_p is not None and top_p < 1:
        c = w[:n].cumsum(0)
        n = max(1, int((c - w[:n] < float(top_p) * float(c[-1])).sum()))
    if min_p is not None and min_p > 0:
        n = max(1, min(n, int((w >= min(float(min_p), 1.0)).sum())))
    ids = order[:n].sort()[0]
    y = torch.exp((x[ids] - m) / t)
    c = y.cumsum(0)
    hit = (c > float(u) * float(c[-1])).nonzero()
    i = int(hit[0]) if len(hit) else int(y.nonzero()[-1])
    return int(ids[i]), n, float(y[i] / c[-1])
