"""The paged cache's operators in 64 bits on the CPU, sequence by sequence, and
batches to try them on."""
import math

import numpy as np
import torch

STEP = 1.0 / 16.0
CTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "q8": torch.float16}
CACHE = {"bf16": torch.bfloat16, "f16": torch.float16, "q8": torch.int8}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def to_cache(x, kind):
    if kind == "q8":
        return torch.clamp(torch.floor(x / STEP + 0.5), -128, 127).to(torch.int8)
    return x.to(CACHE[kind])


def value(x, step=STEP):
    """What a cache's or row's tensor holds, in 64 bits."""
    if x.dtype == torch.int8:
        return x.double() * step
    if x.dtype == torch.int16:
        return x.double() / 256.0
    return x.double()


class Batch:
    """Lengths, a shuffled page table and a pool of random values (CPU)."""

    def __init__(self, seed, nq, kv, kvh, hd, page, kind, pools=None, spare=2):
        self.rng = torch.Generator().manual_seed(seed)
        self.nq, self.kv, self.kvh, self.hd, self.page, self.kind = list(nq), list(kv), kvh, hd, page, kind
        self.qs = np.concatenate([[0], np.cumsum(nq)]).astype(int)
        self.ntok = int(self.qs[-1])
        need = [-(-max(n, 0) // page) for n in kv]
        self.pages = sum(need) + spare
        perm = torch.randperm(self.pages, generator=self.rng).to(torch.int32)
        self.table = torch.full((len(nq), max(need + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        self.k = to_cache(self.randn(self.pages, kvh, page, hd), kind)
        self.v = to_cache(self.randn(self.pages, kvh, page, hd), kind)

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.rng)

    def rows(self, b, t, h, count):
        """The first `count` positions of sequence b and head h of a pool t."""
        pg = self.table[b, :-(-count // self.page)].long()
        return t[pg, h].reshape(-1, self.hd)[:count]

    def device(self):
        i32 = torch.int32
        return (torch.tensor(self.qs, dtype=i32).cuda(), torch.tensor(self.kv, dtype=i32).cuda(), self.table.cuda())


def attend(b, q, heads, scale=None, window=0, k_step=STEP, v_step=STEP):
    """out, lse and the sum of |weight * value| of every row (float64)."""
    grp, hd = heads // b.kvh, b.hd
    scale = hd ** -0.5 if scale is None else scale
    out = torch.zeros(b.ntok, heads, hd, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.full((b.ntok, heads), -math.inf, dtype=torch.float64)
    err = torch.zeros(b.ntok, heads, dtype=torch.float64)
    for s, (n, m) in enumerate(zip(b.nq, b.kv)):
        for r in range(n):
            pos = m - n + r
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            for h in range(b.kvh):
                k = value(b.rows(s, b.k, h, pos + 1)[lo:], k_step)
                v = value(b.rows(s, b.v, h, pos + 1)[lo:], v_step)
                qh = q[b.qs[s] + r, h * grp:(h + 1) * grp].double()
                x = qh @ k.T * scale
                p = torch.softmax(x, 1)
                t = b.qs[s] + r
                sl = slice(h * grp, (h + 1) * grp)
                out[t, sl], mag[t, sl], lse[t, sl] = p @ v, p @ v.abs(), torch.logsumexp(x, 1)
                err[t, sl] = (qh.abs() @ k.abs().T * scale).amax(1)
    return out, lse, mag, err


def attn_bound(b, ctype, ref, mag, dots, out_kind=None):
    """How far a row may be from the definition: each weight rounded to the
    compute type (half a step of it), the sums in 32 bits, the output rounded
    once.  dots: the largest scale * sum |q_i k_i|: a score is off by at most
    (hd + 4) 2^-24 of it (products exact, hd additions, the scale), doubled
    for the exponent's own rounding (its argument times log2 e: 2^-23 of the
    score, and 2^-22 of the value)."""
    n = max(b.kv + [1])
    half = HALF_STEP[ctype]
    e_s = dots[..., None] * (b.hd + 8) * 2.0 ** -22 + 2.0 ** -21
    bound = half * mag + (2 * e_s + 2 * n * 2.0 ** -24) * mag
    if ctype == torch.float16:  # weights below 2^-14 round to 2^-25 at most
        bound = bound + n * 2.0 ** -25 * float(value(b.v).nan_to_num(0, 0, 0).abs().max())
    if out_kind == "q16":
        return bound + 0.5 / 256 * (1 + 2.0 ** -10)
    return bound + half * (ref.abs() + bound) + (2.0 ** -25 if ctype == torch.float16 else 0)


def append(b, x, heads, cos=None, sin=None, half=True, qn=None, kn=None, eps=1e-5):
    """(q, K, V) of every row before their rounding (float64), and a scale of
    the 32-bit arithmetic's error for q and K."""
    hd, kvh = b.hd, b.kvh
    x = value(x).view(b.ntok, heads + 2 * kvh, hd)
    qk, v = x[:, :heads + kvh].clone(), x[:, heads + kvh:]
    if qn is not None:
        w = torch.cat([qn.expand(heads, hd), kn.expand(kvh, hd)]).double()
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + eps) * w
    mag = qk.abs()
    if cos is not None:
        rot = 2 * cos.shape[1]
        for s, (n, m) in enumerate(zip(b.nq, b.kv)):
            for r in range(n):
                pos, t = m - n + r, b.qs[s] + r
                if pos < 0:
                    continue
                c, sn = cos[pos].double(), sin[pos].double()
                i = torch.arange(rot // 2)
                a, d = (i, i + rot // 2) if half else (2 * i, 2 * i + 1)
                y = qk[t].clone()
                qk[t, :, a] = y[:, a] * c - y[:, d] * sn
                qk[t, :, d] = y[:, d] * c + y[:, a] * sn
                mag[t, :, a] = (y[:, a] * c).abs() + (y[:, d] * sn).abs()
                mag[t, :, d] = (y[:, d] * c).abs() + (y[:, a] * sn).abs()
    return qk[:, :heads], qk[:, heads:], v, mag
