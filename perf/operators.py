"""The measured work of a ragged batch over a paged KV cache: append, attend, verify.

A server's step over sequences of different lengths: the projections' q, K and
V rows of every new token are normed, rotated and written into cache pages
(append), the new tokens attend to their sequences' pages (attn), and drafted
tokens are checked against the target's logits (verify).  Head layouts are
MiniMind3-64M's (8 query / 4 KV heads of 96), the LFM2.5-230M-shaped hybrid's
(16 / 8 of 64), the 0.5B ternary body's (16 / 2 of 64) and a generic 32 / 8 of
128; vocabularies are those models' 6400, 64402 and 73448 rows.

A batch is three device arrays: qstart (each sequence's first row, and the
end), kvlen (each sequence's length with its new tokens) and the page table.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-5
STEP = 1.0 / 16.0  # the q8 cache's grid
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "q16": torch.int16, "q8": torch.int8}
HEADS = {"minimind3": (8, 4, 96), "lfm2": (16, 8, 64), "bitcpm": (16, 2, 64), "wide": (32, 8, 128)}
VOCAB = (6400, 64402, 73448)


def listed():
    return [
        # one decoded token's q/K norm, rotation and cache write: the smallest call of a step
        dict(name="append_token", op="append", model="minimind3", cache="bf16", act="q16", page=16, norm=True,
             half=True, nseq=1, q_lo=1, q_hi=1, kv_lo=700, kv_hi=700, lens=1),
        # a decode step of 48 sequences into an 8-bit cache
        dict(name="append_step_q8", op="append", model="bitcpm", cache="q8", act="q16", page=32, norm=False,
             half=True, nseq=48, q_lo=1, q_hi=1, kv_lo=20, kv_hi=800, lens=2),
        # the prompts of six requests at once
        dict(name="append_prompts", op="append", model="wide", cache="bf16", act="bf16", page=64, norm=True,
             half=False, nseq=6, q_lo=300, q_hi=2048, kv_lo=300, kv_hi=6000, lens=3),
        # one token of one conversation
        dict(name="attn_token", op="attn", model="minimind3", cache="bf16", page=16, window=0, lse=False,
             nseq=1, q_lo=1, q_hi=1, kv_lo=700, kv_hi=700, lens=4),
        # one token at the end of a long document
        dict(name="attn_token_long", op="attn", model="wide", cache="bf16", page=64, window=0, lse=False,
             nseq=1, q_lo=1, q_hi=1, kv_lo=130001, kv_hi=130001, lens=5),
        # a decode step of a full server: lengths from short to long, 8-bit pages
        dict(name="attn_step_q8", op="attn", model="wide", cache="q8", page=32, window=0, lse=False,
             nseq=64, q_lo=1, q_hi=1, kv_lo=200, kv_hi=16000, lens=6),
        # the target's pass over drafted tokens
        dict(name="attn_drafts", op="attn", model="bitcpm", cache="f16", page=16, window=0, lse=True,
             nseq=24, q_lo=1, q_hi=6, kv_lo=500, kv_hi=8000, lens=7),
        # a long prompt's second half over its first
        dict(name="attn_prompt", op="attn", model="wide", cache="bf16", page=64, window=0, lse=False,
             nseq=1, q_lo=4000, q_hi=4000, kv_lo=8100, kv_hi=8100, lens=8),
        # prompts, short turns and single tokens in one batch, under a sliding window
        dict(name="attn_mixed", op="attn", model="lfm2", cache="f16", page=16, window=1024, lse=False,
             nseq=20, q_lo=1, q_hi=700, kv_lo=60, kv_hi=4096, lens=9),
        # four proposed tokens of one conversation, no draft model (looked up in its text)
        dict(name="verify_one", op="verify", vocab=6400, logits="q16", draft=False, nseq=1, r_lo=5, r_hi=5, lens=10),
        # a draft model's tokens, its logits kept
        dict(name="verify_draft", op="verify", vocab=73448, logits="f32", draft=True, nseq=32, r_lo=1, r_hi=6,
             lens=11),
        # a full server's step, looked-up drafts of many lengths, some sequences greedy
        dict(name="verify_step", op="verify", vocab=64402, logits="q16", draft=False, nseq=128, r_lo=1, r_hi=9,
             lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "verify"])
    lens = rng.randrange(1 << 30)
    model = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 64, 128])
    if op == "verify":
        nseq = _log(rng, 1, 96)
        r_hi = _log(rng, 1, 9)
        kind = rng.choice(["q16", "f32", "bf16", "f16"])
        return dict(op=op, vocab=rng.choice(VOCAB + (_log(rng, 100, 73000),)), logits=kind,
                    draft=rng.random() < 0.4, nseq=nseq, r_lo=rng.randint(1, r_hi), r_hi=r_hi, lens=lens)
    if op == "append":
        nseq = _log(rng, 1, 64)
        q_hi = _log(rng, 1, 8192 // nseq)
        kv_hi = max(q_hi, _log(rng, 20, 8000))
        return dict(op=op, model=model, cache=rng.choice(["bf16", "f16", "q8"]),
                    act=rng.choice(["q16", "bf16", "f16", "f32"]), page=page, norm=rng.random() < 0.6,
                    half=rng.random() < 0.6, nseq=nseq, q_lo=rng.randint(1, q_hi), q_hi=q_hi,
                    kv_lo=rng.randint(1, kv_hi), kv_hi=kv_hi, lens=lens)
    shape = rng.choice(["token", "step", "drafts", "prompt", "mixed"])
    if shape == "token":
        nseq, q_hi, kv_hi = 1, 1, _log(rng, 1, 130000)
    elif shape == "step":
        nseq = _log(rng, 2, 64)
        q_hi, kv_hi = 1, _log(rng, 20, 16000)
    elif shape == "drafts":
        nseq = _log(rng, 1, 48)
        q_hi, kv_hi = rng.randint(2, 9), _log(rng, 50, 12000)
    elif shape == "prompt":
        nseq, q_hi = 1, _log(rng, 16, 3800)
        kv_hi = q_hi + rng.choice([0, rng.randint(1, 4000)])
    else:
        nseq = rng.randint(2, 24)
        q_hi, kv_hi = _log(rng, 16, 700), _log(rng, 16, 4096)
    kv_hi = max(kv_hi, q_hi)
    kv_lo = kv_hi if nseq == 1 else rng.randint(1, kv_hi)
    return dict(op="attn", model=model, cache=rng.choice(["bf16", "f16", "q8"]), page=page,
                window=rng.choice([0, 0, _log(rng, 16, 4096)]), lse=rng.random() < 0.3, nseq=nseq,
                q_lo=q_hi if shape in ("token", "step", "prompt") else 1, q_hi=q_hi, kv_lo=kv_lo, kv_hi=kv_hi,
                lens=lens)


# ---- inputs ------------------------------------------------------------------

def _lengths(c):
    """Each sequence's new rows and, for the cache's operators, its length with them."""
    rng = random.Random(c["lens"])
    if c["op"] == "verify":
        return [rng.randint(c["r_lo"], c["r_hi"]) for _ in range(c["nseq"])], None
    nq = [_log(rng, c["q_lo"], c["q_hi"]) for _ in range(c["nseq"])]
    kv = [max(n, _log(rng, c["kv_lo"], c["kv_hi"])) for n in nq]
    return nq, kv


def _starts(nq):
    out = [0]
    for n in nq:
        out.append(out[-1] + n)
    return out


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _rand(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _as(x, kind):
    """f32 values in a type: q16 is the activations' grid of 1/256, q8 the cache's of 1/16."""
    if kind == "q16":
        return torch.clamp(torch.round(x * 256.0), -32768, 32767).to(torch.int16)
    if kind == "q8":
        return torch.clamp(torch.floor(x / STEP + 0.5), -128, 127).to(torch.int8)
    return x.to(TYPES[kind])


def _compute_type(cache):
    return torch.bfloat16 if cache == "bf16" else torch.float16


def _gpu():
    """The program's one context of the library."""
    if not _HANDLE:
        sys.path.insert(0, os.path.join(os.getcwd(), "vc4-gles2-inference_amd"))
        from vgx import gpu as vgpu
        _HANDLE.append(vgpu.GPU(0))
    return _HANDLE[0]


_HANDLE = []


def prepare(case, seed):
    g = _gen(seed)
    nq, kv = _lengths(case)
    s = dict(op=case["op"], nq=nq, qstart=_ints(_starts(nq)))
    if case["op"] == "verify":
        return _prepare_verify(s, case, g)
    heads, kvh, hd = HEADS[case["model"]]
    page, ntok, nseq = case["page"], sum(nq), case["nseq"]
    need = [-(-n // page) for n in kv]
    total = sum(need) + 3
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32).cpu()
    table = torch.full((nseq, max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    # what earlier steps wrote, stale values behind the sequences' ends included
    k = _as(_rand(g, total, kvh, page, hd), case["cache"])
    v = _as(_rand(g, total, kvh, page, hd), case["cache"])
    s.update(heads=heads, kvh=kvh, hd=hd, page=page, kv=kv, kvlen=_ints(kv), table=table.cuda(), k=k, v=v,
             cache=case["cache"], ctype=_compute_type(case["cache"]), max_q=max(nq), max_kv=max(kv), ntok=ntok)
    if case["op"] == "append":
        # projections' rows: q, then K, then V of every head
        s["qkv"] = _as(_rand(g, ntok, (heads + 2 * kvh) * hd) * 1.5, case["act"])
        s["act"] = case["act"]
        ang = (torch.arange(max(kv), dtype=torch.float64, device="cuda")[:, None]
               * 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd))
        s["cos"], s["sin"] = torch.cos(ang).float(), torch.sin(ang).float()
        s["half"] = case["half"]
        s["qn"] = 1.0 + 0.2 * _rand(g, hd) if case["norm"] else None
        s["kn"] = 1.0 + 0.2 * _rand(g, hd) if case["norm"] else None
    else:
        s["q"] = (2.0 * _rand(g, ntok, heads, hd)).to(s["ctype"])  # scores of spread 2
        s["window"], s["lse"] = case["window"], case["lse"]
    if own:
        s["pc"] = _gpu().paged_cache(heads=heads, kv_heads=kvh, head_dim=hd, kind=case["cache"], k=k, v=v)
        s["pb"] = s["pc"].batch(s["qstart"], s["kvlen"], s["table"], ntok, max_q=s["max_q"], max_kv=s["max_kv"])
    return s


def _prepare_verify(s, c, g):
    rows, vocab = sum(s["nq"]), c["vocab"]
    draft = 2.5 * _rand(g, rows, vocab)
    pick = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    draft[torch.arange(rows, device="cuda"), pick] += 14.0  # a next token that the text suggests
    target = draft + 0.4 * _rand(g, rows, vocab)
    gum = -torch.log(-torch.log(torch.rand(rows, vocab, device="cuda", generator=g).clamp(1e-12, 1 - 1e-7)))
    chosen = torch.argmax(draft + gum, 1)
    s["tokens"] = torch.roll(chosen, 1).to(torch.int32)  # tokens[r + 1] was drafted from row r
    s["logits"] = _as(target, c["logits"])
    s["draft"] = _as(draft, c["logits"]) if c["draft"] else None
    s["kind"] = c["logits"]
    rng = random.Random(c["lens"] + 1)
    temp = [0.0 if rng.random() < 0.15 and c["nseq"] > 1 else rng.uniform(0.5, 1.3) for _ in s["nq"]]
    s["temp"] = torch.tensor(temp, dtype=torch.float32).cuda()
    s["ua"] = torch.rand(rows, device="cuda", generator=g)
    s["us"] = torch.rand(len(s["nq"]), device="cuda", generator=g)
    if own:
        s["g"] = _gpu()
    return s


# ---- one pass ------------------------------------------------------------------

def run(s):
    if s["op"] == "append":
        q = s["pc"].append(s["pb"], s["qkv"], cos=s["cos"], sin=s["sin"], rope_half=s["half"], q_norm=s["qn"],
                           k_norm=s["kn"], eps=EPS) if own else _plain_append(s)
        return dict(q=q, k=_held(s["k"]), v=_held(s["v"]))
    if s["op"] == "attn":
        o, lse = s["pc"].attend(s["pb"], s["q"], window=s["window"], lse=s["lse"]) if own else _plain_attn(s)
        return dict(out=o, lse=lse) if s["lse"] else dict(out=o)
    if own:
        n, t, p = s["g"].draft_verify(s["qstart"], s["tokens"], s["logits"], s["ua"], s["us"], draft=s["draft"],
                                      temp=s["temp"])
    else:
        n, t, p = _plain_verify(s)
    return dict(accepted=n, next=t, prob=p)


def _held(x):
    """A q8 page's values (level / 16 is a bfloat16)."""
    return x.to(torch.bfloat16) * STEP if x.dtype == torch.int8 else x


def _value(x, kind):
    return x.float() / 256.0 if kind == "q16" else x.float()


def _row_seq(s):
    """Of every row: its sequence, its place among the sequence's rows, and their number."""
    qs = s["qstart"].long()
    row = torch.arange(int(sum(s["nq"])), device="cuda")
    seq = torch.searchsorted(qs[1:].contiguous(), row, right=True)
    return seq, row - qs[seq], qs[seq + 1] - qs[seq]


def _plain_append(s):
    heads, kvh, hd = s["heads"], s["kvh"], s["hd"]
    x = _value(s["qkv"], s["act"]).view(-1, heads + 2 * kvh, hd)
    seq, i, n = _row_seq(s)
    pos = s["kvlen"].long()[seq] - n + i
    qk, v = x[:, :heads + kvh], x[:, heads + kvh:]
    if s["qn"] is not None:
        w = torch.cat([s["qn"].expand(heads, hd), s["kn"].expand(kvh, hd)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    if s["half"]:
        a, b = qk[..., :hd // 2], qk[..., hd // 2:]
        qk = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    else:
        a, b = qk[..., 0::2], qk[..., 1::2]
        qk = torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)
    pg = s["table"][seq, pos // s["page"]].long()
    s["k"][pg, :, pos % s["page"]] = _as(qk[:, heads:], s["cache"])
    s["v"][pg, :, pos % s["page"]] = _as(v, s["cache"])
    return qk[:, :heads].to(s["ctype"])


def _plain_attn(s):
    heads, kvh, hd, page = s["heads"], s["kvh"], s["hd"], s["page"]
    grp, nseq, mq = heads // kvh, len(s["nq"]), s["max_q"]
    npg = -(-s["max_kv"] // page)
    tab = s["table"][:, :npg].long().clamp(min=0)
    unit = STEP if s["cache"] == "q8" else 1.0
    k = s["k"][tab].transpose(1, 2).reshape(nseq, kvh, npg * page, hd).float() * unit
    v = s["v"][tab].transpose(1, 2).reshape(nseq, kvh, npg * page, hd).float() * unit
    seq, i, n = _row_seq(s)
    q = torch.zeros(nseq, mq, heads, hd, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(nseq, mq, kvh, grp, hd).permute(0, 2, 3, 1, 4).reshape(nseq, kvh, grp * mq, hd)
    pos = (s["kvlen"] - (s["qstart"][1:] - s["qstart"][:-1])).long()[:, None] + torch.arange(mq, device="cuda")
    j = torch.arange(npg * page, device="cuda")
    see = (j <= pos[..., None]) & (j < s["kvlen"].long()[:, None, None])
    if s["window"]:
        see &= j > pos[..., None] - s["window"]
    v = torch.where((j < s["kvlen"].long()[:, None])[:, None, :, None], v, 0.0)
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    x = torch.where(see[:, None, None], x.view(nseq, kvh, grp, mq, -1), -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nseq, kvh, grp * mq, -1), v).view(nseq, kvh, grp, mq, hd)
    o = torch.where(z > 0, o / z, 0.0)
    lse = (m + torch.log(z))[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(nseq, mq, heads * hd)[seq, i].to(s["ctype"])
    return o, lse.permute(0, 3, 1, 2).reshape(nseq, mq, heads)[seq, i]


def _plain_verify(s):
    qs = s["qstart"].long()
    seq, i, n = _row_seq(s)
    rows, vocab = s["logits"].shape
    temp = s["temp"].double()
    greedy = temp <= 0
    inv = (1.0 / torch.where(greedy, 1.0, temp))[seq, None]
    x = _value(s["logits"], s["kind"])
    top = x.argmax(1)  # (equal maxima: set to the lowest index below)
    top = torch.where(x == x.gather(1, top[:, None]), torch.arange(vocab, device="cuda"), vocab).amin(1)
    # (probabilities and their sums in 64 bits: a draw next to a border)
    p = torch.softmax(x.double() * inv, 1)
    drafted = i + 1 < n
    tok = torch.roll(s["tokens"], -1).long()
    q = torch.softmax(_value(s["draft"], s["kind"]).double() * inv, 1) if s["draft"] is not None else None
    at = lambda t: t.gather(1, tok[:, None])[:, 0]  # noqa: E731
    sure = (tok == top).double()
    prob = torch.where(drafted, torch.where(greedy[seq], sure, at(p)), 0.0)
    ok = s["ua"].double() * (at(q) if q is not None else 1.0) < at(p)
    ok = torch.where(greedy[seq], sure > 0, ok) & drafted
    # the sequence's first row that is refused or has no draft left
    took = torch.where(ok, n, i)
    acc = torch.full((len(s["nq"]),), vocab + rows, device="cuda").scatter_reduce(0, seq, took, "amin")
    r = qs[:-1] + acc
    refused = (acc + 1 < qs[1:] - qs[:-1])[:, None]
    if q is not None:
        less = q[r]
    else:
        less = (tok[r][:, None] == torch.arange(vocab, device="cuda")).double()
    w = torch.where(refused, (p[r] - less).clamp(min=0), p[r])
    sums = torch.cumsum(w, 1)
    nxt = (sums <= s["us"].double()[:, None] * sums[:, -1:]).sum(1).clamp(max=vocab - 1)
    nxt = torch.where(greedy, top[r], nxt)
    return acc.to(torch.int32), nxt.to(torch.int32), prob.float()


# ---- what one pass cannot do without ---------------------------------------------

def _seen(c, nq, kv):
    """Keys that some row of the sequence sees, and the visible (row, key) pairs."""
    w = c["window"] or 1 << 60
    lo = max(0, kv - nq + 1 - w)
    # row at position p sees min(p + 1, w) keys
    p0, p1 = kv - nq + 1, kv
    full = max(0, min(p1, w) - p0 + 1)
    pairs = full * (2 * p0 + full - 1) // 2 + (nq - full) * min(w, p1)
    return kv - lo, pairs


def work(case):
    nq, kv = _lengths(case)
    size = {"f32": 4, "bf16": 2, "f16": 2, "q16": 2, "q8": 1}
    if case["op"] == "verify":
        rows = sum(nq)
        return dict(bytes=rows * case["vocab"] * size[case["logits"]] * (2 if case["draft"] else 1) + 12 * rows
                    + 20 * len(nq), flops=0)
    heads, kvh, hd = HEADS[case["model"]]
    ntok = sum(nq)
    if case["op"] == "append":
        at = set()
        for n, m in zip(nq, kv):
            at.update(range(m - n, m))
        return dict(bytes=ntok * (heads + 2 * kvh) * hd * size[case["act"]] + 2 * ntok * heads * hd
                    + 2 * ntok * kvh * hd * size[case["cache"]] + len(at) * hd * 4, flops=0)
    keys = pairs = 0
    for n, m in zip(nq, kv):
        a, b = _seen(case, n, m)
        keys, pairs = keys + a, pairs + b
    return dict(bytes=2 * keys * kvh * hd * size[case["cache"]] + 4 * ntok * heads * hd
                + (4 * ntok * heads if case["lse"] else 0), flops=4 * hd * heads * pairs)


# ---- the definitions in 64 bits, sequence by sequence ---------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "verify": _exact_verify}[case["op"]](s)


def _exact_append(s):
    heads, kvh, hd, page = s["heads"], s["kvh"], s["hd"], s["page"]
    x = s["qkv"].double() / (256.0 if s["act"] == "q16" else 1.0)
    k, v = _held(s["k"]).double(), _held(s["v"]).double()
    qs, out = _starts(s["nq"]), []
    for b, (n, m) in enumerate(zip(s["nq"], s["kv"])):
        rows = x[qs[b]:qs[b] + n].view(n, -1, hd)
        parts = [rows[:, :heads], rows[:, heads:heads + kvh]]
        turn = torch.complex(s["cos"][m - n:m].double(), s["sin"][m - n:m].double())[:, None]
        for j, w in enumerate((s["qn"], s["kn"])):
            y = parts[j]
            if w is not None:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / hd + EPS) * w.double()
            if s["half"]:
                z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous()) * turn
                parts[j] = torch.cat([z.real, z.imag], -1)
            else:
                z = torch.view_as_complex(y.reshape(n, -1, hd // 2, 2).contiguous()) * turn
                parts[j] = torch.view_as_real(z).reshape(n, -1, hd)
        out.append(parts[0])
        where = torch.arange(m - n, m, device="cuda")
        pg = s["table"][b].long()[where // page]
        new = [parts[1], rows[:, heads + kvh:]]
        if s["cache"] == "q8":
            new = [torch.floor(y * 16.0 + 0.5).clamp(-128, 127) / 16.0 for y in new]
        k[pg, :, where % page] = new[0]
        v[pg, :, where % page] = new[1]
    return dict(q=torch.cat(out), k=k, v=v)


def _exact_attn(s):
    heads, kvh, hd, page = s["heads"], s["kvh"], s["hd"], s["page"]
    grp, qs = heads // kvh, _starts(s["nq"])
    unit = STEP if s["cache"] == "q8" else 1.0
    outs, sums = [], []
    for b, (n, m) in enumerate(zip(s["nq"], s["kv"])):
        pages = s["table"][b].long()[:-(-m // page)]
        q = s["q"][qs[b]:qs[b] + n].double()
        away = torch.arange(m - n, m, device="cuda")[:, None] - torch.arange(m, device="cuda")
        hide = away < 0
        if s["window"]:
            hide |= away >= s["window"]
        o, l = [], []
        for h in range(kvh):
            k = s["k"][pages, h].reshape(-1, hd)[:m].double() * unit
            v = s["v"][pages, h].reshape(-1, hd)[:m].double() * unit
            for u in range(grp):
                x = (q[:, h * grp + u] @ k.T * hd ** -0.5).masked_fill(hide, -math.inf)
                o.append(torch.softmax(x, 1) @ v)
                l.append(torch.logsumexp(x, 1))
        outs.append(torch.cat(o, 1))
        sums.append(torch.stack(l, 1))
    return dict(out=torch.cat(outs), lse=torch.cat(sums)) if s["lse"] else dict(out=torch.cat(outs))


def _exact_verify(s):
    qs, acc, nxt, prob = _starts(s["nq"]), [], [], []
    unit = 256.0 if s["kind"] == "q16" else 1.0
    tok, ua, us, temp = (s[k].cpu().tolist() for k in ("tokens", "ua", "us", "temp"))
    for b, n in enumerate(s["nq"]):
        x = s["logits"][qs[b]:qs[b] + n].double() / unit
        d = s["draft"][qs[b]:qs[b] + n].double() / unit if s["draft"] is not None else None
        best = [int((r == r.max()).nonzero()[0]) for r in x]
        t = temp[b]
        if t > 0:
            x = torch.exp((x - x.amax(1, keepdim=True)) / t)
            x = x / x.sum(1, keepdim=True)
            if d is not None:
                d = torch.exp((d - d.amax(1, keepdim=True)) / t)
                d = d / d.sum(1, keepdim=True)
        got, open_ = 0, True
        for i in range(n - 1):
            w = tok[qs[b] + i + 1]
            pr = float(x[i, w]) if t > 0 else float(w == best[i])
            prob.append(pr)
            against = ua[qs[b] + i] * (float(d[i, w]) if d is not None and t > 0 else 1.0)
            open_ = open_ and (against < pr)
            got += open_
        prob.append(0.0)
        acc.append(got)
        if t <= 0:
            nxt.append(best[got])
            continue
        w = x[got].clone()
        if got < n - 1 and d is not None:
            w = (w - d[got]).clamp(min=0)
        elif got < n - 1:
            w[tok[qs[b] + got + 1]] = 0
        sums = w.cumsum(0)
        nxt.append(int((sums > us[b] * float(sums[-1])).nonzero()[0]))
    return dict(accepted=_ints(acc), next=_ints(nxt), prob=torch.tensor(prob, dtype=torch.float64))
