"""The measured work of decoding over drafted trees: attend, sample, accept and keep, copy.

A server drafts a tree of tokens for each sequence and appends all its rows to
the paged cache.  The rows attend to their sequence and to their ancestors in
the tree (tree), every row's logits give a token (sample), the tree is walked
down as far as it holds those tokens and the rows of that path become the
sequence's next positions (keep).  Pages are copied where sequences fork or the
pool is compacted (copy).  Head layouts are MiniMind3-64M's (8 query / 4 KV
heads of 96), the LFM2.5-230M-shaped hybrid's (16 / 8 of 64), the 0.5B ternary
body's (16 / 2 of 64) and a generic 32 / 8 of 128; vocabularies are those
models' 6400, 64402 and 73448 rows.

A tree is each row's parent among its sequence's rows (-1: the first row, the
token that the sequence ended with); parents come before their children.
"""
import math
import os
import random
import sys

import torch

own = False

STEP = 1.0 / 16.0  # the q8 cache's grid
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "q16": torch.int16, "q8": torch.int8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "q16": 2, "q8": 1}
HEADS = {"minimind3": (8, 4, 96), "lfm2": (16, 8, 64), "bitcpm": (16, 2, 64), "wide": (32, 8, 128)}
VOCAB = (6400, 64402, 73448)


def listed():
    return [
        # one conversation, a small tree looked up in its text
        dict(name="tree_one", op="tree", model="minimind3", cache="bf16", page=16, window=0, lse=False, nseq=1,
             q_lo=8, q_hi=8, kv_lo=700, kv_hi=700, lens=1),
        # a server's step: trees of many sizes over lengths from short to long
        dict(name="tree_step", op="tree", model="lfm2", cache="f16", page=16, window=0, lse=True, nseq=24, q_lo=5,
             q_hi=61, kv_lo=300, kv_hi=8000, lens=2),
        # the same with 8-bit pages, few KV heads and a sliding window
        dict(name="tree_window_q8", op="tree", model="bitcpm", cache="q8", page=32, window=4096, lse=False, nseq=48,
             q_lo=9, q_hi=33, kv_lo=500, kv_hi=14000, lens=3),
        # a wide tree at the end of a long document
        dict(name="tree_long", op="tree", model="wide", cache="bf16", page=64, window=0, lse=False, nseq=2, q_lo=64,
             q_hi=64, kv_lo=60001, kv_hi=60001, lens=4),
        # the next token of one conversation
        dict(name="sample_one", op="sample", vocab=6400, logits="q16", rows=1, cut="k40p", lens=5),
        # a decode step of requests that each set their own cuts
        dict(name="sample_step", op="sample", vocab=73448, logits="f32", rows=48, cut="mix", lens=6),
        # a larger step, every request by top-p alone
        dict(name="sample_top_p", op="sample", vocab=64402, logits="bf16", rows=160, cut="p", lens=7),
        # every row of a step's trees
        dict(name="sample_trees", op="sample", vocab=64402, logits="q16", rows=640, cut="k", lens=8),
        # one conversation's tree walked, its path kept in every layer
        dict(name="keep_one", op="keep", model="minimind3", cache="bf16", page=16, layers=8, nseq=1, q_lo=12, q_hi=12,
             kv_lo=300, kv_hi=300, lens=9),
        # a server's step of trees in every layer
        dict(name="keep_step", op="keep", model="lfm2", cache="f16", page=16, layers=14, nseq=64, q_lo=5, q_hi=61,
             kv_lo=80, kv_hi=400, lens=10),
        # four conversations forked: their last pages, partly filled
        dict(name="copy_fork", op="copy", model="minimind3", cache="bf16", page=16, layers=8, pages=4, part=True,
             lens=11),
        # pages gathered into the front of a pool
        dict(name="copy_compact", op="copy", model="wide", cache="bf16", page=64, layers=8, pages=301, part=False,
             lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "sample", "sample", "keep", "copy"])
    lens = rng.randrange(1 << 30)
    model = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 64, 128])
    if op == "sample":
        return dict(op=op, vocab=rng.choice(VOCAB + (_log(rng, 100, 73000),)),
                    logits=rng.choice(["q16", "f32", "bf16", "f16"]), rows=_log(rng, 1, 280),
                    cut=rng.choice(["k", "p", "k40p", "m", "t", "mix"]), lens=lens)
    if op == "copy":
        pages = _log(rng, 1, 150)
        return dict(op=op, model=model, cache=rng.choice(["bf16", "f16"]), page=page, layers=rng.randint(1, 16),
                    pages=pages, part=rng.random() < 0.5, lens=lens)
    nseq = _log(rng, 1, 48)
    q_hi = _log(rng, 2, 64)
    if op == "keep":
        kv_hi = max(q_hi, _log(rng, 20, 400))
        return dict(op=op, model=model, cache=rng.choice(["bf16", "f16"]), page=page, layers=rng.randint(1, 16),
                    nseq=nseq, q_lo=rng.randint(1, q_hi), q_hi=q_hi, kv_lo=rng.randint(1, kv_hi), kv_hi=kv_hi,
                    lens=lens)
    kv_hi = max(q_hi, _log(rng, 50, 100000 if nseq < 4 else 8000))
    return dict(op=op, model=model, cache=rng.choice(["bf16", "f16", "q8"]), page=page,
                window=rng.choice([0, 0, _log(rng, 16, 4096)]), lse=rng.random() < 0.3, nseq=nseq,
                q_lo=rng.randint(1, q_hi), q_hi=q_hi, kv_lo=rng.randint(1, kv_hi), kv_hi=kv_hi, lens=lens)


# ---- inputs ------------------------------------------------------------------

def _lengths(c):
    """Each sequence's rows and its length with them."""
    rng = random.Random(c["lens"])
    nq = [_log(rng, c["q_lo"], c["q_hi"]) for _ in range(c["nseq"])]
    return nq, [max(n, _log(rng, c["kv_lo"], c["kv_hi"])) for n in nq]


def _starts(nq):
    out = [0]
    for n in nq:
        out.append(out[-1] + n)
    return out


def _parents(c, nq):
    """Each sequence's tree: any earlier row may be a row's parent.  Where a
    path is kept it is the tree's last rows (at most half of them), so that a
    second pass over the same pages finds the rows it moves as they were."""
    rng = random.Random(c["lens"] + 1)
    trees, paths = [], []
    for n in nq:
        d = rng.randint(0, min(6, (n - 1) // 2)) if c["op"] == "keep" else 0
        p = [-1] + [rng.randint(0, i - 1) for i in range(1, n - d)]
        chain = list(range(n - d, n))
        trees.append(p + ([0] + chain[:-1] if d else []))
        paths.append([0] + chain)
    return trees, paths


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
    if case["op"] == "sample":
        return _prepare_sample(case, g)
    heads, kvh, hd = HEADS[case["model"]]
    page, kind = case["page"], case["cache"]
    s = dict(op=case["op"], heads=heads, kvh=kvh, hd=hd, page=page, cache=kind)
    if case["op"] == "copy":
        return _prepare_copy(s, case, g)
    nq, kv = _lengths(case)
    trees, paths = _parents(case, nq)
    need = [-(-n // page) for n in kv]
    total, layers = sum(need) + 3, case.get("layers", 1)
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32).cpu()
    table = torch.full((len(nq), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    s.update(nq=nq, kv=kv, trees=trees, qstart=_ints(_starts(nq)), kvlen=_ints(kv), table=table.cuda(),
             parent=_ints(sum(trees, [])), max_q=max(nq), max_kv=max(kv), ntok=sum(nq),
             k=[_as(_rand(g, total, kvh, page, hd), kind) for _ in range(layers)],
             v=[_as(_rand(g, total, kvh, page, hd), kind) for _ in range(layers)])
    # the rows that each row sees (itself and its ancestors) and its depth: a step's
    # masks, made once for all layers
    see = torch.zeros(len(nq), s["max_q"], s["max_q"], dtype=torch.bool)
    depth = torch.zeros(len(nq), s["max_q"], dtype=torch.int64)
    for b, tree in enumerate(trees):
        for i, p in enumerate(tree):
            if p >= 0:
                see[b, i] = see[b, p]
                depth[b, i] = depth[b, p] + 1
            see[b, i, i] = True
    s["see"], s["depth"] = see.cuda(), depth.cuda()
    if case["op"] == "tree":
        s["ctype"] = torch.bfloat16 if kind == "bf16" else torch.float16
        s["q"] = (2.0 * _rand(g, s["ntok"], heads, hd)).to(s["ctype"])  # scores of spread 2
        s["window"], s["lse"] = case["window"], case["lse"]
    else:
        # drafted tokens, and the one that each row's logits gave: on the path its next row's
        tok = torch.randperm(32000, device="cuda", generator=g)[:s["ntok"]].to(torch.int32)
        chosen = torch.randint(32000, 64402, (s["ntok"],), device="cuda", generator=g).to(torch.int32)
        qs = _starts(nq)
        rows = torch.tensor([qs[b] + i for b, p in enumerate(paths) for i in p[:-1]], dtype=torch.int64).cuda()
        then = torch.tensor([qs[b] + i for b, p in enumerate(paths) for i in p[1:]], dtype=torch.int64).cuda()
        chosen[rows] = tok[then]
        s["tokens"], s["chosen"] = tok, chosen
    if own:
        gpu = _gpu()
        pcs = [gpu.paged_cache(heads=heads, kv_heads=kvh, head_dim=hd, kind=kind, k=k, v=v)
               for k, v in zip(s["k"], s["v"])]
        s["pc"], s["pl"] = pcs[0], gpu.paged_layers(pcs)
        s["pb"] = s["pc"].batch(s["qstart"], s["kvlen"], s["table"], s["ntok"], max_q=s["max_q"], max_kv=s["max_kv"])
        if case["op"] == "tree":
            s["pt"] = s["pb"].tree(s["parent"], window=s["window"])
    return s


def _prepare_copy(s, c, g):
    n, kind, total = c["pages"], c["cache"], 2 * c["pages"] + 3
    perm = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    s["src"], s["dst"] = perm[:n].contiguous(), perm[n:2 * n].contiguous()
    s["rows"] = torch.randint(1, c["page"] + 1, (n,), device="cuda", generator=g).to(torch.int32) if c["part"] else None
    s["k"], s["v"] = ([_as(_rand(g, total, s["kvh"], c["page"], s["hd"]), kind) for _ in range(c["layers"])]
                      for _ in range(2))
    if own:
        gpu = _gpu()
        s["pl"] = gpu.paged_layers([gpu.paged_cache(heads=s["heads"], kv_heads=s["kvh"], head_dim=s["hd"], kind=kind,
                                                    k=k, v=v) for k, v in zip(s["k"], s["v"])])
    return s


def _cuts(c):
    """Each row's temperature (0: greedy), top-k (0: all), top-p (1: all) and min-p (0: all)."""
    rng = random.Random(c["lens"] + 2)
    temp, top_k, top_p, min_p = [], [], [], []
    for _ in range(c["rows"]):
        cut = c["cut"] if c["cut"] != "mix" else rng.choice(["k", "p", "k40p", "m", "t", "p"])
        temp.append(0.0 if c["cut"] == "mix" and rng.random() < 0.1 else rng.uniform(0.5, 1.3))
        top_k.append({"k": rng.choice([1, 20, 50, 50, 100, 400]), "k40p": 40}.get(cut, 0))
        top_p.append(rng.choice([0.8, 0.9, 0.95, 0.95, 0.99]) if cut in ("p", "k40p") else 1.0)
        min_p.append(rng.choice([0.02, 0.05, 0.1]) if cut == "m" else 0.0)
    return temp, top_k, top_p, min_p


def _prepare_sample(c, g):
    rows, vocab = c["rows"], c["vocab"]
    x = 2.0 * _rand(g, rows, vocab)
    # the tokens that a text suggests, their weights falling as their rank does, from sure rows to open ones
    n = min(vocab, 64)
    at = torch.randint(0, vocab, (rows, n), device="cuda", generator=g)
    fall = 1.5 * torch.log(torch.arange(1, n + 1, dtype=torch.float32, device="cuda"))
    x.scatter_(1, at, 16.0 + 2.0 * _rand(g, rows, 1) - fall + 0.3 * _rand(g, rows, n))
    temp, top_k, top_p, min_p = _cuts(c)
    f = lambda v: torch.tensor(v, dtype=torch.float32).cuda()  # noqa: E731
    s = dict(op="sample", x=_as(x, c["logits"]), kind=c["logits"], u=torch.rand(rows, device="cuda", generator=g),
             temp=f(temp), top_k=_ints(top_k) if any(top_k) else None, top_p=f(top_p) if min(top_p) < 1 else None,
             min_p=f(min_p) if any(min_p) else None)
    if own:
        s["g"] = _gpu()
    return s


# ---- one pass ------------------------------------------------------------------

def run(s):
    if s["op"] == "tree":
        o, lse = s["pc"].attend(s["pb"], s["q"], window=s["window"], lse=s["lse"], tree=s["pt"]) if own \
            else _plain_tree(s)
        return dict(out=o, lse=lse) if s["lse"] else dict(out=o)
    if s["op"] == "sample":
        t, n, p = s["g"].sample(s["x"], s["u"], temp=s["temp"], top_k=s["top_k"], top_p=s["top_p"],
                                min_p=s["min_p"]) if own else _plain_sample(s)
        return dict(token=t, kept=n, prob=p)
    if s["op"] == "keep":
        if own:
            path, acc, nxt = s["pb"].accept(s["parent"], s["tokens"], s["chosen"])
            s["pl"].keep(s["pb"], path, acc)
        else:
            path, acc, nxt = _plain_keep(s)
        return dict(path=path, accepted=acc, next=nxt, k=s["k"], v=s["v"])
    if own:
        s["pl"].copy(s["src"], s["dst"], rows=s["rows"])
    else:
        _plain_copy(s)
    return dict(k=s["k"], v=s["v"])


def _row_seq(s):
    """Of every row: its sequence and its place among the sequence's rows."""
    qs = s["qstart"].long()
    row = torch.arange(s["ntok"], device="cuda")
    seq = torch.searchsorted(qs[1:].contiguous(), row, right=True)
    return seq, row - qs[seq]


def _plain_tree(s):
    heads, kvh, hd, page = s["heads"], s["kvh"], s["hd"], s["page"]
    grp, nseq, mq = heads // kvh, len(s["nq"]), s["max_q"]
    npg = -(-s["max_kv"] // page)
    tab = s["table"][:, :npg].long().clamp(min=0)
    unit = STEP if s["cache"] == "q8" else 1.0
    k = s["k"][0][tab].transpose(1, 2).reshape(nseq, kvh, npg * page, hd).float() * unit
    v = s["v"][0][tab].transpose(1, 2).reshape(nseq, kvh, npg * page, hd).float() * unit
    seq, i = _row_seq(s)
    q = torch.zeros(nseq, mq, heads, hd, device="cuda")
    q[seq, i] = s["q"].float()
    q = q.view(nseq, mq, kvh, grp, hd).permute(0, 2, 3, 1, 4).reshape(nseq, kvh, grp * mq, hd)
    base = (s["kvlen"] - (s["qstart"][1:] - s["qstart"][:-1])).long()[:, None, None]
    j = torch.arange(npg * page, device="cuda")
    t = (j - base).expand(nseq, mq, -1)  # a key's place among the rows
    see = (t < 0) | ((t < mq) & s["see"].gather(2, t.clamp(0, mq - 1)))
    if s["window"]:
        key = torch.where(t < 0, t, s["depth"][:, None].expand(nseq, mq, mq).gather(2, t.clamp(0, mq - 1)))
        see &= key > s["depth"][..., None] - s["window"]
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    x = torch.where(see[:, None, None], x.view(nseq, kvh, grp, mq, -1), -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nseq, kvh, grp * mq, -1), v).view(nseq, kvh, grp, mq, hd) / z
    lse = (m + torch.log(z))[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(nseq, mq, heads * hd)[seq, i].to(s["ctype"])
    return o, lse.permute(0, 3, 1, 2).reshape(nseq, mq, heads)[seq, i]


def _plain_sample(s):
    # (weights and sums in 64 bits: a draw or a cut next to a border)
    x = s["x"].double() / (256.0 if s["kind"] == "q16" else 1.0)
    rows, vocab = x.shape
    greedy = s["temp"] <= 0
    x, rank = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1.0, s["temp"].double())[:, None])
    place = torch.arange(vocab, device="cuda")
    keep = (place == 0) | ~greedy[:, None]
    if s["top_k"] is not None:
        keep &= (place < s["top_k"][:, None]) | (s["top_k"][:, None] <= 0)
        w = w * keep
    if s["top_p"] is not None:
        sums = torch.cumsum(w, 1)
        keep &= (s["top_p"][:, None] >= 1) | (sums - w < s["top_p"].double()[:, None] * sums[:, -1:])
        keep[:, 0] = True
    if s["min_p"] is not None:
        keep &= w >= s["min_p"].double()[:, None]
        keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, rank, w * keep)  # in the tokens' order again
    sums = torch.cumsum(w, 1)
    token = (sums <= s["u"].double()[:, None] * sums[:, -1:]).sum(1).clamp(max=vocab - 1)
    prob = w.gather(1, token[:, None])[:, 0] / sums[:, -1]
    return token.to(torch.int32), keep.sum(1).to(torch.int32), prob.float()


def _plain_keep(s):
    seq, i = _row_seq(s)
    qs, par = s["qstart"].long(), s["parent"].long()
    row = torch.arange(s["ntok"], device="cuda")
    fits = (par < 0) | (s["chosen"][(qs[seq] + par).clamp(min=0)] == s["tokens"])
    # on the path: a row that fits, as all its ancestors do
    good = torch.ones(s["see"].shape[:2], dtype=torch.bool, device="cuda")
    good[seq, i] = fits
    on = ~(s["see"] & ~good[:, None]).any(2)[seq, i]
    acc = torch.full((len(s["nq"]),), -1, device="cuda").index_add_(0, seq, on.long())
    depth = s["depth"][seq, i]
    path = torch.full((s["ntok"],), -1, dtype=torch.int32, device="cuda")
    path[(qs[seq] + depth)[on]] = i[on].to(torch.int32)
    nxt = s["chosen"][qs[:-1] + path[qs[:-1] + acc].long()]
    base = s["kvlen"].long()[seq] - (qs[1:] - qs[:-1])[seq]
    take = path >= 0
    frm, to = (base + path.long())[take], (base + row - qs[seq])[take]
    at = lambda p: (s["table"][seq[take], p // s["page"]].long(), p % s["page"])  # noqa: E731
    (fp, fs), (tp, ts) = at(frm), at(to)
    for x in s["k"] + s["v"]:  # (a layer's K or V: a tensor of its own)
        x[tp, :, ts] = x[fp, :, fs]
    return path, acc.to(torch.int32), nxt


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    if s["rows"] is not None:
        part = (torch.arange(s["page"], device="cuda") < s["rows"][:, None])[:, None, :, None]
    for x in s["k"] + s["v"]:
        x[dst] = x[src] if s["rows"] is None else torch.where(part, x[src], x[dst])


# ---- what one pass cannot do without ---------------------------------------------

def work(case):
    if case["op"] == "sample":
        return dict(bytes=case["rows"] * (case["vocab"] * SIZE[case["logits"]] + 32), flops=0)
    heads, kvh, hd = HEADS[case["model"]]
    size = SIZE[case["cache"]]
    if case["op"] == "copy":
        rng = case["pages"] * (case["page"] + 1) // 2 if case["part"] else case["pages"] * case["page"]
        return dict(bytes=4 * case["layers"] * rng * kvh * hd * size + 12 * case["pages"], flops=0)
    nq, kv = _lengths(case)
    trees, paths = _parents(case, nq)
    ntok = sum(nq)
    if case["op"] == "keep":
        moved = sum(i != k for p in paths for k, i in enumerate(p))
        return dict(bytes=4 * case["layers"] * moved * kvh * hd * size + 16 * ntok, flops=0)
    w, keys, pairs = case["window"] or 1 << 60, 0, 0
    for n, m, tree in zip(nq, kv, trees):
        depth = []
        for p in tree:
            depth.append(depth[p] + 1 if p >= 0 else 0)
        keys += n + min(m - n, w - 1)
        pairs += sum(min(m - n + d + 1, w) for d in depth)
    return dict(bytes=2 * keys * kvh * hd * size + 4 * ntok * heads * hd + (4 * ntok * heads if case["lse"] else 0),
                flops=4 * hd * heads * pairs)


# ---- the definitions in 64 bits, sequence by sequence ---------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "sample": _exact_sample, "keep": _exact_keep, "copy": _exact_copy}[case["op"]](s)


def _exact_tree(s):
    heads, kvh, hd, page = s["heads"], s["kvh"], s["hd"], s["page"]
    grp, qs = heads // kvh, _starts(s["nq"])
    unit = STEP if s["cache"] == "q8" else 1.0
    outs, sums = [], []
    for b, (n, m) in enumerate(zip(s["nq"], s["kv"])):
        pages = s["table"][b].long()[:-(-m // page)]
        q = s["q"][qs[b]:qs[b] + n].double()
        hide = torch.zeros(n, m, dtype=torch.bool)
        hide[:, m - n:] = True
        lines = []
        for i, p in enumerate(s["trees"][b]):
            lines.append((lines[p] if p >= 0 else []) + [i])  # from the first row down
            hide[i, [m - n + t for t in lines[i]]] = False
            if s["window"]:
                far = len(lines[i]) - s["window"]  # of the line's rows, those behind the window
                hide[i, [m - n + t for t in lines[i][:max(far, 0)]]] = True
                hide[i, :min(max(m - n + far, 0), m - n)] = True
        hide = hide.cuda()
        o, l = [], []
        for h in range(kvh):
            k = s["k"][0][pages, h].reshape(-1, hd)[:m].double() * unit
            v = s["v"][0][pages, h].reshape(-1, hd)[:m].double() * unit
            for u in range(grp):
                x = (q[:, h * grp + u] @ k.T * hd ** -0.5).masked_fill(hide, -math.inf)
                o.append(torch.softmax(x, 1) @ v)
                l.append(torch.logsumexp(x, 1))
        outs.append(torch.cat(o, 1))
        sums.append(torch.stack(l, 1))
    return dict(out=torch.cat(outs), lse=torch.cat(sums)) if s["lse"] else dict(out=torch.cat(outs))


def _exact_sample(s):
    token, kept, prob = [], [], []
    lists = [s[k].cpu().tolist() if s[k] is not None else None for k in ("u", "temp", "top_k", "top_p", "min_p")]
    for r in range(s["x"].shape[0]):
        u, t, k, p, mp = (v[r] if v is not None else None for v in lists)
        x = s["x"][r].double() / (256.0 if s["kind"] == "q16" else 1.0)
        if t <= 0:
            token.append(int((x == x.max()).nonzero()[0]))
            kept.append(1)
            prob.append(1.0)
            continue
        # by value, then by the lower token: the flipped row's ascending stable sort, read backwards
        order = x.numel() - 1 - torch.sort(x.flip(0), stable=True)[1].flip(0)
        w = torch.exp(x[order] / t - x.max() / t)
        n = min(k, len(w)) if k else len(w)
        if p is not None and p < 1:
            before = torch.cat([w.new_zeros(1), w[:n].cumsum(0)])
            n = int((before[:-1] < p * before[-1]).sum())
        if mp:
            n = min(n, int((w >= mp).sum()))
        n = max(n, 1)
        ids = order[:n].sort()[0]
        y = torch.exp((x[ids] - x.max()) / t)
        c = y.cumsum(0)
        i = int((c > u * float(c[-1])).nonzero()[0])
        token.append(int(ids[i]))
        kept.append(n)
        prob.append(float(y[i] / c[-1]))
    return dict(token=_ints(token), kept=_ints(kept), prob=torch.tensor(prob, dtype=torch.float64))


def _exact_keep(s):
    qs, page = _starts(s["nq"]), s["page"]
    tok, chosen, table = (s[k].cpu().tolist() for k in ("tokens", "chosen", "table"))
    path, acc, nxt, moves = [-1] * s["ntok"], [], [], []
    for b, n in enumerate(s["nq"]):
        at, line = 0, [0]
        while True:
            fit = [i for i in range(at + 1, n) if s["trees"][b][i] == at and tok[qs[b] + i] == chosen[qs[b] + at]]
            if not fit:
                break
            at = fit[0]
            line.append(at)
        path[qs[b]:qs[b] + len(line)] = line
        acc.append(len(line) - 1)
        nxt.append(chosen[qs[b] + at])
        base = s["kv"][b] - n
        moves += [(table[b][(base + i) // page], (base + i) % page, table[b][(base + k) // page], (base + k) % page)
                  for k, i in enumerate(line)]
    fp, fs, tp, ts = (torch.tensor(v).cuda() for v in zip(*moves))
    out = []
    for x in s["k"] + s["v"]:
        y = x.double()
        y[tp, :, ts] = x[fp, :, fs].double()
        out.append(y)
    return dict(path=_ints(path), accepted=_ints(acc), next=_ints(nxt), k=out[:len(s["k"])], v=out[len(s["k"]):])


def _exact_copy(s):
    rows = s["rows"].cpu().tolist() if s["rows"] is not None else [s["page"]] * s["src"].numel()
    out = []
    for x in s["k"] + s["v"]:
        y = x.double()
        for a, b, n in zip(s["src"].cpu().tolist(), s["dst"].cpu().tolist(), rows):
            y[b, :, :n] = x[a, :, :n].double()
        out.append(y)
    return dict(k=out[:len(s["k"])], v=out[len(s["k"]):])
