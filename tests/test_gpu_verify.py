"""vgx_draft_verify against its definition in 64 bits, and what it refuses."""
import ctypes
import math

import pytest
import torch

from vgx import lib as vl

FLT_MAX = torch.finfo(torch.float32).max


def expect(qs, tokens, logits, ua, un, draft=None, temp=None):
    """The definition, row by row in float64 on the CPU."""
    acc, nxt, prob = [], [], [0.0] * len(tokens)

    def val(t):
        x = t.double() / (256.0 if t.dtype == torch.int16 else 1.0)
        return torch.where(x.isnan(), -math.inf, x.clamp(max=FLT_MAX))

    def soft(x, t):
        m = x.max()
        if m == -math.inf:
            return torch.zeros_like(x)
        e = torch.where(x == -math.inf, 0.0, torch.exp((x - m) / t))
        return e / e.sum()

    for s in range(len(qs) - 1):
        n, t = qs[s + 1] - qs[s], 1.0 if temp is None else float(temp[s])
        if n <= 0:
            acc.append(0)
            nxt.append(-1)
            continue
        for i in range(n):
            r = qs[s] + i
            x = val(logits[r])
            best = int((x == x.max()).nonzero()[0]) if x.max() > -math.inf else -1
            greedy = not t > 0
            p = None if greedy else soft(x, t)
            q = soft(val(draft[r]), t) if draft is not None and not greedy else None
            if i == n - 1:
                break
            w = int(tokens[r + 1])
            inside = 0 <= w < len(x)
            pr = float(w == best) if greedy else float(p[w]) if inside else 0.0
            prob[r] = pr
            if not (pr > 0 if greedy else float(ua[r]) * (1.0 if q is None else float(q[w]) if inside else 0.0) < pr):
                break
        for j in range(i + 1, n - 1):  # the rows behind keep their probabilities
            r = qs[s] + j
            y = val(logits[r])
            v = int(tokens[r + 1])
            if greedy:
                prob[r] = float(y.max() > -math.inf and v == int((y == y.max()).nonzero()[0]))
            else:
                prob[r] = float(soft(y, t)[v]) if 0 <= v < len(y) else 0.0
        acc.append(i)
        if greedy or x.max() == -math.inf:
            nxt.append(best)
            continue
        if i < n - 1:
            if q is not None:
                p = (p - q).clamp(min=0) if bool((p > q).any()) else p
            elif inside:
                p = p.clone()
                p[w] = 0
        c = p.cumsum(0)
        past = (c > float(un[s]) * float(c[-1])).nonzero()
        nxt.append(int(past[0]) if len(past) else -1)
    return acc, nxt, torch.tensor(prob, dtype=torch.float64)


def case(seed, nq, vocab, kind, with_draft, temp=None, hint=9.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    qs = [0]
    for n in nq:
        qs.append(qs[-1] + n)
    rows = qs[-1]
    d = 2.0 * torch.randn(rows, vocab, generator=g)
    d[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] += hint
    x = d + 0.5 * torch.randn(rows, vocab, generator=g)
    gum = -torch.log(-torch.log(torch.rand(rows, vocab, generator=g).clamp(1e-9, 1 - 1e-7)))
    tokens = torch.roll(torch.argmax(d + gum, 1), 1).to(torch.int32)

    def cast(t):
        t = (t * 256).round().clamp(-32768, 32767).to(torch.int16) if kind == torch.int16 else t.to(kind)
        out = torch.zeros(rows, vocab + pad, dtype=t.dtype)
        out[:, :vocab] = t
        return out[:, :vocab]

    ua, un = torch.rand(rows, generator=g), torch.rand(len(nq), generator=g)
    if temp is not None:
        temp = torch.tensor(temp, dtype=torch.float32)
    return qs, tokens, cast(x), ua, un, cast(d) if with_draft else None, temp


def run(gpu, qs, tokens, logits, ua, un, draft=None, temp=None):
    def dev(t):
        if t is None:
            return None
        if t.dim() == 2 and not t.is_contiguous():  # keep the rows' padding
            base = torch.empty(t.shape[0], t.stride(0), dtype=t.dtype)
            base[:, :t.shape[1]] = t
            return base.cuda()[:, :t.shape[1]]
        return t.cuda()

    a, n, p = gpu.draft_verify(torch.tensor(qs, dtype=torch.int32).cuda(), *map(dev, (tokens, logits, ua, un)),
                               draft=dev(draft), temp=dev(temp))
    return a.cpu().tolist(), n.cpu().tolist(), p.cpu().double()


def check(gpu, *c):
    got, want = run(gpu, *c), expect(*c)
    assert got[0] == want[0] and got[1] == want[1]
    # one rounding to float32 of a value good to about 2^-45
    assert ((got[2] - want[2]).abs() <= want[2] * 2.0 ** -23 + 2.0 ** -149).all()
    return got


KINDS = [torch.float32, torch.bfloat16, torch.float16, torch.int16]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab, pad", [(1, 0), (7, 0), (100, 0), (6400, 0), (6401, 3), (20011, 0)])
def test_definition(gpu, kind, with_draft, vocab, pad):
    got = check(gpu, *case(1, [5, 1, 3, 8, 2, 6, 4, 9], vocab, kind, with_draft, pad=pad))
    if vocab >= 6400:
        assert 0 < sum(got[0]) < 30  # some taken, some refused


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_temperatures(gpu, kind):
    t = [0.7, 0.0, 1.3, 1e-3, -1.0, math.nan, 50.0, 1e-38, math.inf]
    check(gpu, *case(2, [4, 4, 4, 4, 4, 4, 4, 4, 4], 3001, kind, True, t))
    check(gpu, *case(3, [4, 4, 4, 4, 4, 4, 4, 4, 4], 3001, kind, False, t))


@pytest.mark.gpu
@pytest.mark.parametrize("with_draft", [False, True])
def test_empty_and_long_sequences(gpu, with_draft):
    check(gpu, *case(4, [0, 1, 0, 70, 0], 500, torch.float32, with_draft, hint=14.0))
    check(gpu, *case(5, [3] * 100 + [0] * 40 + [1], 50, torch.int16, with_draft))


@pytest.mark.gpu
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("vocab", [3, 4001, 70001])
def test_q16_rails(gpu, vocab, with_draft):
    """Distances from the maximum up to 65535 steps, by rows that hold both
    ends, only the lowest value, or a maximum of every low byte."""
    t = [1.0, 40.0, 0.05, 0.0, 1e-30, 300.0]
    qs, tok, x, ua, un, d, temp = case(24, [5] * 6, vocab, torch.int16, with_draft, t)
    g = torch.Generator().manual_seed(25)
    for y in (x, d) if with_draft else (x,):
        y[::4] = torch.randint(-32768, 32768, y[::4].shape, generator=g).to(torch.int16)
        y[1::4, ::2] = -32768
        y[2::8] = -32768
        y[3::8, vocab // 2:] = 32767
    check(gpu, qs, tok, x, ua, un, d, temp)


@pytest.mark.gpu
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("kind, vocab", [(torch.float32, 300007), (torch.int16, 600011), (torch.bfloat16, 530001)])
def test_more_chunks_than_lanes(gpu, kind, vocab, with_draft):
    """Rows of over 64 chunks; also the last of them alone holding the weight."""
    c = case(21, [3, 1, 4], vocab, kind, with_draft, [0.9, 0.0, 1.2])
    check(gpu, *c)
    if kind != torch.int16:
        c[2][:, :vocab - 5] = -math.inf
        check(gpu, *c)


@pytest.mark.gpu
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("kind", KINDS)
def test_many_rows(gpu, kind, with_draft):
    """Enough rows that a thread takes four pieces of a chunk."""
    check(gpu, *case(22, [9] * 14 + [5], 20011, kind, with_draft, [0.8, 0.0, 1.0] * 5, pad=1))


@pytest.mark.gpu
@pytest.mark.parametrize("at", [31, 32, 33, 50, 63, 64, 68])
@pytest.mark.parametrize("with_draft, temp", [(False, 0.0), (False, 1.0), (True, 1.0)])
def test_refused_far_into_a_sequence(gpu, at, with_draft, temp):
    """Drafts that are the rows' maxima and pass, up to one that cannot."""
    qs, tok, x, ua, un, d, _ = case(23, [2, 70], 300, torch.float32, with_draft)
    tok[1:] = x[:-1].argmax(1).to(torch.int32)
    ua.zero_()
    tok[2 + at + 1] = 299
    x[2 + at, 299] = -math.inf
    t = torch.tensor([temp, temp])
    got = check(gpu, qs, tok, x, ua, un, d, t)
    assert got[0][1] == at


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_draft", [False, True])
def test_masked_and_odd_logits(gpu, kind, with_draft):
    qs, tok, x, ua, un, d, _ = case(6, [3, 3, 3, 3, 3], 900, kind, with_draft)
    x[0, ::2] = -math.inf          # half the row masked
    x[3, :] = -math.inf            # a mask that leaves nothing
    x[6, 17] = math.nan
    x[6, int(tok[7])] = math.nan   # the draft itself
    x[9, [5, 800]] = math.inf      # two infinities share the row
    x[12, :] = -math.inf
    x[12, 33] = 1.0                # one token left, which is not the draft
    tok[13] = 34
    if with_draft:
        d[12, 40:] = -math.inf
    check(gpu, qs, tok, x, ua, un, d, None)
    check(gpu, qs, tok, x, ua, un, d, torch.zeros(5))


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 900, 2 ** 31 - 1, -2 ** 31])
def test_drafts_outside_the_vocabulary(gpu, bad):
    qs, tok, x, ua, un, d, _ = case(7, [3, 3], 900, torch.float32, True)
    tok[1] = tok[5] = bad
    check(gpu, qs, tok, x, ua, un, d, None)
    check(gpu, qs, tok, x, ua, un, None, torch.tensor([1.0, 0.0]))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_ties_go_to_the_lowest_index(gpu, kind):
    qs, tok, x, ua, un, d, _ = case(8, [2, 2], 30000, kind, False)
    x.zero_()
    x[0, [29000, 12345, 12346]] = 5
    x[2, [8192, 8191]] = 5
    tok[1], tok[3] = 12345, 8192
    got = check(gpu, qs, tok, x, ua, un, None, torch.zeros(2))
    assert got[0] == [1, 0] and got[1] == [0, 8191]


@pytest.mark.gpu
def test_random_numbers_at_the_ends(gpu):
    """u = 0 takes any draft of weight and the first token of weight; u next to 1 the last."""
    qs, tok, x, _, _, d, _ = case(9, [2, 2, 1, 1], 5000, torch.float32, True)
    x[4, :7] = -math.inf
    x[4, 4990:] = -math.inf
    x[5] = x[4]
    top = 1 - 2.0 ** -24
    ua, un = torch.tensor([0.0, 0, top, 0, 0, 0]), torch.tensor([0.0, 0.0, 0.0, top])
    got = check(gpu, qs, tok, x, ua, un, d, None)
    assert got[0][0] == 1 and got[1][2] == 7


@pytest.mark.gpu
def test_same_distributions_take_every_draft(gpu):
    qs, tok, x, ua, un, d, _ = case(10, [6] * 8, 4000, torch.float32, True)
    got = check(gpu, qs, tok, d, torch.full_like(ua, 1 - 2.0 ** -24), un, d, None)
    assert got[0] == [5] * 8


@pytest.mark.gpu
def test_the_draws_follow_the_target(gpu):
    """20000 sequences of one draft over five tokens: what is emitted first
    (the draft or its replacement) is distributed as the target, whatever the
    draft's distribution: 5 standard deviations of each count."""
    g = torch.Generator().manual_seed(11)
    n = 20000
    lt, ld = torch.tensor([0.5, 1.5, -0.3, 0.0, 1.0]), torch.tensor([1.5, -0.5, 0.8, 0.0, -1.0])
    p, q = torch.softmax(lt.double(), 0), torch.softmax(ld.double(), 0)
    first = torch.multinomial(q, n, True, generator=g)
    tok = torch.zeros(2 * n, dtype=torch.int32)
    tok[1::2] = first.int()
    x, d = lt.expand(2 * n, 5).contiguous(), ld.expand(2 * n, 5).contiguous()
    a, nx, _ = run(gpu, list(range(0, 2 * n + 1, 2)), tok, x, torch.rand(2 * n, generator=g), torch.rand(n, generator=g), d)
    out = torch.where(torch.tensor(a) == 1, first, torch.tensor(nx))
    cnt = torch.bincount(out, minlength=5).double()
    assert ((cnt - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p))).all()


@pytest.mark.gpu
def test_rows_of_no_sequence_stay(gpu):
    qs, tok, x, ua, un, _, _ = case(12, [3, 2], 700, torch.float32, False)
    x2, tok2, ua2 = torch.cat([x, x]), torch.cat([tok, tok]), torch.cat([ua, ua])
    prob = torch.full((10,), -3.0, device="cuda")
    out = torch.empty(4, dtype=torch.int32, device="cuda")
    L = vl.load()
    t = [t.cuda() for t in (torch.tensor(qs, dtype=torch.int32), tok2, x2, ua2, un)]
    need = L.vgx_draft_verify_ws(2, 10, 700, vl.E_F32, 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    a = vl.Draft(2, 10, 700, t[0].data_ptr(), t[1].data_ptr(), vl.E_F32, t[2].data_ptr(), 700, 0, 0, 0, t[3].data_ptr(),
                 t[4].data_ptr(), out.data_ptr(), out.data_ptr() + 8, prob.data_ptr(), ws.data_ptr(), need)
    vl.check(L.vgx_draft_verify(gpu.ctx, ctypes.byref(a)))
    want = expect(qs, tok, x, ua, un)
    assert out.cpu().tolist() == want[0] + want[1]
    assert (prob[5:] == -3).all() and (prob[:5] >= 0).all()


@pytest.mark.gpu
def test_stream_and_graph(gpu):
    c = case(13, [4, 1, 6], 9000, torch.bfloat16, True, [0.8, 0.0, 1.1])
    t = [None if v is None else v.cuda() for v in c[1:]]
    qs = torch.tensor(c[0], dtype=torch.int32).cuda()
    f = lambda: gpu.draft_verify(qs, *t[:4], draft=t[4], temp=t[5])  # noqa: E731
    f()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s = f()
    side.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = f()
    assert [v.cpu().tolist() for v in s[:2]] == list(expect(*c)[:2])
    for i in range(3):
        t[2].copy_(torch.rand(11))
        t[1].copy_(torch.roll(t[1], 1, 0))
        gr.replay()
        torch.cuda.synchronize()
        e = f()
        assert all(torch.equal(a, b) for a, b in zip(o, e)), i


TIED = [
    # (vocabulary, u, the tokens of equal logits): a draw on the border of two
    (1024, 0.875, [6, 12, 15, 44, 77, 126, 146, 151, 205, 307, 338, 360, 436, 442, 456, 468, 493, 529, 553, 569, 586, 597,
                   613, 617, 630, 655, 693, 716, 779, 834, 837, 842, 861, 862, 865, 903, 918, 933, 977, 997]),
    (256, 0.5, [28, 75, 90, 93, 100, 101, 108, 109, 110, 119, 124, 134, 141, 156, 157, 168, 178, 216, 217, 218]),
]


def tied_cases():
    g = torch.Generator().manual_seed(31)
    out = list(TIED)
    for vocab in (1024, 5000, 70001):
        for _ in range(100):
            n = int(torch.randint(1, 60, (1,), generator=g))
            at = torch.randperm(vocab, generator=g)[:n].sort().values.tolist()
            out.append((vocab, int(torch.randint(0, 16, (1,), generator=g)) / 16, at))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("how", ["last", "refused", "drafted"])
def test_few_tokens_of_equal_weight(gpu, kind, how):
    """Rows whose mask leaves n tokens of one logit, and draws on a border
    between two: token floor(u n) of them, exactly.  "last": a row without a
    draft; "refused": one whose draft is a further token of that logit;
    "drafted": p = q, every draft a token without weight."""
    for vocab in (256, 1024, 5000, 70001):
        some = [c for c in tied_cases() if c[0] == vocab]
        one = 1 if how == "last" else 2
        x = torch.full((one * len(some), vocab), -128.0 if kind == torch.int16 else -math.inf)
        tok = torch.zeros(one * len(some), dtype=torch.int32)
        want = []
        for i, (_, u, at) in enumerate(some):
            x[one * i, at] = 3.0
            want.append(at[int(u * len(at))])
            if how == "refused":
                w = next(j for j in range(i % vocab, 2 * vocab) if j % vocab not in at) % vocab
                x[one * i, w] = 3.0
                tok[one * i + 1] = w
            elif how == "drafted":
                tok[one * i + 1] = next(j for j in range(vocab) if j not in at)
            if one == 2:
                x[2 * i + 1, 0] = 0.0
        x = (x * 256).to(torch.int16) if kind == torch.int16 else x.to(kind)
        # (q16 has no mask: its lowest value at T = 1/16, e^-2096 of the others)
        temp = torch.full((len(some),), 1.0 / 16 if kind == torch.int16 else 1.0)
        ua = torch.full((len(tok),), 1 - 2.0 ** -24)
        un = torch.tensor([c[1] for c in some])
        qs = list(range(0, len(tok) + 1, one))
        a, n, _ = run(gpu, qs, tok, x, ua, un, x.clone() if how == "drafted" else None, temp)
        assert a == [0] * len(some) and n == want, vocab


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [4100, 70001])
def test_refused_draft_alone_in_its_chunk(gpu, kind, vocab):
    """What is left beside a refused draft is next to nothing, or nothing: the
    draw goes by the tokens that have a weight, in the draft's chunk or past it."""
    x = torch.full((12, vocab), -math.inf)
    tok = torch.zeros(12, dtype=torch.int32)
    want = []
    # the draft 689.5 below the maximum, its neighbours past the cut at e^-690
    x[0, :900], x[0, 7], x[0, 4000:4010] = -691.0, -689.5, 0.0
    # a neighbour well inside it
    x[2, :900], x[2, 7], x[2, 30], x[2, 4000:4010] = -691.0, -689.5, -600.0, 0.0
    # the draft the maximum, 1999 neighbours with 10^-6 of its weight together, and nothing else
    x[4, :2000], x[4, 7] = -21.5, 0.0
    # ... and as much in two chunks
    x[6, :1000], x[6, 7], x[6, 3100:4100] = -21.5, 0.0, -21.5
    # the draft the only token: it is taken, and row 9 has token 0 alone
    x[8, 7] = 0.0
    # the draft at the row's end, its chunk-mates masked
    x[10, vocab - 1], x[10, 3] = 5.0, -8.0
    un = torch.tensor([0.0, 0.0, 0.5, 0.75, 0.5, 0.0])
    # row 4: 1999 equal weights, u 999.5 of them: the 1000th, at 1000 (behind the draft);
    # row 6: 999 and 1000, u 1499.25: the 501st of the second, at 3600
    want = [4000, 30, 1000, 3600, 0, 3]
    tok[1::2] = 7
    tok[11] = vocab - 1
    x[1::2, 0] = 0.0
    ua = torch.full((12,), 1 - 2.0 ** -24)
    a, n, _ = run(gpu, list(range(0, 13, 2)), tok, x.to(kind), ua, un)
    assert a == [0, 0, 0, 0, 1, 0] and n == want


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [5, 6401, 40003])
def test_rows_that_begin_anywhere(gpu, kind, vocab):
    """Logits and the draft's of other strides and first addresses: their rows
    begin at different places of a 16-byte piece."""
    qs, tok, x, ua, un, d, _ = case(26, [5, 1, 3, 8, 2, 6], vocab, kind, True)
    dev = [t.cuda() for t in (torch.tensor(qs, dtype=torch.int32), tok, ua, un)]
    want = expect(qs, tok, x, ua, un, d)

    def placed(t, before, width):
        base = torch.full((t.shape[0], width), 9, dtype=t.dtype, device="cuda")
        base[:, before:before + vocab] = t.cuda()
        return base[:, before:before + vocab]

    for (bx, wx), (bd, wd) in (((0, vocab), (1, vocab + 3)), ((3, vocab + 5), (0, vocab + 1)), ((7, vocab + 7), (2, vocab + 9))):
        a, n, p = gpu.draft_verify(dev[0], dev[1], placed(x, bx, wx), dev[2], dev[3], draft=placed(d, bd, wd))
        assert a.cpu().tolist() == want[0] and n.cpu().tolist() == want[1]
        assert ((p.cpu().double() - want[2]).abs() <= want[2] * 2.0 ** -23 + 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [300, 6401, 20003])
def test_equal_distributions_that_begin_elsewhere(gpu, kind, vocab):
    """p = q, rows at different places of a 16-byte piece (so their sums are
    added in different orders), and a draft that no token is: the draw is from
    p, as where the rows lie alike."""
    n = 64
    qs, tok, x, ua, un, _, _ = case(27, [2] * n, vocab, kind, False, hint=0.0)
    tok[1::2] = vocab
    want = expect(qs, tok, x, ua, un, x)
    dev = [t.cuda() for t in (torch.tensor(qs, dtype=torch.int32), tok, ua, un)]
    base = torch.zeros(2 * n, vocab + 9, dtype=x.dtype, device="cuda")
    for before in (0, 1, 3, 5):
        d = base[:, before:before + vocab]
        d.copy_(x)
        a, nx, _ = gpu.draft_verify(dev[0], dev[1], x.cuda(), dev[2], dev[3], draft=d)
        assert a.cpu().tolist() == [0] * n and nx.cpu().tolist() == want[1], before


BUF = 1 << 20


def args(**kw):
    d = dict(nseq=2, ntok=6, vocab=100, qstart=BUF, tokens=BUF, kind=vl.E_F32, logits=BUF, stride=100, draft=0,
             draft_stride=0, temp=0, u_accept=BUF, u_next=BUF, accepted=BUF, next=BUF, prob=0, ws=BUF, ws_bytes=1 << 16)
    d.update(kw)
    return vl.Draft(**d)


@pytest.mark.parametrize("bad, what", [
    (dict(nseq=-1), "nseq"), (dict(ntok=65536), "ntok"), (dict(nseq=65536), "nseq"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 26) + 1), "vocab"), (dict(kind=vl.E_Q8), "f32"), (dict(qstart=0), "NULL qstart"),
    (dict(accepted=0), "NULL"), (dict(next=0), "NULL"), (dict(u_next=0), "NULL"), (dict(logits=0), "NULL logits"),
    (dict(tokens=0), "tokens"), (dict(u_accept=0), "u_accept"), (dict(stride=99), "stride"),
    (dict(draft=BUF, draft_stride=99), "stride"), (dict(logits=BUF + 2), "aligned"),
    (dict(draft=BUF + 1, draft_stride=100), "aligned"), (dict(ws=0), "workspace"), (dict(ws_bytes=95), "workspace"),
    (dict(ws=BUF + 8), "workspace"), (dict(), "no context"),
])
def test_refusals(bad, what):
    L = vl.load()
    assert L.vgx_draft_verify(None, ctypes.byref(args(**bad))) == vl.VGX_EINVAL
    assert what in L.vgx_last_error().decode()


def test_more_than_a_launch_holds():
    """65535 rows of 2^26 logits: refused by the library, not by the launch."""
    L = vl.load()
    big = dict(ntok=65535, vocab=1 << 26, stride=1 << 26, ws_bytes=1 << 60)
    assert L.vgx_draft_verify(None, ctypes.byref(args(**big))) == vl.VGX_ERANGE
    assert "too many" in L.vgx_last_error().decode()
    assert L.vgx_draft_verify(None, ctypes.byref(args(nseq=65535, vocab=1 << 24, stride=1 << 24,
                                                      ws_bytes=1 << 60))) == vl.VGX_ERANGE


def test_workspace_sizes():
    L = vl.load()
    assert L.vgx_draft_verify_ws(2, 6, 100, vl.E_F32, 0) == 6 * 16
    assert L.vgx_draft_verify_ws(2, 6, 100, vl.E_F32, 1) == 12 * 16 + 16
    assert L.vgx_draft_verify_ws(2, 6, 0, vl.E_F32, 0) == 0
    assert L.vgx_draft_verify(None, None) == vl.VGX_EINVAL
