"""vgx_sample against its definition in 64 bits."""
import math

import pytest
import torch

import tree_ref as tr

pytestmark = pytest.mark.gpu

KINDS = [torch.float32, torch.bfloat16, torch.float16, torch.int16]
NONE = dict(temp=None, top_k=None, top_p=None, min_p=None)


def cast(x, kind, pad=0):
    x = (x * 256).round().clamp(-32768, 32767).to(torch.int16) if kind == torch.int16 else x.to(kind)
    out = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype)
    out[:, :x.shape[1]] = x
    return out[:, :x.shape[1]]


def rows_of(seed, rows, vocab, kind, spread=2.0, top=12.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    n = min(vocab, 40)
    at = torch.randint(0, vocab, (rows, n), generator=g)
    x.scatter_(1, at, top + torch.randn(rows, 1, generator=g) - 1.5 * torch.log(torch.arange(1.0, n + 1)))
    return cast(x, kind, pad), torch.rand(rows, generator=g)


def run(gpu, x, u, **cuts):
    f = lambda v, t: None if v is None else torch.tensor(v, dtype=t).cuda()  # noqa: E731
    base = torch.zeros(x.shape[0], x.stride(0) if x.shape[0] > 1 else x.shape[1], dtype=x.dtype)
    base[:, :x.shape[1]] = x
    out = gpu.sample(base.cuda()[:, :x.shape[1]], u.cuda(), temp=f(cuts.get("temp"), torch.float32),
                     top_k=f(cuts.get("top_k"), torch.int32), top_p=f(cuts.get("top_p"), torch.float32),
                     min_p=f(cuts.get("min_p"), torch.float32))
    return [t.cpu() for t in out]


def check(gpu, x, u, **cuts):
    token, kept, prob = run(gpu, x, u, **cuts)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).item()  # noqa: E731
    for r in range(x.shape[0]):
        c = {k: None if v is None else (v[r] if k == "top_k" else f32(v[r])) for k, v in {**NONE, **cuts}.items()}
        t, n, p = tr.sample(x[r], u[r], **c)
        assert (int(token[r]), int(kept[r])) == (t, n), (r, c)
        # one rounding to float32 of a value good to about 2^-40
        assert abs(float(prob[r]) - p) <= p * 2.0 ** -23, (r, c)
    return token, kept, prob


CUTS = [dict(), dict(top_k=[1, 2, 5, 40, 50, 100, 0, 20]), dict(top_p=[0.1, 0.5, 0.8, 0.9, 0.95, 0.99, 0.999, 1.0]),
        dict(min_p=[0.5, 0.2, 0.1, 0.05, 0.02, 0.01, 1e-4, 0.0]),
        dict(top_k=[40] * 8, top_p=[0.9] * 8, min_p=[0.0, 0.1] * 4),
        dict(top_k=[3, 1000, 0, 10, 100, 0, 7, 2000], top_p=[0.3, 0.99, 0.7, 1.0, 0.9, 1.0, 1.0, 0.999],
             min_p=[0.0, 0.01, 0.3, 0.0, 0.02, 0.1, 0.05, 1e-5])]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cuts", range(len(CUTS)))
@pytest.mark.parametrize("vocab, pad", [(1, 0), (7, 1), (100, 0), (6400, 0), (6401, 3), (20011, 1), (64402, 0)])
def test_definition(gpu, kind, cuts, vocab, pad):
    x, u = rows_of(1, 8, vocab, kind, pad=pad)
    check(gpu, x, u, temp=[0.7, 1.0, 1.3, 0.5, 0.9, 2.0, 0.8, 1.1], **CUTS[cuts])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cuts", range(len(CUTS)))
def test_open_rows(gpu, kind, cuts):
    """No token stands out: thousands stay."""
    x, u = rows_of(2, 8, 30011, kind, spread=1.0, top=1.0)
    check(gpu, x, u, temp=[0.7, 1.0, 1.3, 5.0, 0.9, 2.0, 0.8, 100.0], **CUTS[cuts])


@pytest.mark.parametrize("kind", KINDS)
def test_temperatures(gpu, kind):
    t = [0.0, -1.0, math.nan, 1e-3, 1e-38, 50.0, math.inf, 0.3]
    x, u = rows_of(3, 8, 3001, kind)
    check(gpu, x, u, temp=t)
    check(gpu, x, u, temp=t, top_k=[50] * 8, top_p=[0.9] * 8)
    check(gpu, x, u, temp=t, top_p=[0.9] * 8, min_p=[0.05] * 8)
    check(gpu, x, u)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [5, 3000, 20011])
def test_cuts_out_of_range(gpu, kind, vocab):
    """Counts past the vocabulary, negative ones, probabilities of 0, below and
    above, and no numbers."""
    x, u = rows_of(4, 8, vocab, kind)
    check(gpu, x, u, top_k=[vocab, vocab + 1, 2 ** 31 - 1, -1, -2 ** 31, 0, vocab - 1, 1])
    check(gpu, x, u, top_p=[0.0, -1.0, math.nan, 2.0, math.inf, 1e-30, 1 - 2.0 ** -24, -math.inf])
    check(gpu, x, u, min_p=[1.0, 1.5, math.nan, -1.0, math.inf, 1e-30, 1 - 2.0 ** -24, 0.0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [64, 5000, 70000])
def test_ties(gpu, kind, vocab):
    """Equal logits: the lower indices stay, at every cut; sums of ones are exact."""
    g = torch.Generator().manual_seed(5)
    x = torch.zeros(8, vocab)
    x[4:] = torch.randint(0, 3, (4, vocab), generator=g).float()
    x[6, ::7] = -0.0
    x = cast(x, kind)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.1, 0.3, 0.6, 1 - 2.0 ** -24])
    check(gpu, x, u)
    check(gpu, x, u, top_k=[1, 2, 16, 33, 50, 64, 10, vocab - 1])
    check(gpu, x, u, top_p=[0.5, 0.25, 0.125, 0.75, 0.5, 0.9, 0.3, 0.99])
    check(gpu, x, u, top_k=[32] * 8, top_p=[0.5] * 8)
    check(gpu, x, u, min_p=[1.0] * 8)
    check(gpu, x, u, top_k=[40] * 8, min_p=[0.2] * 8)


@pytest.mark.parametrize("kind", KINDS[:3])
def test_masked_and_odd_logits(gpu, kind):
    x, u = rows_of(6, 8, 5000, kind)
    x[0] = -math.inf
    x[1, ::2] = -math.inf
    x[2] = -math.inf
    x[2, 4321] = -3.0
    x[3, 100] = math.inf
    x[4, ::3] = math.nan
    x[5] = math.nan
    x[6, 17:29] = math.inf
    x[7] = -math.inf
    x[7, [0, 4999]] = torch.finfo(kind).min
    for cuts in (dict(), dict(top_k=[50] * 8), dict(top_p=[0.9] * 8), dict(min_p=[0.1] * 8),
                 dict(top_k=[4000] * 8, top_p=[0.5] * 8)):
        check(gpu, x, u, **cuts)


def test_q16_rails(gpu):
    g = torch.Generator().manual_seed(7)
    x = torch.randint(-32768, 32768, (6, 9001), generator=g).to(torch.int16)
    x[1] = -32768
    x[2, ::2] = -32768
    x[3] = 32767
    u = torch.rand(6, generator=g)
    for t in (1.0, 30.0, 300.0):
        check(gpu, x, u, temp=[t] * 6)
        check(gpu, x, u, temp=[t] * 6, top_p=[0.9] * 6)
        check(gpu, x, u, temp=[t] * 6, top_k=[300] * 6, top_p=[0.7] * 6)


@pytest.mark.parametrize("kind", [torch.float32, torch.int16])
@pytest.mark.parametrize("vocab", [131072, 300007, 2 ** 21])
def test_large_vocabularies(gpu, kind, vocab):
    x, u = rows_of(8, 3, vocab, kind)
    check(gpu, x, u, top_p=[0.9, 0.5, 0.99], temp=[1.2, 0.8, 0.4])
    check(gpu, x, u, top_k=[50, 3000, 100000])
    check(gpu, x, u)


@pytest.mark.parametrize("kind", KINDS)
def test_many_rows(gpu, kind):
    x, u = rows_of(9, 700, 3001, kind, pad=5)
    g = torch.Generator().manual_seed(10)
    pick = lambda v: [v[i] for i in torch.randint(0, len(v), (700,), generator=g).tolist()]  # noqa: E731
    check(gpu, x, u, temp=pick([0.0, 0.7, 1.0, 1.4]), top_k=pick([0, 0, 1, 20, 50, 400]),
          top_p=pick([1.0, 0.8, 0.95]), min_p=pick([0.0, 0.0, 0.05]))


def test_draws_follow_the_distribution(gpu):
    """Draws of one row by evenly spaced numbers: each token as often as its
    share says, to one."""
    x, _ = rows_of(11, 1, 500, torch.float32, spread=1.0, top=4.0)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    token, kept, prob = run(gpu, x.expand(n, -1).contiguous(), u, top_p=[0.9] * n)
    count = torch.bincount(token.long(), minlength=500).double()
    p = torch.zeros(500, dtype=torch.float64)
    p[token.long()] = prob.double()
    assert (kept == kept[0]).all() and (token[1:] >= token[:-1]).all()
    assert ((count / n - p).abs() <= 1.0 / n + 2.0 ** -20).all()


def test_rows_do_not_depend_on_others(gpu):
    """A row alone, in a batch and at another alignment draws the same."""
    x, u = rows_of(12, 9, 20011, torch.float32, pad=3)
    cuts = dict(temp=[1.3] * 9, top_p=[0.97] * 9)
    token, kept, prob = run(gpu, x, u, **cuts)
    for r in range(9):
        one = run(gpu, x[r:r + 1].contiguous(), u[r:r + 1], temp=[1.3], top_p=[0.97])
        assert [int(one[0]), int(one[1])] == [int(token[r]), int(kept[r])]
        assert abs(float(one[2]) - float(prob[r])) <= float(prob[r]) * 2.0 ** -23


def test_numbers_outside_their_range(gpu):
    """A number of 1 or more, or none, takes the last token that has a weight; a
    negative one the first."""
    x, _ = rows_of(13, 6, 1000, torch.float32, spread=0.5, top=1.0)
    u = torch.tensor([1.0, 7.0, math.nan, math.inf, -1.0, -math.inf])
    token = run(gpu, x, u)[0].tolist()
    assert token == [999, 999, 999, 999, 0, 0]


def test_nothing_to_do(gpu):
    e = lambda t: torch.empty(0, dtype=t).cuda()  # noqa: E731
    token, kept, prob = gpu.sample(torch.empty(0, 100).cuda(), e(torch.float32))
    assert token.shape == kept.shape == prob.shape == (0,)


def test_graph_and_streams(gpu):
    from vgx import gpu as vg
    g = vg.GPU(0)
    x, u = rows_of(14, 40, 20011, torch.float32)
    x, u = x.cuda(), u.cuda()
    top_p = torch.full((40,), 0.9).cuda()
    want = g.sample(x, u, top_p=top_p)
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        got = g.sample(x, u, top_p=top_p)
    for i in range(3):
        u.copy_(torch.rand(40, generator=torch.Generator().manual_seed(i)))
        gr.replay()
        want = g.sample(x, u, top_p=top_p)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x * 0.5
        a = g.sample(y, u, top_p=top_p)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, g.sample(y, u, top_p=top_p)))
    g.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, vocab", [(1, 30011), (40, 64402), (5, 400009)])
def test_thousands_stay(gpu, kind, rows, vocab):
    """Rows without a peak, by top-p alone: what stays is past what is gathered."""
    x, u = rows_of(15, rows, vocab, kind, spread=2.0, top=9.0, pad=1)
    p = [[0.9, 0.5, 0.99, 0.999, 0.7][i % 5] for i in range(rows)]
    t = [[1.0, 1.5, 2.0, 1.3, 0.9, 4.0, 1e3][i % 7] for i in range(rows)]
    kept = check(gpu, x, u, temp=t, top_p=p)[1]
    assert int(kept.max()) > 4096
    check(gpu, x, u, temp=t, min_p=[1e-4] * rows)
    check(gpu, x, u, temp=t, top_p=p, min_p=[1e-6] * rows)
    check(gpu, x, u, temp=t, top_k=[5000] * rows, top_p=p)


@pytest.mark.parametrize("shift", [-1e30, -3e5, -1000.0, 1000.0, 3e5, 1e30])
@pytest.mark.parametrize("temp", [1e-6, 0.7, 3.0])
def test_far_from_zero(gpu, shift, temp):
    """Logits whose bins are no whole numbers, or far from 0."""
    x, u = rows_of(16, 4, 9001, torch.float32)
    x = x + shift
    check(gpu, x, u, temp=[temp] * 4, top_p=[0.9] * 4)
    check(gpu, x, u, temp=[temp] * 4, top_k=[100] * 4)
    check(gpu, x, u, temp=[temp] * 4, min_p=[0.1] * 4)
    check(gpu, x, u, temp=[temp] * 4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [4099, 5000, 8000, 30011, 64402, 200003])
def test_large_top_k(gpu, kind, vocab):
    """Top-k by thousands: past the groups, past what is gathered."""
    k = [v for v in (300, 700, 1000, 1500, 2500, 3300, 4000, 4096, 4097, 9000, 60000) if v < vocab]
    x, u = rows_of(17, len(k), vocab, kind, spread=2.0, top=9.0, pad=1)
    check(gpu, x, u, top_k=k, temp=[1.3] * len(k))
    check(gpu, x, u, top_k=k, top_p=[0.9] * len(k), min_p=[1e-5] * len(k))
    x[:, : vocab // 2] = -32768 if kind == torch.int16 else -math.inf
    check(gpu, x, u, top_k=k, temp=[2.0] * len(k))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab, per", [(6400, 4), (6400, 8), (64402, 64)])
def test_top_k_of_logits_in_order(gpu, kind, vocab, per):
    """The first ones lie one a group, so fewer reach what groups' maxima do than
    logits without an order would; or side by side, so that far more do."""
    i = torch.arange(vocab)
    even = 10.0 - (i % per) * (16.0 / per) - (i // per) * (3.0 / vocab)
    row = torch.stack([even, 10.0 - i * (16.0 / vocab)])
    x, u = cast(row.repeat(4, 1), kind), rows_of(18, 8, 8, kind)[1]
    for k in (vocab // per * 3 // 4, vocab // per - 9):
        check(gpu, x, u, top_k=[k] * 8, temp=[1.5] * 8)
        check(gpu, x, u, top_k=[k] * 8, temp=[1.5] * 8, top_p=[0.8] * 8)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows, vocab", [(3, 6000), (9, 30011), (700, 9001)])
def test_cuts_left_out_or_open(gpu, kind, rows, vocab):
    """No array of cuts and one that keeps all are the same."""
    x, u = rows_of(19, rows, vocab, kind)
    for cuts in (dict(), dict(top_k=[50] * rows), dict(min_p=[0.03] * rows), dict(temp=[0.0] * rows)):
        given = {**dict(temp=[1.0] * rows, top_k=[0] * rows, top_p=[1.0] * rows, min_p=[0.0] * rows), **cuts}
        for a, b in zip(run(gpu, x, u, **cuts), run(gpu, x, u, **given)):
            assert torch.equal(a, b)
