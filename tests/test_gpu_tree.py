"""Drafted trees over a paged cache against their definitions in 64 bits."""
import math

import pytest
import torch

import paged_ref as ref
import tree_ref as tr
from paged_ref import Batch
from test_gpu_paged import make, tables

pytestmark = pytest.mark.gpu


def trees_of(nq, seed, wide=False):
    return [tr.random_tree(n, seed + i, wide) for i, n in enumerate(nq)]


def flat(parents):
    return torch.tensor(sum(parents, []), dtype=torch.int32).cuda()


def check(gpu, b, heads, parents, window=0, scale=None, q=None, out=None, cache=None, batch=None, see=None,
          spread=2.0, **bounds):
    """attend over trees of parents (or any masks: see, lists of rows)."""
    ct = ref.CTYPE[b.kind]
    if q is None:
        q = (spread * b.randn(b.ntok, heads, b.hd)).to(ct)
    if cache is None:
        cache, batch = make(gpu, b, heads, **bounds)
    depth, mine = (sum(x, []) for x in zip(*[tr.lines(p, window) for p in parents]))
    tree = batch.tree(flat(parents), window)
    if see is not None:
        mine = see
        tree.see.copy_(tr.masks(see, tree.words))
    o, lse = cache.attend(batch, q.cuda(), scale=scale or 0.0, window=window, lse=True, out=out, tree=tree)
    batch.check()
    want, wl, mag, dots = tr.attend(b, q, heads, depth, mine, scale, window)
    kind = "q16" if o.dtype == torch.int16 else None
    bound = ref.attn_bound(b, ct, want, mag, dots, kind)
    got = ref.value(o.cpu())[:b.ntok].view_as(want)
    worst = (got - want).abs() - bound
    off = (~(worst <= 0)).nonzero()  # (a NaN too)
    assert not len(off), "%d values off, the first (row, head, dim) %s by %g" % (
        len(off), off[:3].tolist(), float(worst.nan_to_num(9e9).max()))
    lse = lse.cpu().double()
    empty = wl == -math.inf
    assert (lse[empty] == -math.inf).all() and (got[empty] == 0).all()
    tol = dots * (b.hd + 8) * 2.0 ** -22 + (max(b.kv + [1]) + 32) * 2.0 ** -24 + wl.abs() * 2.0 ** -22
    assert ((lse - wl).abs()[~empty] <= tol[~empty]).all()
    return o


@pytest.mark.parametrize("nq", [[1], [5, 0, 3], [64, 63, 65, 1], [130, 2], [1000]])
@pytest.mark.parametrize("window", [0, 1, 3])
def test_masks(gpu, nq, window):
    b = Batch(1, nq, nq, 1, 16, 16, "bf16")
    _, batch = make(gpu, b, 1)
    parents = trees_of(nq, 2)
    for p in parents:  # what is no earlier row makes a root
        if len(p) > 4:
            p[1], p[2], p[3] = 1, -7, 2 ** 31 - 1
    tree = batch.tree(flat(parents), window)
    batch.check()
    depth, see = (sum(x, []) for x in zip(*[tr.lines(p, window) for p in parents]))
    assert tree.depth.cpu().tolist() == depth
    assert tree.words == -(-sum(nq) // 64)
    assert torch.equal(tree.see.cpu(), tr.masks(see, tree.words))


HEADS = [(8, 4, 96), (16, 2, 64), (4, 1, 128), (3, 3, 16), (6, 2, 80), (5, 1, 144), (2, 1, 256)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("heads, kvh, hd", HEADS)
@pytest.mark.parametrize("nq", [[5, 1, 0, 2, 3], [9, 40, 1, 64, 20]])
def test_heads_and_types(gpu, kind, heads, kvh, hd, nq):
    b = Batch(3, nq, [5, 31, 9, 700, 130], kvh, hd, 16, kind)
    check(gpu, b, heads, trees_of(nq, 4))


@pytest.mark.parametrize("page", [1, 5, 16, 48, 64, 1000])
@pytest.mark.parametrize("nq", [[6, 1], [60, 45]])
def test_pages(gpu, page, nq):
    check(gpu, Batch(5, nq, [301, 97], 2, 64, page, "f16"), 4, trees_of(nq, 6))


@pytest.mark.parametrize("base", [0, 1, 31, 32, 33, 63, 64, 65, 127, 500])
@pytest.mark.parametrize("n", [1, 7, 12, 33, 64, 70])
def test_where_the_rows_begin(gpu, base, n):
    """The first new row at every place of a tile of keys."""
    check(gpu, Batch(7, [n], [base + n], 1, 64, 16, "bf16"), 4, trees_of([n], 8), max_q=n)


@pytest.mark.parametrize("window", [1, 2, 4, 31, 64, 65, 200, 5000])
@pytest.mark.parametrize("nq", [[4, 3, 1, 2], [64, 40, 1, 30]])
def test_window(gpu, window, nq):
    check(gpu, Batch(9, nq, [150, 333, 900, 30], 2, 64, 16, "bf16"), 4, trees_of(nq, 10), window=window)
    deep = [list(range(-1, n - 1)) for n in nq]  # chains: the deepest rows
    check(gpu, Batch(11, nq, [150, 333, 900, 70], 1, 128, 64, "f16"), 4, deep, window=window)


@pytest.mark.parametrize("n", [100, 256, 1000])
@pytest.mark.parametrize("heads, kvh, hd", [(2, 1, 64), (2, 2, 128), (1, 1, 256)])
def test_many_words(gpu, n, heads, kvh, hd):
    nq = [n, 3]
    check(gpu, Batch(12, nq, [n + 77, 600], kvh, hd, 16, "bf16"), heads, trees_of(nq, 13, wide=True), max_q=n)


@pytest.mark.parametrize("heads, nq", [(2, [6, 3, 1]), (8, [9, 64, 12]), (4, [100, 3, 70])])
@pytest.mark.parametrize("base", [0, 50])
def test_any_masks(gpu, heads, nq, base):
    """Masks that name later rows, not the row itself, no row at all, or rows
    that are not there."""
    b = Batch(14, nq, [n + base for n in nq], 1, 64, 16, "bf16")
    g = torch.Generator().manual_seed(15)
    see = []
    for n in nq:
        for r in range(n):
            pick = (torch.rand(64 * -(-sum(nq) // 64), generator=g) < 0.3).nonzero()[:, 0].tolist()
            see.append([] if r % 5 == 2 else pick)
    check(gpu, b, heads, trees_of(nq, 16), see=see)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("heads, nq", [(2, [6, 3]), (8, [30, 64])])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_values_that_a_row_does_not_see(gpu, kind, heads, nq, bad):
    """Infinities and NaN in the K and V of rows outside a row's line, and
    behind the sequence's end, do not reach it; in its own line's V they do."""
    b = Batch(17, nq, [n + 41 for n in nq], 1, 64, 16, kind)
    parents = [[-1] + [0] * (n - 1) for n in nq]  # each row sees the first and itself
    q = (2 * b.randn(b.ntok, heads, 64)).to(ref.CTYPE[kind])
    clean = check(gpu, b, heads, parents, q=q).cpu().view(b.ntok, heads, 64)
    last = []
    for s, n in enumerate(nq):  # the last row's, and what stands behind it in its page
        pos = b.kv[s] - 1
        pg, sl = int(b.table[s, pos // 16]), pos % 16
        b.v[pg, 0, sl, ::3] = bad
        b.k[pg, 0, sl + 1:] = bad
        b.v[pg, 0, sl + 1:] = bad
        last.append(int(b.qs[s]) + n - 1)
    cache, batch = make(gpu, b, heads)
    o = cache.attend(batch, q.cuda(), tree=batch.tree(flat(parents)))[0].cpu().view(b.ntok, heads, 64)
    rest = [t for t in range(b.ntok) if t not in last]
    assert torch.equal(o[rest], clean[rest])
    for t in last:
        assert torch.equal(o[t, :, 1::3], clean[t, :, 1::3])
        hit = o[t, :, ::3]
        assert (hit.isnan() if math.isnan(bad) else hit == bad).all()


@pytest.mark.parametrize("heads, n", [(2, 8), (4, 33), (4, 64)])
@pytest.mark.parametrize("window", [0, 3000])
def test_long_sequences_are_split(gpu, heads, n, window):
    nq = [n, 2]
    b = Batch(18, nq, [9000, 2500], 2, 64, 64, "bf16")
    parents = trees_of(nq, 19)
    q = (2 * b.randn(b.ntok, heads, 64)).to(torch.bfloat16)
    a = check(gpu, b, heads, parents, window=window, q=q)
    assert torch.equal(a, check(gpu, b, heads, parents, window=window, q=q))


@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_many_sequences(gpu, kind):
    nq = [1 + i * 7 % 30 for i in range(60)]
    kv = [n + i * 37 % 400 for i, n in enumerate(nq)]
    check(gpu, Batch(20, nq, kv, 2, 64, 16, kind), 16, trees_of(nq, 21), max_q=30, max_kv=max(kv))


@pytest.mark.parametrize("nq", [[3, 1], [40, 9]])
def test_q16_out_and_scale(gpu, nq):
    b = Batch(22, nq, [60, 300], 2, 64, 16, "q8")
    out = torch.full((b.ntok + 2, 256), 77, dtype=torch.int16, device="cuda")
    check(gpu, b, 4, trees_of(nq, 23), out=out, scale=0.2)
    assert (out[b.ntok:] == 77).all()


@pytest.mark.parametrize("nq", [[5, 3], [40, 20]])
def test_more_rows_than_positions(gpu, nq):
    """Rows before position 0 are in no slot; what is left is seen."""
    check(gpu, Batch(24, nq, [3, 0], 1, 64, 16, "bf16"), 2, trees_of(nq, 25))


def test_faults(gpu):
    from vgx import lib as vl
    b = Batch(26, [4, 3], [20, 30], 1, 64, 16, "bf16")
    parents = trees_of([4, 3], 27)
    q = b.randn(b.ntok, 2, 64).to(torch.bfloat16).cuda()
    for change, word in ((lambda b_: b_.table.__setitem__((0, 1), 99), "page"), (lambda b_: b_.kv.__setitem__(1, 900), "length")):
        c = Batch(26, [4, 3], [20, 30], 1, 64, 16, "bf16")
        change(c)
        cache, batch = make(gpu, c, 2)
        tree = batch.tree(flat(parents))
        cache.attend(batch, q, tree=tree)
        with pytest.raises(vl.VgxError, match=word):
            batch.check()
    cache, batch = make(gpu, b, 2, max_q=3)  # the first sequence has four
    batch.tree(flat(parents))
    with pytest.raises(vl.VgxError, match="length"):
        batch.check()
    # depths that no tree has: the row is written nowhere
    cache, batch = make(gpu, b, 2)
    tree = batch.tree(flat(parents))
    tree.depth[1], tree.depth[5] = 2, -1
    x = b.randn(b.ntok, 4 * 64).to(torch.bfloat16).cuda()
    q = torch.full((b.ntok, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    cache.append(batch, x, out=q, tree=tree)
    with pytest.raises(vl.VgxError, match="length"):
        batch.check()
    assert (q[[1, 5]] == 7).all() and not (q[[0, 2, 3, 4, 6]] == 7).all(-1).any()


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("half", [True, False])
def test_append_turns_by_depth(gpu, kind, half):
    """A row's queries and keys are those of a chain's row of its depth."""
    nq, kv, heads = [9, 1, 20], [40, 5, 20], 4
    b = Batch(28, nq, kv, 2, 64, 16, kind)
    parents = trees_of(nq, 29)
    cos, sin = (t.cuda() for t in tables(60, 64))
    x = (1.5 * b.randn(b.ntok, 8 * 64)).to(torch.bfloat16).cuda()
    norm = dict(q_norm=(1 + 0.3 * b.randn(64)).cuda(), k_norm=(1 + 0.3 * b.randn(64)).cuda())
    cache, batch = make(gpu, b, heads)
    q = cache.append(batch, x, cos, sin, half, tree=batch.tree(flat(parents)), **norm)
    batch.check()
    depth = sum((tr.lines(p)[0] for p in parents), [])
    for s, n in enumerate(nq):
        for r in range(n):
            t, base = int(b.qs[s]) + r, kv[s] - n
            # the same row alone, as a sequence of base + depth + 1 positions
            one = Batch(30, [1], [base + depth[t] + 1], 2, 64, 16, kind)
            c1, b1 = make(gpu, one, heads)
            q1 = c1.append(b1, x[t:t + 1], cos, sin, half, **norm)
            assert torch.equal(q[t], q1[0])
            at, to = base + depth[t], base + r
            for pool, mine in ((c1.k, cache.k), (c1.v, cache.v)):
                assert torch.equal(mine[int(b.table[s, to // 16]), :, to % 16],
                                   pool[int(one.table[0, at // 16]), :, at % 16])


@pytest.mark.parametrize("nq", [[1], [0, 5, 1, 0, 12], [64, 65, 200, 1000]])
def test_accept(gpu, nq):
    b = Batch(31, nq, nq, 1, 16, 16, "bf16")
    _, batch = make(gpu, b, 1, max_q=max(nq))
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        parents = trees_of(nq, 32 + seed, wide=True)
        tok = torch.randint(0, 3, (b.ntok,), generator=g).to(torch.int32)  # few values: equal siblings
        chosen = torch.randint(0, 3, (b.ntok,), generator=g).to(torch.int32)
        path, acc, nxt = (x.cpu() for x in batch.accept(flat(parents), tok.cuda(), chosen.cuda()))
        for s, n in enumerate(nq):
            sl = slice(int(b.qs[s]), int(b.qs[s + 1]))
            want, then = tr.accept(parents[s], tok[sl].tolist(), chosen[sl].tolist())
            assert int(acc[s]) == max(len(want) - 1, 0) and int(nxt[s]) == then
            assert path[sl].tolist() == want + [-1] * (n - len(want))
    batch.check()


def test_a_row_without_a_token_ends_the_way(gpu):
    """A masked row's -1 is not the -1 of a padded child."""
    b = Batch(31, [4, 3], [4, 3], 1, 16, 16, "bf16")
    _, batch = make(gpu, b, 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    parent = torch.tensor([-1, 0, 1, 2, -1, 0, 0], **i32)
    tokens = torch.tensor([5, 6, -1, -1, 5, -1, 7], **i32)
    chosen = torch.tensor([6, -1, -1, 3, -1, 9, 9], **i32)
    path, acc, nxt = (x.tolist() for x in batch.accept(parent, tokens, chosen))
    assert path == [0, 1, -1, -1, 0, -1, -1] and acc == [1, 0] and nxt == [-1, -1]


def layer_pools(b, n, strided=False):
    """The K and V of n layers: the batch's, and others of random values."""
    out = []
    for i in range(n):
        k, v = (ref.to_cache(b.randn(b.pages, b.kvh, b.page, b.hd), b.kind) for _ in range(2))
        if strided:
            base = torch.zeros(b.pages, 2, b.page, b.kvh, b.hd + 16, dtype=k.dtype, device="cuda")
            ks, vs = (base[:, j].transpose(1, 2)[..., :b.hd] for j in (0, 1))
            ks.copy_(k)
            vs.copy_(v)
            out.append((ks, vs))
        else:
            out.append((k.cuda(), v.cuda()))
    return out


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("kvh, hd, page, strided", [(2, 64, 16, False), (4, 96, 7, True), (1, 16, 1, False), (8, 256, 64, True)])
@pytest.mark.parametrize("layers", [1, 3])
def test_keep(gpu, kind, kvh, hd, page, strided, layers):
    check_keep(gpu, kind, kvh, hd, page, strided, layers)


def test_keep_many_layers(gpu):
    """More layers than one launch takes."""
    check_keep(gpu, "bf16", 2, 64, 16, False, 70)


def check_keep(gpu, kind, kvh, hd, page, strided, layers):
    nq, kv = [12, 1, 0, 30, 64], [12, 9, 4, 77, 500]
    b = Batch(40, nq, kv, kvh, hd, page, kind)
    pools = layer_pools(b, layers, strided)
    caches = [gpu.paged_cache(kvh, kvh, hd, kind, k, v) for k, v in pools]
    batch = caches[0].batch(*b.device(), b.ntok)
    # rows that overlap their own targets, none, all of them, and one kept in place
    paths = [[0, 2, 3, 4, 7, 11], [0], [], [0] + list(range(1, 30)), [0, 1, 5, 6, 9, 40, 41, 42, 63]]
    path = torch.full((b.ntok,), -1, dtype=torch.int32)
    for s, p in enumerate(paths):
        path[int(b.qs[s]):int(b.qs[s]) + len(p)] = torch.tensor(p, dtype=torch.int32)
    acc = torch.tensor([max(len(p) - 1, 0) for p in paths], dtype=torch.int32)
    want = [(k.cpu().clone(), v.cpu().clone()) for k, v in pools]
    old = [(k.cpu().clone(), v.cpu().clone()) for k, v in pools]
    for s, p in enumerate(paths):
        base = kv[s] - nq[s]
        for i, r in enumerate(p):
            at, to = base + r, base + i
            for (wk, wv), (ok, ov) in zip(want, old):
                for w, o in ((wk, ok), (wv, ov)):
                    w[int(b.table[s, to // page]), :, to % page] = o[int(b.table[s, at // page]), :, at % page]
    gpu.paged_layers(caches).keep(batch, path.cuda(), acc.cuda())
    batch.check()
    for (k, v), (wk, wv) in zip(pools, want):
        assert same_bits(k.cpu(), wk) and same_bits(v.cpu(), wv)


def test_keep_faults(gpu):
    """A path that goes backwards or past the rows, a count past them and a bad
    page: reported, and only what is sound is moved."""
    from vgx import lib as vl
    b = Batch(41, [6, 6, 6, 4], [26, 26, 26, 0], 1, 64, 16, "bf16")
    cache, batch = make(gpu, b, 1)
    old = cache.k.cpu().clone()
    layers = gpu.paged_layers([cache])

    def go(paths, acc, word):
        path = torch.zeros(b.ntok, dtype=torch.int32)
        for s, p in enumerate(paths):
            path[int(b.qs[s]):int(b.qs[s]) + len(p)] = torch.tensor(p, dtype=torch.int32)
        layers.keep(batch, path.cuda(), torch.tensor(acc, dtype=torch.int32).cuda())
        if word is None:
            batch.check()
        else:
            with pytest.raises(vl.VgxError, match=word):
                batch.check()

    go([[0, 0], [0], [0], [0]], [1, 0, 0, 0], "length")
    go([[0, 6], [0], [0], [0]], [1, 0, 0, 0], "length")
    go([[0, -1], [0], [0], [0]], [1, 0, 0, 0], "length")
    go([[0, 1], [0], [0], [0]], [6, 0, 0, 0], "length")
    go([[0, 1], [0], [0], [0]], [-1, 0, 0, 0], "length")
    assert torch.equal(cache.k.cpu(), old)
    go([[0, 1, 2], [0], [0], [0, 1]], [2, 0, 0, 1], None)  # (rows before position 0: nothing to move)
    assert torch.equal(cache.k.cpu(), old)
    b.table[1, 1] = 1000
    _, batch = make(gpu, b, 1)
    go([[0], [0, 2], [0, 3], [0]], [0, 1, 1, 0], "page")
    want = old.clone()
    pg = b.table[2]
    want[int(pg[21 // 16]), :, 21 % 16] = old[int(pg[23 // 16]), :, 23 % 16]
    assert torch.equal(cache.k.cpu(), want)


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("kvh, hd, page, strided", [(2, 64, 16, False), (4, 96, 7, True), (1, 16, 1, False),
                                                    (8, 256, 64, True), (8, 128, 64, False), (3, 80, 100, False)])
@pytest.mark.parametrize("part", [False, True])
def test_copy(gpu, kind, kvh, hd, page, strided, part):
    b = Batch(42, [0], [20 * page], kvh, hd, page, kind)
    pools = layer_pools(b, 3, strided)
    caches = [gpu.paged_cache(kvh, kvh, hd, kind, k, v) for k, v in pools]
    src, dst = [3, 3, 0, 19, 7], [1, 2, 21, 4, 7]
    rows = [page, 0, 1, (page + 1) // 2, page] if part else None
    old = [(k.cpu().clone(), v.cpu().clone()) for k, v in pools]
    dev = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    layers = gpu.paged_layers(caches)
    layers.copy(dev(src), dev(dst), dev(rows) if part else None)
    layers.check()
    for (k, v), (ok, ov) in zip(pools, old):
        for got, o in ((k, ok), (v, ov)):
            w = o.clone()
            for i, (a, t) in enumerate(zip(src, dst)):
                n = rows[i] if part else page
                w[t, :, :n] = o[a, :, :n]
            assert same_bits(got.cpu(), w)


def test_copy_of_many_pages_and_none(gpu):
    b = Batch(43, [0], [16 * 4000], 1, 64, 16, "bf16")
    cache, _ = make(gpu, b, 1)
    layers = gpu.paged_layers([cache])
    old = cache.k.clone()
    perm = torch.randperm(b.pages, generator=b.rng).to(torch.int32).cuda()
    src, dst = perm[:2000].contiguous(), perm[2000:4000].contiguous()
    layers.copy(src, dst)
    layers.check()
    want = old.clone()
    want[dst.long()] = old[src.long()]
    assert torch.equal(cache.k, want)
    layers.copy(src[:0], dst[:0])
    layers.check()


def test_copy_faults(gpu):
    from vgx import lib as vl
    b = Batch(44, [0], [64], 1, 64, 16, "bf16")
    cache, _ = make(gpu, b, 1)
    layers = gpu.paged_layers([cache])
    dev = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    old = cache.k.clone()
    for src, dst, rows, word in ((dev(-1), dev(0), None, "page"), (dev(0), dev(b.pages), None, "page"),
                                 (dev(0), dev(1), dev(17), "rows"), (dev(0), dev(1), dev(-1), "rows")):
        layers.copy(src, dst, rows)
        with pytest.raises(vl.VgxError, match=word):
            layers.check()
    assert torch.equal(cache.k, old)


def step_inputs(b, heads, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    width = (heads + 2 * b.kvh) * b.hd
    x = (1.5 * torch.randn(b.ntok, width, generator=g)).to(torch.bfloat16).cuda()
    head = (torch.randn(heads * b.hd, vocab, generator=g) * 0.3).to(torch.bfloat16).cuda()
    tok = torch.randint(0, vocab, (b.ntok,), generator=g).to(torch.int32).cuda()
    u = torch.rand(b.ntok, generator=g).cuda()
    return x, head, tok, u


def test_a_drafted_step(gpu):
    """append, attend, sample, accept and keep as a server runs them: the pages
    then hold what a sequence grown by the accepted rows alone would hold, and
    the next step sees the same."""
    nq, kv, heads, vocab = [12, 1, 25, 40], [40, 17, 25, 300], 4, 7
    b = Batch(45, nq, kv, 2, 64, 16, "bf16")
    parents = trees_of(nq, 46, wide=True)
    cos, sin = (t.cuda() for t in tables(400, 64))
    x, head, tok, u = step_inputs(b, heads, vocab, 47)
    caches = [make(gpu, b, heads)[0] for _ in range(2)]
    batch = caches[0].batch(*b.device(), b.ntok)
    tree = batch.tree(flat(parents))
    for c in caches:
        q = c.append(batch, x, cos, sin, tree=tree)
        o, _ = c.attend(batch, q, tree=tree)
    logits = (o @ head).float()
    chosen, kept, prob = gpu.sample(logits, u, temp=torch.full((b.ntok,), 0.8).cuda(),
                                    top_k=torch.full((b.ntok,), 3, dtype=torch.int32).cuda())
    path, acc, nxt = batch.accept(flat(parents), tok, chosen)
    gpu.paged_layers(caches).keep(batch, path, acc)
    batch.check()
    acc, path = acc.cpu().tolist(), path.cpu().tolist()
    assert max(acc) > 0 and (kept <= 3).all()
    # the accepted rows alone, appended to the old pages
    rows = [int(b.qs[s]) + path[int(b.qs[s]) + k] for s in range(4) for k in range(acc[s] + 1)]
    lens = [kv[s] - nq[s] + acc[s] + 1 for s in range(4)]
    plain, _ = make(gpu, b, heads)
    dev = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    starts = [0]
    for a in acc:
        starts.append(starts[-1] + a + 1)
    grown = plain.batch(dev(starts), dev(lens), b.table.cuda(), starts[-1])
    plain.append(grown, x[rows].contiguous(), cos, sin)
    grown.check()
    for c in caches:
        for mine, pool in ((c.k, plain.k), (c.v, plain.v)):
            for s in range(4):
                assert torch.equal(b_rows(b, s, mine, lens[s]), b_rows(b, s, pool, lens[s]))
    then = caches[1].batch(dev([0, 1, 2, 3, 4]), dev(lens), b.table.cuda(), 4)
    ref_then = plain.batch(dev([0, 1, 2, 3, 4]), dev(lens), b.table.cuda(), 4)
    q4 = torch.randn(4, heads, 64, device="cuda").to(torch.bfloat16)
    assert torch.equal(caches[1].attend(then, q4)[0], plain.attend(ref_then, q4)[0])


def b_rows(b, s, pool, count):
    pg = b.table[s, :-(-count // b.page)].long().cuda()
    return pool[pg].transpose(1, 2).reshape(-1, b.kvh, b.hd)[:count]


def test_a_captured_step(gpu):
    """The whole step in a graph, replayed with other trees, tokens and lengths
    between eager work, on its own stream."""
    from vgx import gpu as vg
    nq, heads, vocab = [12, 3, 25], 4, 9
    b = Batch(48, nq, [200, 200, 200], 2, 64, 16, "bf16")
    g = vg.GPU(0)
    cos, sin = (t.cuda() for t in tables(300, 64))
    cache = make(g, b, heads)[0]
    layers = g.paged_layers([cache])
    qs, kvlen, table = b.device()
    batch = cache.batch(qs, kvlen, table, b.ntok)
    parent = flat(trees_of(nq, 50))
    x, head, tok, u = step_inputs(b, heads, vocab, 51)
    temp = torch.full((b.ntok,), 0.7).cuda()
    tree = batch.tree(parent)
    k0, v0 = cache.k.clone(), cache.v.clone()

    def step():
        tree.update(parent)
        q = cache.append(batch, x, cos, sin, tree=tree)
        o, _ = cache.attend(batch, q, tree=tree)
        chosen, kept, prob = g.sample((o @ head).float(), u, temp=temp)
        path, acc, nxt = batch.accept(parent, tok, chosen)
        layers.keep(batch, path, acc)
        return o, chosen, kept, prob, path, acc, nxt

    step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    for i in range(4):
        parent.copy_(flat(trees_of(nq, 60 + i)))
        kvlen.copy_(torch.tensor([40 + 50 * i, 3 + i, 25 + i], dtype=torch.int32))
        y, _, t, w = step_inputs(b, heads, vocab, 70 + i)
        for a, c in ((x, y), (tok, t), (u, w)):
            a.copy_(c)
        res = []
        for run in (gr.replay, None):
            cache.k.copy_(k0)
            cache.v.copy_(v0)
            if run:
                run()
                out = [t.clone() for t in got]
            else:
                out = step()
            torch.cuda.synchronize()
            res.append((out, cache.k.clone(), cache.v.clone()))
        for a, c in zip(res[0][0], res[1][0]):
            assert torch.equal(a, c)
        assert torch.equal(res[0][1], res[1][1]) and torch.equal(res[0][2], res[1][2])
    batch.check()
    g.close()


def test_rows_behind_the_last_sequence(gpu):
    """A padded batch: rows of no sequence keep what they had."""
    nq = [5, 9]
    b = Batch(52, nq, [30, 50], 1, 64, 16, "bf16")
    parents = trees_of(nq, 53)
    cache, _ = make(gpu, b, 2)
    qs, kvlen, table = b.device()
    ntok = b.ntok + 6
    batch = cache.batch(qs, kvlen, table, ntok, max_q=9)
    pad = torch.cat([flat(parents), torch.zeros(6, dtype=torch.int32, device="cuda")])
    tree = batch.tree(pad)
    tree.depth[b.ntok:], tree.see[b.ntok:] = 5, 6
    tree.update(pad)
    assert (tree.depth[b.ntok:] == 5).all() and (tree.see[b.ntok:] == 6).all()
    q = b.randn(ntok, 2, 64).to(torch.bfloat16).cuda()
    out = torch.full((ntok, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    cache.attend(batch, q, out=out, tree=tree)
    assert (out[b.ntok:] == 3).all() and not (out[:b.ntok] == 3).all(1).any()
    batch.check()


@pytest.mark.parametrize("n", [8, 40])
def test_two_streams_at_once(gpu, n):
    nq = [n, n]
    b = Batch(54, nq, [3000, 2000], 2, 128, 64, "bf16")
    parents = flat(trees_of(nq, 55))
    cache, batch = make(gpu, b, 8)
    tree = batch.tree(parents)
    q = [b.randn(b.ntok, 8, 128).to(torch.bfloat16).cuda() for _ in range(2)]
    want = [cache.attend(batch, x, tree=tree)[0] for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attend(batch, q[i], tree=tree)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_part_of_a_batch(gpu):
    """Some of a batch's sequences, named by their entries of qstart: the rows
    before and behind them are left as they are, and are no fault."""
    nq, kv = [6, 3, 12, 5], [60, 30, 50, 90]
    b = Batch(56, nq, kv, 1, 64, 16, "bf16")
    parents = trees_of(nq, 57)
    cache, _ = make(gpu, b, 2)
    qs, kvlen, table = b.device()
    some = cache.batch(qs[1:4], kvlen[1:3], table[1:3], b.ntok)
    tree = some.tree(flat(parents))
    cos, sin = (t.cuda() for t in tables(100, 64))
    x = b.randn(b.ntok, 4 * 64).cuda()
    q = torch.full((b.ntok, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    tree.depth[:6], tree.depth[21:] = 99, -5
    cache.append(some, x, cos, sin, out=q, tree=tree)
    out = torch.full((b.ntok, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    cache.attend(some, q, out=out, tree=tree)
    some.check()
    rest = list(range(6)) + list(range(21, 26))
    assert (q[rest] == 7).all() and (out[rest] == 3).all()
    assert not (q[6:21] == 7).all(-1).any() and not (out[6:21] == 3).all(-1).any()


def check_append_past_the_start(gpu, kind, parents, kv, rotated):
    """Sequences of more rows than positions: a row before position 0 has no
    slot and is skipped; one with a slot is written, or, where it has no angle
    (its depth's position is before 0), reported and written nowhere."""
    from vgx import lib as vl
    nq, heads, hd = [len(p) for p in parents], 4, 64
    b = Batch(59, nq, kv, 2, hd, 16, kind)
    angles = [t.cuda() for t in tables(60, hd)] if rotated else []
    x = (1.5 * b.randn(b.ntok, (heads + 4) * hd)).to(torch.bfloat16).cuda()
    cache, batch = make(gpu, b, heads)
    q = torch.full((b.ntok, heads, hd), 7.0, dtype=ref.CTYPE[kind], device="cuda")
    cache.append(batch, x, *angles, out=q, tree=batch.tree(flat(parents)))
    want_k, want_v, fault = b.k.clone().cuda(), b.v.clone().cuda(), False
    for s, n in enumerate(nq):
        depth = tr.lines(parents[s])[0]
        for r in range(n):
            t, pos, at = int(b.qs[s]) + r, kv[s] - n + r, kv[s] - n + depth[r]
            lost = rotated and pos >= 0 and at < 0
            fault = fault or lost
            if pos < 0 or lost:
                assert (q[t] == 7).all(), (s, r)
                continue
            # the same row alone, as a sequence that ends at its angles' position
            one = Batch(60, [1], [max(at, 0) + 1], 2, hd, 16, kind)
            c1, b1 = make(gpu, one, heads)
            assert torch.equal(q[t], c1.append(b1, x[t:t + 1], *angles)[0]), (s, r)
            src = (int(one.table[0, max(at, 0) // 16]), slice(None), max(at, 0) % 16)
            dst = (int(b.table[s, pos // 16]), slice(None), pos % 16)
            want_k[dst], want_v[dst] = c1.k[src], c1.v[src]
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    if fault:
        with pytest.raises(vl.VgxError, match="length"):
            batch.check()
    else:
        batch.check()
    return fault


@pytest.mark.parametrize("kind", ["bf16", "q8"])
@pytest.mark.parametrize("rotated", [False, True])
def test_append_of_more_rows_than_positions(gpu, kind, rotated):
    wide = [[-1] + [0] * 4, [-1, 0, 0, 1, 3, 4, 5, 6, 7, 8, 9, 2], [-1, 0, 1]]
    assert check_append_past_the_start(gpu, kind, wide, [3, 7, 0], rotated) == rotated
    chains = [list(range(-1, n - 1)) for n in (5, 12, 3)]  # a row's depth is its number
    assert not check_append_past_the_start(gpu, kind, chains, [3, 7, 0], rotated)


def test_a_batch_over_caches_of_other_strides(gpu):
    """What a batch keeps of one cache's calls does not serve another's whose
    rows lie further apart: the same results as by a batch of its own."""
    nq, kv, heads, hd = [61, 20, 2], [3000, 2500, 3500], 2, 64
    b = Batch(61, nq, kv, 1, hd, 16, "f16")
    parents = trees_of(nq, 62)
    row = 1 << 25  # 64 MiB between a page's positions
    pool = torch.zeros(16 * row, dtype=torch.float16, device="cuda")
    far = [pool.as_strided((b.pages, 1, 16, hd), (hd, hd, row, 1), i * b.pages * hd) for i in range(2)]
    far[0].copy_(b.k)
    far[1].copy_(b.v)
    spread = gpu.paged_cache(heads, 1, hd, "f16", *far)
    near, own = make(gpu, b, heads, max_q=61, max_kv=3500)
    q = b.randn(b.ntok, heads, hd).to(torch.float16).cuda()
    want = near.attend(own, q, tree=own.tree(flat(parents)))[0]
    both = spread.batch(*b.device(), b.ntok, max_q=61, max_kv=3500)
    check(gpu, b, heads, parents, q=q.cpu(), cache=spread, batch=both)
    assert torch.equal(near.attend(both, q, tree=both.tree(flat(parents)))[0], want)


def test_workspace_of_many_trees(gpu):
    """Where the tiles alone fill the chip their splits end: 16 rounds of
    resident workgroups (two a CU, three for heads of 64), 128 columns each, of
    hd + 2 floats, whatever the bounds."""
    import ctypes

    from test_paged_refusals import batch, cache
    from vgx import lib as vl
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    for heads, kvh, hd in ((32, 8, 128), (16, 8, 64), (16, 2, 64), (8, 4, 96), (4, 1, 256)):
        c = cache(heads=heads, kv_heads=kvh, head_dim=hd, num_pages=1 << 20, k_row=hd, v_row=hd, k_head=16 * hd,
                  v_head=16 * hd, k_page=16 * hd * kvh, v_page=16 * hd * kvh)
        for nseq in (2, 24, 128, 256, 1000):
            for bound in (300, 8192, 32768, 1 << 20):
                for window in (0, 4096):
                    b = batch(nseq=nseq, ntok=64 * nseq, max_q=64, max_kv=bound, table_cols=1 << 16, table_stride=1 << 16)
                    ws = vl.load().vgx_paged_attn_tree_ws(gpu.ctx, ctypes.byref(c), ctypes.byref(b), window)
                    most = 16 * cus * (3 if hd <= 64 else 2) * 128 * (hd + 2) * 4 + b.ntok * heads * 8
                    assert ws <= most, (heads, kvh, hd, nseq, bound, window, ws)


def test_many_trees_that_fill_the_chip(gpu):
    """1600 workgroups of tiles, their splits ended: short sequences and two
    that take several."""
    nq = [17] * 200
    kv = [17 + i * 37 % 200 for i in range(200)]
    kv[3], kv[150] = 3001, 1409
    b = Batch(63, nq, kv, 4, 64, 16, "bf16")
    b.table = torch.nn.functional.pad(b.table, (0, 563 - b.table.shape[1]), value=-1)  # (room for the bound)
    check(gpu, b, 32, trees_of(nq, 64), max_q=17, max_kv=9000)
