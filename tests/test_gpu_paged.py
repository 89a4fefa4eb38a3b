"""The paged cache's append and attention against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

import paged_ref as ref
from paged_ref import STEP, Batch

pytestmark = pytest.mark.gpu


def make(gpu, b, heads, k=None, v=None, **kw):
    c = gpu.paged_cache(heads, b.kvh, b.hd, b.kind, (b.k if k is None else k).cuda() if k is None else k,
                        (b.v if v is None else v).cuda() if v is None else v)
    return c, c.batch(*b.device(), b.ntok, **kw)


def tables(npos, rot, seed=3):
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand(npos, rot // 2, generator=g, dtype=torch.float64) * 6.28
    return torch.cos(ang).float(), torch.sin(ang).float()


def check_append(gpu, b, heads, act, rot, half, norm, x=None, cache=None, batch=None):
    width = (heads + 2 * b.kvh) * b.hd
    if x is None:
        x = b.randn(b.ntok, width) * 1.5
        x = torch.clamp(torch.round(x * 256), -32768, 32767).to(torch.int16) if act == torch.int16 else x.to(act)
    qn = 1 + 0.3 * b.randn(b.hd) if norm else None
    kn = 1 + 0.3 * b.randn(b.hd) if norm else None
    cos, sin = tables(max(b.kv + [1]), rot) if rot else (None, None)
    if cache is None:
        cache, batch = make(gpu, b, heads)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    out = torch.full((b.ntok + 2, heads, b.hd), 7.0, dtype=ref.CTYPE[b.kind], device="cuda")
    cache.append(batch, x.cuda(), dev(cos), dev(sin), half, dev(qn), dev(kn), out=out)
    batch.check()
    q, k, v, mag = ref.append(b, x, heads, cos, sin, half, qn, kn)
    # 32-bit: head_dim additions, the root, three products and the rotation's two
    err = mag * (b.hd + 24) * 2.0 ** -24
    got_q, got_k, got_v = out.cpu(), cache.k.cpu(), cache.v.cpu()
    want_k, want_v = b.k.clone(), b.v.clone()
    for s, (n, m) in enumerate(zip(b.nq, b.kv)):
        for r in range(n):
            pos, t = m - n + r, int(b.qs[s]) + r
            if pos < 0:
                assert (got_q[t] == 7.0).all()
                continue
            pg, sl = int(b.table[s, pos // b.page]), pos % b.page
            tiny = 2.0 ** -25 if b.kind != "bf16" else 0.0  # float16's subnormal step
            half_q = ref.HALF_STEP[ref.CTYPE[b.kind]]
            assert ((got_q[t].double() - q[t]).abs() <= q[t].abs() * half_q + 2 * err[t, :heads] + tiny).all()
            for got, val, e, want in ((got_k, k, err[t, heads:], want_k), (got_v, v, v[t].abs() * 2.0 ** -23, want_v)):
                g = got[pg, :, sl]
                if b.kind == "q8":
                    c = val[t].clamp(-128 * STEP, 127 * STEP)
                    assert ((ref.value(g) - c).abs() <= STEP / 2 + e).all()
                else:
                    assert ((g.double() - val[t]).abs() <= val[t].abs() * half_q + 2 * e + tiny).all()
                want[pg, :, sl] = g
    # nothing else of the pool, nor the rows behind the last sequence, was written
    assert torch.equal(got_k.view(torch.uint8), want_k.view(torch.uint8))
    assert torch.equal(got_v.view(torch.uint8), want_v.view(torch.uint8))
    assert (got_q[int(b.qs[-1]):] == 7.0).all()
    return x, cache, batch


ACTS = [torch.int16, torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("act", ACTS)
def test_append_types(gpu, kind, act):
    b = Batch(1, [1, 5, 0, 33], [17, 5, 9, 70], 2, 64, 16, kind)
    check_append(gpu, b, 4, act, 64, True, True)


@pytest.mark.parametrize("heads, kvh, hd", [(8, 4, 96), (3, 1, 16), (6, 2, 80), (5, 5, 128), (4, 2, 144), (2, 1, 256)])
@pytest.mark.parametrize("half", [True, False])
def test_append_heads(gpu, heads, kvh, hd, half):
    b = Batch(2, [1, 3, 20], [300, 3, 41], kvh, hd, 32, "bf16")
    check_append(gpu, b, heads, torch.float32, hd, half, True)
    check_append(gpu, Batch(3, [2, 1], [2, 65], kvh, hd, 7, "q8"), heads, torch.int16, hd // 32 * 16, half, False)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 100, 4096])
def test_append_pages(gpu, page):
    b = Batch(4, [4, 130, 1], [4, 333, 1000], 2, 32, page, "f16")
    check_append(gpu, b, 2, torch.float16, 0, True, False)


def test_append_more_rows_than_positions(gpu):
    """Rows before position 0 have no place: nothing of theirs is written."""
    b = Batch(5, [6, 2, 3], [2, 0, 3], 1, 48, 16, "bf16")
    check_append(gpu, b, 2, torch.bfloat16, 48, True, True)


def test_append_many_sequences(gpu):
    rng = np.random.default_rng(0)
    nq = rng.integers(0, 4, 200).tolist()
    kv = [n + int(m) for n, m in zip(nq, rng.integers(0, 40, 200))]
    check_append(gpu, Batch(6, nq, kv, 1, 64, 16, "bf16"), 2, torch.int16, 64, True, True)


def strided_pools(b):
    """Position-major pages with room between the rows, both in one allocation."""
    base = torch.zeros(b.pages, 2, b.page, b.kvh, b.hd + 16, dtype=b.k.dtype, device="cuda")
    k, v = (base[:, i].transpose(1, 2)[..., :b.hd] for i in (0, 1))
    k.copy_(b.k)
    v.copy_(b.v)
    return k, v


def test_strides(gpu):
    b = Batch(7, [3, 40, 1], [100, 40, 64], 2, 64, 16, "bf16")
    k, v = strided_pools(b)
    cache, batch = make(gpu, b, 4, k=k, v=v)
    wide = torch.zeros(b.ntok, 640, dtype=torch.bfloat16)
    wide[:, 64:576] = (b.randn(b.ntok, 512)).to(torch.bfloat16)
    x, cos_sin = wide[:, 64:576], tables(100, 64)
    q = torch.empty(b.ntok, 4, 96, dtype=torch.bfloat16, device="cuda").flatten(1)[:, :256]
    xd = wide.cuda()[:, 64:576]
    got = cache.append(batch, xd, cos_sin[0].cuda(), cos_sin[1].cuda(), out=q)
    dense, dbatch = make(gpu, b, 4)
    want = dense.append(dbatch, x.contiguous().cuda(), cos_sin[0].cuda(), cos_sin[1].cuda())
    assert torch.equal(got, want.flatten(1))
    assert torch.equal(k, dense.k) and torch.equal(v, dense.v)
    o = torch.empty(b.ntok, 300, dtype=torch.bfloat16, device="cuda")[:, 8:264]
    with pytest.raises(Exception):  # rows 600 bytes apart: not whole 16-byte steps
        cache.attend(batch, q, out=o)
    o = torch.empty(b.ntok, 512, dtype=torch.bfloat16, device="cuda")[:, 8:264]
    cache.attend(batch, q, out=o)
    assert torch.equal(o, dense.attend(dbatch, want)[0])


def check_attn(gpu, b, heads, window=0, scale=None, q=None, out=None, cache=None, batch=None, spread=2.0):
    ct = ref.CTYPE[b.kind]
    if q is None:
        q = (spread * b.randn(b.ntok, heads, b.hd)).to(ct)
    if cache is None:
        cache, batch = make(gpu, b, heads)
    o, lse = cache.attend(batch, q.cuda(), scale=scale or 0.0, window=window, lse=True, out=out)
    batch.check()
    want, wl, mag, dots = ref.attend(b, q, heads, scale, window)
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


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("heads, kvh, hd", [(8, 4, 96), (16, 2, 64), (4, 1, 128), (3, 3, 16), (6, 2, 80), (5, 1, 144),
                                            (2, 1, 256), (32, 1, 32)])
def test_attn_tokens(gpu, kind, heads, kvh, hd):
    b = Batch(11, [1, 1, 1, 1, 1], [1, 31, 33, 130, 700], kvh, hd, 16, kind)
    check_attn(gpu, b, heads)


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("heads, kvh, hd", [(8, 4, 96), (16, 2, 64), (4, 1, 128), (3, 3, 16), (6, 2, 80), (5, 1, 144),
                                            (2, 1, 256)])
def test_attn_chunks(gpu, kind, heads, kvh, hd):
    b = Batch(12, [130, 1, 0, 64, 7], [130, 500, 20, 100, 263], kvh, hd, 32, kind)
    check_attn(gpu, b, heads)


@pytest.mark.parametrize("page", [1, 5, 16, 48, 64, 1000])
@pytest.mark.parametrize("nq", [[2, 1], [90, 45]])
def test_attn_pages(gpu, page, nq):
    check_attn(gpu, Batch(13, nq, [301, 97], 2, 64, page, "f16"), 4)


@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 200, 5000])
@pytest.mark.parametrize("nq", [[1, 3, 1, 2], [150, 40, 1, 70]])
def test_attn_window(gpu, window, nq):
    check_attn(gpu, Batch(14, nq, [150, 333, 900, 70], 2, 64, 16, "bf16"), 4, window=window)


@pytest.mark.parametrize("nq", [[5, 2, 1], [70, 40, 1]])
def test_attn_empty_rows(gpu, nq):
    """More rows than positions: the first see nothing and give zeros."""
    check_attn(gpu, Batch(15, nq, [3, 0, 1], 2, 64, 16, "bf16"), 4)


@pytest.mark.parametrize("n", [1, 6, 40])
def test_attn_long_splits(gpu, n):
    """Few sequences, many keys: the keys are split over workgroups."""
    b = Batch(16, [n, 1], [9000, 2500], 2, 64, 64, "bf16")
    cache, batch = make(gpu, b, 4)
    o = check_attn(gpu, b, 4, cache=cache, batch=batch)
    assert batch.ws and min(batch.ws.values()) > 0  # the split path ran
    # and without the workspace
    import ctypes
    from vgx import lib as vl
    q = (2.0 * b.randn(b.ntok, 4, b.hd)).to(torch.bfloat16).cuda()
    got = torch.empty_like(o)
    r = vl.PagedQuery(q.data_ptr(), 256, 0.0, 0, vl.E_BF16, got.data_ptr(), 256, 0, 0, 0)
    vl.check(vl.load().vgx_paged_attn(gpu.ctx, cache.ref, batch.ref, ctypes.byref(r)))
    want = cache.attend(batch, q)[0]
    # both within the same bound of the definition, so within twice of one another
    w, _, mag, dots = ref.attend(b, q.cpu(), 4)
    bound = 2 * ref.attn_bound(b, torch.bfloat16, w, mag, dots)
    assert ((got.double() - want.double()).abs().cpu().view_as(w) <= bound).all()


@pytest.mark.parametrize("nq", [[1, 2], [80, 3]])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38])
def test_attn_behind_the_end(gpu, nq, bad):
    """What the last page holds behind a sequence's end, and the pages that
    are not its own, do not reach its rows."""
    b = Batch(17, nq, [85, 37], 2, 64, 32, "bf16")
    clean = b.k.clone(), b.v.clone()
    used = torch.zeros(b.pages, b.page, dtype=torch.bool)
    for s, m in enumerate(b.kv):
        for p in range(m):
            used[int(b.table[s, p // b.page]), p % b.page] = True
    q = (2 * b.randn(b.ntok, 4, 64)).to(torch.bfloat16)
    want = make(gpu, b, 4)
    want = want[0].attend(want[1], q.cuda())[0]
    for t in (b.k, b.v):
        t.masked_fill_(~used[:, None, :, None], bad)
    got = make(gpu, b, 4)
    assert torch.equal(got[0].attend(got[1], q.cuda())[0], want)
    b.k, b.v = clean


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("nq, window", [([4, 2], 0), ([100, 30], 0), ([100, 30], 20), ([3, 1], 7)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attn_masked_values(gpu, kind, nq, window, bad):
    """A NaN or infinity at a position reaches only the rows that see it."""
    b = Batch(18, nq, [140, 61], 2, 64, 16, kind)
    q = (2 * b.randn(b.ntok, 4, 64)).to(ref.CTYPE[kind])
    want, _, mag, dots = ref.attend(b, q, 4, None, window)
    bound = ref.attn_bound(b, ref.CTYPE[kind], want, mag, dots)
    at = [(0, 138), (0, 110), (1, 59), (1, 45)]
    for s, p in at:
        pg, sl = int(b.table[s, p // 16]), p % 16
        b.k[pg, :, sl, 5] = bad
        b.v[pg, :, sl, 9] = bad
    c, bt = make(gpu, b, 4)
    got = c.attend(bt, q.cuda(), window=window)[0].cpu().double().view_as(want)
    for s, (n, m) in enumerate(zip(b.nq, b.kv)):
        for r in range(n):
            pos, t = m - n + r, int(b.qs[s]) + r
            sees = any(ss == s and p <= pos and (not window or p > pos - window) for ss, p in at)
            if sees:
                assert not torch.isfinite(got[t, :, 9]).any()
            else:
                assert ((got[t] - want[t]).abs() <= bound[t]).all(), (s, r)


def test_attn_scores_past_every_exponent(gpu):
    """Scores of +-30000: weights of one key, no overflow."""
    b = Batch(19, [1, 90], [200, 90], 1, 64, 16, "bf16")
    q = (100 * b.randn(b.ntok, 2, 64)).to(torch.bfloat16)
    b.k = (30 * b.k.float()).to(torch.bfloat16)
    o, _ = (lambda c: c[0].attend(c[1], q.cuda()))(make(gpu, b, 2))
    want, _, mag, dots = ref.attend(b, q, 2)
    assert torch.isfinite(o).all()
    bound = ref.attn_bound(b, torch.bfloat16, want, mag, dots)
    assert ((o.cpu().double().view_as(want) - want).abs() <= bound).all()


@pytest.mark.parametrize("kind", ["bf16", "q8"])
@pytest.mark.parametrize("nq", [[1, 1], [70, 3]])
def test_attn_q16_out(gpu, kind, nq):
    """The output as vgx_gemm's input; rows behind the last sequence stay."""
    b = Batch(20, nq, [300, 50], 2, 96, 16, kind)
    out = torch.full((b.ntok + 3, 4 * 96), 77, dtype=torch.int16, device="cuda")
    check_attn(gpu, b, 4, out=out)
    assert (out[b.ntok:] == 77).all()


def test_rows_behind_the_last_sequence(gpu):
    b = Batch(21, [2, 60, 0], [20, 90, 5], 2, 64, 16, "bf16")
    cache, _ = make(gpu, b, 4)
    batch = cache.batch(*b.device(), b.ntok + 9)  # nine rows of nobody's
    q = torch.randn(b.ntok + 9, 4, 64, device="cuda").to(torch.bfloat16)
    out = torch.full((b.ntok + 9, 256), 5.0, dtype=torch.bfloat16, device="cuda")
    before = cache.k.clone()
    cache.attend(batch, q, out=out)
    assert (out[b.ntok:] == 5).all() and not (out[:b.ntok] == 5).all(1).any()
    x = torch.randn(b.ntok + 9, 512, device="cuda")
    qo = torch.full((b.ntok + 9, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    cache.append(batch, x, out=qo)
    assert (qo[b.ntok:] == 5).all()
    same = (cache.k == before).all(-1).all(1)
    assert int((~same).sum()) == sum(b.nq)
    batch.check()


def test_nothing_to_do(gpu):
    b = Batch(22, [0, 0], [5, 0], 2, 64, 16, "bf16")
    cache, batch = make(gpu, b, 4)
    assert cache.append(batch, torch.empty(0, 512, device="cuda")).shape == (0, 4, 64)
    o, z = cache.attend(batch, torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), lse=True)
    assert o.shape == (0, 256) and z.shape == (0, 4)


def test_far_pages(gpu):
    """Offsets past 32 bits: pages 6 GiB apart in the pool."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 14 GiB")
    b = Batch(23, [1, 40], [70, 64], 1, 64, 16, "bf16")
    far = 3 << 30  # elements
    base = torch.empty(far + (b.pages + 1) * 1024, dtype=torch.bfloat16, device="cuda")
    step = far // (b.pages - 1) // 8 * 8
    assert step * (b.pages - 1) * 2 > 1 << 32
    k = base.as_strided((b.pages, 1, 16, 64), (step, 1024, 64, 1))
    v = base.as_strided((b.pages, 1, 16, 64), (step, 1024, 64, 1), 1024)
    k.copy_(b.k)
    v.copy_(b.v)
    cache, batch = make(gpu, b, 4, k=k, v=v)
    check_append(gpu, b, 4, torch.float32, 64, True, True, cache=cache, batch=batch)
    b.k, b.v = k.cpu(), v.cpu()
    check_attn(gpu, b, 4, cache=cache, batch=batch)


def test_faults_are_reported(gpu):
    """A length past the table and a page outside the pool raise at check();
    neither's rows are written, every other sequence's are."""
    from vgx import lib as vl
    b = Batch(24, [1, 1, 1], [20, 40, 33], 2, 64, 16, "bf16")
    cache, batch = make(gpu, b, 4)
    qs, kv, table = b.device()
    x = torch.randn(3, 512, device="cuda")
    q = torch.randn(3, 4, 64, device="cuda").to(torch.bfloat16)
    good = cache.attend(batch, q)[0]
    kv2 = kv.clone()
    kv2[1] = 10 ** 6
    bad = cache.batch(qs, kv2, table, 3)
    before, before_v = cache.k.clone(), cache.v.clone()
    cache.append(bad, x)
    with pytest.raises(vl.VgxError, match="length"):
        bad.check()
    bad.check()  # cleared
    changed = (cache.k != before).any(-1).any(1).nonzero()
    assert {int(p) for p in changed[:, 0]} == {int(b.table[0, 1]), int(b.table[2, 2])}
    cache.k.copy_(before)
    cache.v.copy_(before_v)
    t2 = table.clone()
    t2[1, 2] = b.pages
    t2[2, 2] = -1
    bad = cache.batch(qs, kv, t2, 3)
    o = cache.attend(bad, q)[0]
    with pytest.raises(vl.VgxError, match="page"):
        bad.check()
    assert torch.equal(o[0], good[0])
    before = cache.k.clone()
    cache.append(bad, x)
    with pytest.raises(vl.VgxError, match="page"):
        bad.check()
    changed = (cache.k != before).any(-1).any(1).nonzero()
    assert {int(p) for p in changed[:, 0]} == {int(b.table[0, 1])}


def test_bounds_are_held(gpu):
    """A sequence longer than max_q or max_kv promised: reported, in bounds."""
    from vgx import lib as vl
    b = Batch(25, [3, 40], [20, 90], 2, 64, 16, "bf16")
    cache, _ = make(gpu, b, 4)
    q = torch.randn(b.ntok, 4, 64, device="cuda").to(torch.bfloat16)
    for kw in (dict(max_q=4), dict(max_kv=64)):
        batch = cache.batch(*b.device(), b.ntok, **kw)
        cache.attend(batch, q)
        with pytest.raises(vl.VgxError, match="length"):
            batch.check()


def test_other_stream(gpu):
    """On a side stream, with the default stream busy; the context's own
    stream is what it was."""
    from vgx import lib as vl
    b = Batch(26, [1, 50], [3000, 80], 2, 64, 16, "bf16")
    cache, batch = make(gpu, b, 4)
    q = torch.randn(b.ntok, 4, 64, device="cuda").to(torch.bfloat16)
    want = cache.attend(batch, q)[0]
    was = vl.load().vgx_ctx_stream(gpu.ctx)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [cache.attend(batch, q)[0] for _ in range(4)]
    assert vl.load().vgx_ctx_stream(gpu.ctx) == was
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_graph_replays_with_new_lengths(gpu):
    """A captured append + attention, replayed as the sequences grow; two
    graphs captured from one batch, replayed in turn."""
    b = Batch(27, [1, 1, 1], [100, 37, 2000], 2, 64, 16, "bf16", spare=8)
    cache, _ = make(gpu, b, 4)
    qs, kv, table = b.device()
    table = torch.cat([table, torch.arange(b.pages - 3, b.pages, dtype=torch.int32).cuda()[:, None]], 1)
    for s in range(3):  # a spare page after each sequence's last
        table[s, -(-b.kv[s] // 16)] = b.pages - 3 + s
    batch = cache.batch(qs, kv, table, 3, max_q=1, max_kv=2016)
    x = torch.randn(3, 512, device="cuda")
    cos, sin = (t.cuda() for t in tables(2100, 64))

    def step():
        q = cache.append(batch, x, cos, sin)
        return cache.attend(batch, q)[0]

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step()
        graphs.append((g, o))
    for i in range(4):
        kv += 1
        x.copy_(torch.randn(3, 512, device="cuda"))
        for g, o in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, step()), i
    batch.check()


def test_a_step_with_the_quantised_path(gpu):
    """qkv from vgx_gemm (q16), append, attention, and its q16 output into
    vgx_gemm: a chunk at once equals the same tokens one after another."""
    import oracle as o
    from vgx import mmcf
    rng = np.random.default_rng(5)
    heads, kvh, hd, dim = 8, 4, 96, 768

    def mat(r, c):
        q, unit, plane = mmcf.q8_per_row(rng.standard_normal((r, c)).astype(np.float32) * 0.03)
        return gpu.upload(mmcf.Matrix("q8", r, c, (q.view(np.uint8) ^ 0x80).ravel(), unit, True, plane))

    wqkv, wo = mat((heads + 2 * kvh) * hd, dim), mat(dim, heads * hd)
    x = torch.from_numpy(np.stack([o.quantize_act(rng.standard_normal(dim).astype(np.float32)) for _ in range(40)])).cuda()
    cos, sin = (t.cuda() for t in tables(64, hd))
    qn = torch.rand(hd, device="cuda") + 0.5
    res = {}
    for mode in ("chunk", "tokens"):
        b = Batch(28, [40], [40], kvh, hd, 16, "bf16")
        cache, batch = make(gpu, b, heads)
        qs, kv, table = b.device()
        if mode == "chunk":
            q = cache.append(batch, gpu.gemm(wqkv, x), cos, sin, q_norm=qn, k_norm=qn)
            att = cache.attend(batch, q, out=torch.empty(40, heads * hd, dtype=torch.int16, device="cuda"))[0]
            res[mode] = gpu.gemm(wo, att, x)
        else:
            outs = []
            for t in range(40):
                one = cache.batch(torch.tensor([0, 1], dtype=torch.int32).cuda(),
                                  torch.tensor([t + 1], dtype=torch.int32).cuda(), table, 1)
                q = cache.append(one, gpu.gemm(wqkv, x[t:t + 1].contiguous()), cos, sin, q_norm=qn, k_norm=qn)
                att = cache.attend(one, q, out=torch.empty(1, heads * hd, dtype=torch.int16, device="cuda"))[0]
                outs.append(gpu.gemm(wo, att, x[t:t + 1].contiguous()))
            res[mode] = torch.cat(outs)
        pool = cache.k.clone(), cache.v.clone()
        res[mode + "kv"] = pool
    assert all(torch.equal(a, c) for a, c in zip(res["chunkkv"], res["tokenskv"]))
    # attention's values are averages of V (|V| below 5 here), each side off by
    # at most 2^-8 of that: the projection sums 768 of them times 0.03-sized
    # weights, in root mean square 2^-8 * 5 * 0.03 * sqrt(768) / sqrt(3) < 0.01
    d = (res["chunk"].float() - res["tokens"].float()) / 256
    assert float(d.square().mean().sqrt()) < 0.02 and float(d.abs().max()) < 0.15


def test_shared_prefix(gpu):
    """Two sequences whose tables name the same first pages."""
    b = Batch(30, [1, 1], [100, 100], 2, 64, 16, "bf16")
    b.table[1, :3] = b.table[0, :3]
    check_attn(gpu, b, 8)
    b = Batch(31, [40, 70], [120, 120], 2, 64, 16, "bf16")
    b.table[1, :3] = b.table[0, :3]
    check_attn(gpu, b, 4)


def test_capture_without_a_call_before(gpu):
    """The first calls of a context and of a batch inside a capture."""
    from vgx import gpu as vg
    b = Batch(32, [1, 2], [1500, 90], 2, 128, 16, "f16")
    g = vg.GPU(0)
    cache = g.paged_cache(8, 2, 128, "f16", b.k.cuda(), b.v.cuda())
    batch = cache.batch(*b.device(), b.ntok)
    x = torch.randn(b.ntok, 12 * 128, device="cuda")
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        q = cache.append(batch, x)
        o = cache.attend(batch, q)[0]
    for _ in range(3):
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, cache.attend(batch, cache.append(batch, x))[0])
    batch.check()
    g.close()


@pytest.mark.parametrize("hd, kvh, heads", [(64, 2, 4), (128, 1, 4)])
def test_results_repeat(gpu, hd, kvh, heads):
    """The same call gives the same bits, split or not."""
    b = Batch(33, [1, 3, 1], [5000, 700, 64], kvh, hd, 16, "q8")
    cache, batch = make(gpu, b, heads)
    q = torch.randn(b.ntok, heads, hd, device="cuda").half()
    want = cache.attend(batch, q, lse=True)
    for _ in range(20):
        got = cache.attend(batch, q, lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_drafted_decode(gpu):
    """A step as a server runs it: the rows' projections (vgx_gemm), append,
    attend, the head and the drafts' check, with the lengths kept on the
    device.  Greedy sequences give the tokens of decoding one at a time,
    whatever was drafted."""
    import oracle as o
    from vgx import mmcf
    rng = np.random.default_rng(9)
    heads, kvh, hd, dim, vocab, nseq, steps = 4, 2, 64, 128, 512, 3, 14

    def mat(r, c, s):
        q, unit, plane = mmcf.q8_per_row(rng.standard_normal((r, c)).astype(np.float32) * s)
        return gpu.upload(mmcf.Matrix("q8", r, c, (q.view(np.uint8) ^ 0x80).ravel(), unit, True, plane))

    wqkv, wo, head = mat((heads + 2 * kvh) * hd, dim, 0.08), mat(dim, heads * hd, 0.08), mat(vocab, dim, 0.2)
    emb = torch.from_numpy(np.stack([o.quantize_act(rng.standard_normal(dim).astype(np.float32))
                                     for _ in range(vocab)])).cuda()
    cos, sin = (t.cuda() for t in tables(64, hd))
    table = torch.randperm(nseq * 4, generator=torch.Generator().manual_seed(1)).int().view(nseq, 4).cuda()
    zeros = torch.zeros(nseq, device="cuda")  # greedy

    def logits(cache, batch, tokens):
        x = emb[tokens.long()].contiguous()
        q = cache.append(batch, gpu.gemm(wqkv, x), cos, sin)
        att = cache.attend(batch, q, out=torch.empty(len(tokens), heads * hd, dtype=torch.int16, device="cuda"))[0]
        return gpu.gemm(head, gpu.gemm(wo, att, x))

    def cache_of():
        k = torch.zeros(nseq * 4, kvh, 16, hd, dtype=torch.bfloat16, device="cuda")
        return gpu.paged_cache(heads, kvh, hd, "bf16", k, k.clone())

    first = torch.tensor([5, 77, 300], dtype=torch.int32).cuda()
    # one token at a time
    cache, kv = cache_of(), torch.zeros(nseq, dtype=torch.int32).cuda()
    qs = torch.arange(nseq + 1, dtype=torch.int32).cuda()
    batch = cache.batch(qs, kv, table, nseq, max_q=1)
    tok, want = first, [first.cpu()]
    for _ in range(steps):
        kv += 1
        tok = gpu.argmax_rows(logits(cache, batch, tok))
        want.append(tok.cpu())
    want = torch.stack(want, 1)  # (nseq, steps + 1)
    # drafts: the right tokens, spoilt at some places; ragged numbers of them
    for spoil in (0.0, 0.4, 1.0):
        cache, kv = cache_of(), torch.zeros(nseq, dtype=torch.int32).cuda()
        got = [[int(t)] for t in first]
        while min(len(g) for g in got) <= steps:
            rows, starts = [], [0]
            for s in range(nseq):
                n = int(rng.integers(0, 5))
                d = [int(want[s, min(len(got[s]) + i, steps)]) for i in range(n)]
                d = [int(rng.integers(0, vocab)) if rng.random() < spoil else t for t in d]
                rows += [got[s][-1]] + d
                starts.append(len(rows))
            qs = torch.tensor(starts, dtype=torch.int32).cuda()
            tokens = torch.tensor(rows, dtype=torch.int32).cuda()
            kv += qs[1:] - qs[:-1]
            batch = cache.batch(qs, kv, table, len(rows), max_q=5)
            l = logits(cache, batch, tokens)
            u = torch.rand(len(rows), device="cuda")
            acc, nxt, prob = gpu.draft_verify(qs, tokens, l, u, zeros, temp=zeros)
            batch.check()
            kv -= qs[1:] - qs[:-1] - 1 - acc  # refused drafts leave the cache
            for s in range(nseq):
                a = int(acc[s])
                got[s] += rows[starts[s] + 1:starts[s] + 1 + a] + [int(nxt[s])]
            if max(len(g) for g in got) > 56:
                break
        for s in range(nseq):
            assert got[s][:steps + 1] == want[s].tolist()


@pytest.mark.parametrize("kind", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("hd", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("nq", [[2, 4, 1, 0], [6, 3, 1, 5]])
def test_attn_drafts(gpu, kind, hd, nq):
    """17 to 48 columns a KV head (8 query heads each): two and three blocks of
    columns, over one split and over several."""
    check_attn(gpu, Batch(34, nq, [70, 33, 500, 9], 1, hd, 16, kind), 8)
    b = Batch(35, nq, [70, 2100, 500, 9], 1, hd, 16, kind)
    check_attn(gpu, b, 8, window=600 if kind == "q8" else 0)


def test_attn_masked_values_drafts(gpu):
    b = Batch(36, [6, 5], [140, 61], 1, 64, 16, "bf16")
    q = (2 * b.randn(b.ntok, 8, 64)).to(torch.bfloat16)
    want, _, mag, dots = ref.attend(b, q, 8)
    bound = ref.attn_bound(b, torch.bfloat16, want, mag, dots)
    b.v[int(b.table[0, 8]), :, 9, 3] = math.nan   # position 137 of 140
    b.v[int(b.table[1, 3]), :, 10, 60] = -math.inf  # position 58 of 61
    c, bt = make(gpu, b, 8)
    got = c.attend(bt, q.cuda())[0].cpu().double().view_as(want)
    for t in range(11):
        dim, sees = (3, t >= 3) if t < 6 else (60, t >= 6 + 2)
        if sees:
            assert not torch.isfinite(got[t, :, dim]).any()
        rest = [d for d in range(64) if d != dim or not sees]
        assert ((got[t][:, rest] - want[t][:, rest]).abs() <= bound[t][:, rest]).all()


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_attn_many_sequences(gpu, kind):
    """More workgroups than half the CUs, one a sequence and head."""
    rng = np.random.default_rng(2)
    kv = rng.integers(1, 400, 80).tolist()
    check_attn(gpu, Batch(37, [1] * 80, kv, 2, 64, 16, kind), 4)
    nq = rng.integers(0, 3, 80).tolist()
    check_attn(gpu, Batch(38, nq, [k + 2 for k in kv], 2, 128, 32, kind), 8)


def test_attn_chunks_split(gpu):
    """A chunk of few tiles over a long cache: its keys are split too."""
    b = Batch(39, [90, 70], [3000, 1200], 1, 128, 64, "f16")
    cache, batch = make(gpu, b, 2)
    check_attn(gpu, b, 2, cache=cache, batch=batch)
    assert min(batch.ws.values()) > 0
    check_attn(gpu, Batch(40, [150], [4000], 2, 64, 16, "q8"), 4, window=900)


@pytest.mark.parametrize("kind, hd, heads, kvh", [("bf16", 64, 4, 2), ("q8", 128, 8, 1), ("f16", 80, 3, 3),
                                                  ("bf16", 96, 36, 2), ("bf16", 256, 4, 2), ("f16", 32, 50, 1)])
def test_attn_prompts_and_tokens(gpu, kind, hd, heads, kvh):
    """Chunks and single tokens in one batch, with long caches among the short
    rows' sequences: both kernels run, and both split."""
    b = Batch(41, [100, 1, 2, 0, 1, 61], [150, 3000, 2500, 7, 9, 1700], kvh, hd, 16, kind)
    cache, batch = make(gpu, b, heads)
    check_attn(gpu, b, heads, cache=cache, batch=batch)
    if heads // kvh <= 16:
        assert min(batch.ws.values()) > 0
    check_attn(gpu, b, heads, window=700)


@pytest.mark.parametrize("nq, kv", [([8, 3], [3, 9]), ([90, 70], [60, 200]), ([300, 1], [33, 40])])
def test_attn_widest_window(gpu, nq, kv):
    """The largest windows mask nothing, also where rows lie before position 0."""
    b = Batch(34, nq, kv, 2, 64, 16, "bf16")
    cache, batch = make(gpu, b, 4)
    q = torch.randn(b.ntok, 4, 64, device="cuda").bfloat16()
    want = cache.attend(batch, q)[0]
    for w in (max(kv), 2 ** 31 - 40, 2 ** 31 - 1):
        assert torch.equal(cache.attend(batch, q, window=w)[0], want)
    check_attn(gpu, b, 4, window=2 ** 31 - 1)


@pytest.mark.parametrize("part", [(1, 3), (2, 4), (0, 2)])
def test_part_of_a_batch(gpu, part):
    """Some of a batch's sequences, named by their entries of qstart: the rows
    before and behind them are left as they are."""
    b = Batch(35, [70, 1, 3, 90], [100, 2500, 300, 1800], 2, 64, 16, "bf16")
    cache, whole = make(gpu, b, 4)
    qs, kv, table = b.device()
    q = torch.randn(b.ntok, 4, 64, device="cuda").bfloat16()
    lo, hi = part
    for kw in (dict(), dict(max_q=90, max_kv=2500)):
        some = cache.batch(qs[lo:hi + 1], kv[lo:hi], table[lo:hi], b.ntok, **kw)
        out = torch.full((b.ntok, 256), 5.0, dtype=torch.bfloat16, device="cuda")
        z = cache.attend(some, q, out=out, lse=True)[1]
        r0, r1 = int(b.qs[lo]), int(b.qs[hi])
        assert (out[:r0] == 5).all() and (out[r1:] == 5).all()
        sub = Batch(35, b.nq[lo:hi], b.kv[lo:hi], 2, 64, 16, "bf16")
        sub.k, sub.v, sub.table, sub.pages = b.k, b.v, b.table[lo:hi], b.pages
        want, wl, mag, dots = ref.attend(sub, q[r0:r1].cpu(), 4)
        bound = ref.attn_bound(sub, torch.bfloat16, want, mag, dots)
        assert ((out[r0:r1].cpu().double().view_as(want) - want).abs() <= bound).all()
        assert torch.isfinite(z[r0:r1]).all()
    x = torch.randn(b.ntok, 512, device="cuda")
    before = cache.k.clone()
    qo = torch.full((b.ntok, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    cache.append(some, x, out=qo)
    assert (qo[:r0] == 5).all() and (qo[r1:] == 5).all()
    assert int((cache.k != before).any(-1).any(1).sum()) == sum(b.nq[lo:hi])
    some.check()


def test_append_bad_page(gpu):
    """Nothing of the row goes into either pool; its query is written."""
    from vgx import lib as vl
    b = Batch(36, [2, 1], [20, 40], 2, 64, 16, "q8")
    cache, _ = make(gpu, b, 4)
    qs, kv, table = b.device()
    table[1, 2] = b.pages
    batch = cache.batch(qs, kv, table, 3)
    qo = torch.full((3, 4, 64), 5.0, dtype=torch.float16, device="cuda")
    before = cache.k.clone(), cache.v.clone()
    cache.append(batch, torch.randn(3, 512, device="cuda"), out=qo)
    with pytest.raises(vl.VgxError, match="page"):
        batch.check()
    assert not (qo == 5).all(-1).any()
    assert torch.equal((cache.v != before[1]).any(-1), (cache.k != before[0]).any(-1))
    changed = (cache.k != before[0]).any(-1).any(1).nonzero()
    assert {int(p) for p in changed[:, 0]} == {int(b.table[0, 1])}


@pytest.mark.parametrize("kind, hd, page, window", [("bf16", 64, 16, 0), ("q8", 80, 5, 0), ("f16", 64, 16, 19000),
                                                    ("f16", 128, 32, 0)])
def test_attn_bounds_far_above(gpu, kind, hd, page, window):
    """Bounds far above most lengths: few, longer splits, also of the one
    sequence that reaches them."""
    kv = [int(m) for m in torch.randint(0, 300, (40,), generator=torch.Generator().manual_seed(2))]
    kv[3], kv[17], kv[39] = 24000, 1900, 17001
    b = Batch(37, [1] * 39 + [3], kv, 8, hd, page, kind)
    cache, batch = make(gpu, b, 8, max_q=4, max_kv=24000)
    check_attn(gpu, b, 8, window=window, cache=cache, batch=batch)
    # (the table's own size as the bound, and more rows than sequences have)
    b.table = torch.cat([b.table, torch.full((40, 60000 // page), -1, dtype=torch.int32)], 1)
    check_attn(gpu, b, 8, window=window, cache=cache, batch=cache.batch(*b.device(), b.ntok, 5))


def test_two_streams_at_once(gpu):
    """Calls in flight together, each with a workspace of its own."""
    b = Batch(38, [1, 3, 1, 200], [9000, 700, 20000, 5000], 2, 64, 16, "bf16")
    cache, batch = make(gpu, b, 8, max_q=200)
    qs = [torch.randn(b.ntok, 8, 64, device="cuda").bfloat16() for _ in range(2)]
    want = [cache.attend(batch, q, lse=True) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(cache.attend(batch, qs[i], lse=True))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(o, w[0]) and torch.equal(z, w[1]) for o, z in g)


def test_two_graphs(gpu):
    """Two captured steps replayed in turn and together, eager work between."""
    b = Batch(39, [1, 2, 1], [6000, 40, 1500], 2, 64, 16, "q8")
    cache, batch = make(gpu, b, 8, max_q=2)
    qs = [torch.randn(b.ntok, 8, 64, device="cuda").half() for _ in range(2)]
    want = [cache.attend(batch, q)[0] for q in qs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(cache.attend(batch, q)[0])
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in qs]
    for i in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(cache.attend(batch, qs[0])[0], want[0])
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), i


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("nq, kv", [([1, 2], [800, 130]), ([1], [9000]), ([90, 40], [800, 130]), ([100, 1], [100, 3000])])
@pytest.mark.parametrize("size", [1500, 6000, 20000])
def test_attn_scores_far_from_zero(gpu, kind, nq, kv, size):
    """Scores of up to 2^31 and their differences: where the two largest of a
    row are further apart than their 32-bit sums can be off, it is the largest
    one's value that comes out."""
    b = Batch(43, nq, kv, 2, 64, 16, kind)
    b.k = (size * b.k.float()).clamp(-60000, 60000).to(b.k.dtype)
    q = (size * b.randn(b.ntok, 4, 64)).clamp(-60000, 60000).to(ref.CTYPE[kind])
    cache, batch = make(gpu, b, 4)
    o, lse = cache.attend(batch, q.cuda(), lse=True)
    o, lse = o.cpu().double().view(b.ntok, 4, 64), lse.cpu().double()
    assert torch.isfinite(o).all() and torch.isfinite(lse).all()
    clear = 0
    for s, (n, m) in enumerate(zip(b.nq, b.kv)):
        for r in range(n):
            t = int(b.qs[s]) + r
            for h in range(4):
                k, v = (ref.value(b.rows(s, x, h // 2, m - n + r + 1)) for x in (b.k, b.v))
                x = k @ q[t, h].double() / 8
                # 64 additions of 32 bits each side, and 40 more: e^-40 of the values
                off = 2 * 64 * 2.0 ** -24 * float((k.abs() @ q[t, h].double().abs()).max()) / 8 + 40
                top = x.topk(min(2, len(x))).values
                if len(x) > 1 and top[0] - top[1] < off:
                    continue
                clear += 1
                want = v[int(x.argmax())]
                assert ((o[t, h] - want).abs() <= want.abs() * 2.0 ** -8).all()
                assert abs(lse[t, h] - top[0]) <= off
    assert clear >= b.ntok


def tail_batch(seed, nq, kv, hd, kind, kvh, score, sink):
    """One key a sequence whose score is `score`, all others' being 0, and its
    value 0: what comes out is the others' share.  The queries that go with it."""
    b = Batch(seed, nq, kv, kvh, hd, 16, kind)
    b.k.zero_()
    b.v = ref.to_cache(5 + 0.4 * b.randn(b.pages, kvh, 16, hd), kind)
    for s, m in enumerate(kv):
        p = {"first": 0, "middle": m // 2, "last": m - max(nq[s], 1)}[sink]
        pg, sl = int(b.table[s, p // 16]), p % 16
        b.k[pg, :, sl, 0] = 64 if kind == "q8" else 4  # 4 on the grid of 1/16
        b.v[pg, :, sl] = 0
    q = torch.randn(b.ntok, 2 * kvh, hd, generator=b.rng)
    q[..., 0] = score / 4 * hd ** 0.5
    return b, q.to(ref.CTYPE[kind])


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("score", [10.0, 14.0, 17.5, 20.0])
@pytest.mark.parametrize("sink", ["first", "middle", "last"])
@pytest.mark.parametrize("nq, kv, hd", [([1], [5000], 64), ([3, 1], [5000, 700], 128), ([7, 1], [2000, 900], 144),
                                        ([150], [3000], 64), ([140, 1], [1500, 4000], 64), ([70], [1200], 256)])
def test_attn_many_small_weights(gpu, kind, score, sink, nq, kv, hd):
    """Thousands of equal weights far below the largest add up.  A weight is at
    least 2^9 of f16's units of the largest (so it is off by at most half a step
    of itself or 2^-25 of those), the denominator at least the largest weight."""
    b, q = tail_batch(42, nq, kv, hd, kind, 1, score, sink)
    want, wl, mag, dots = ref.attend(b, q, 2)
    n, half = max(kv), ref.HALF_STEP[torch.float16]
    e_s = dots[..., None] * (hd + 8) * 2.0 ** -22 + 2.0 ** -21
    bound = half * mag + (2 * e_s + 2 * n * 2.0 ** -24) * mag + n * 2.0 ** -34 * float(ref.value(b.v).abs().max())
    bound = bound + half * (want.abs() + bound) + 2.0 ** -25
    cache, batch = make(gpu, b, 2)
    o, lse = cache.attend(batch, q.cuda(), lse=True)
    got = o.cpu().double().view_as(want)
    assert ((got - want).abs() <= bound).all()
    tol = dots * (hd + 8) * 2.0 ** -22 + (n + 32) * 2.0 ** -24 + wl.abs() * 2.0 ** -22
    assert ((lse.cpu().double() - wl).abs() <= tol).all()


def test_check_waits_for_every_stream(gpu):
    """A fault on a busy side stream is seen by a check() from the default one,
    and one raised right after it by the next."""
    from vgx import lib as vl
    b = Batch(44, [1, 1], [20, 40], 2, 64, 16, "bf16")
    cache, _ = make(gpu, b, 4)
    qs, kv, table = b.device()
    kv[1] = 10 ** 6
    batch = cache.batch(qs, kv, table, 2)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            cache.attend(batch, q)
        with pytest.raises(vl.VgxError, match="length"):
            batch.check()
    batch.check()


def test_more_splits_than_a_number_holds(gpu):
    """A batch whose splits would pass 2^31 partial results needs no workspace:
    its sequences stay whole."""
    import ctypes
    from vgx import lib as vl
    at = 1 << 20  # (nothing is read)
    c = vl.Paged(256, 8, 16, 16, 1 << 20, vl.E_BF16, 0.0, 0.0, at, at, 2048, 256, 16, 2048, 256, 16)
    for nseq, split in ((1 << 16, True), (1 << 20, False)):
        b = vl.Ragged(nseq, nseq, 1, 1 << 20, at, at, at, 1 << 16, 1 << 16, 0)
        need = vl.load().vgx_paged_attn_ws(gpu.ctx, ctypes.byref(c), ctypes.byref(b), 0)
        assert (need > 0) == split and need < 1 << 39


def guarded(n, dtype, fill):
    """n values of device memory between two runs of 4096 bytes of a pattern;
    the whole as bytes, and the n."""
    size = torch.tensor([], dtype=dtype).element_size()
    raw = torch.full((8192 + (n * size + 15) // 16 * 16,), 0xA5, dtype=torch.uint8, device="cuda")
    mid = raw[4096:4096 + n * size]
    mid.fill_(fill)
    return raw, mid.view(dtype)


@pytest.mark.parametrize("kind", ["bf16", "q8"])
@pytest.mark.parametrize("nq, kv, max_q, max_kv", [
    ([3, 40], [20, 90], 4, 0), ([40, 3], [90, 20], 0, 64),          # whole, more rows or positions than promised
    ([2, 9], [5000, 7000], 3, 0), ([2, 2], [3000, 9000], 2, 4096),  # split
    ([1, 90], [6000, 5000], 60, 0), ([100, 1], [7000, 300], 100, 2000),  # prompts beside single tokens
])
def test_bounds_are_held_in_every_buffer(gpu, kind, nq, kv, max_q, max_kv):
    """Beside a sequence past its bounds the other one's rows are right, and
    nothing is written around out, lse and the workspace, whose partial
    results hold 0xff where no workgroup writes them."""
    import ctypes
    from vgx import lib as vl
    hd, heads = 64, 4
    b = Batch(45, nq, kv, 2, hd, 16, kind)
    cache, _ = make(gpu, b, heads)
    batch = cache.batch(*b.device(), b.ntok, max_q=max_q, max_kv=max_kv)
    q = (2 * b.randn(b.ntok, heads, hd)).to(ref.CTYPE[kind])
    L = vl.load()
    need = int(L.vgx_paged_attn_ws(gpu.ctx, cache.ref, batch.ref, 0))
    ws_raw, ws = guarded(max(need, 16), torch.uint8, 0xFF)
    out_raw, out = guarded(b.ntok * heads * hd, cache.qtype, 0xFF)
    lse_raw, lse = guarded(b.ntok * heads, torch.float32, 0xFF)
    qd = q.cuda()
    r = vl.PagedQuery(qd.data_ptr(), heads * hd, 0.0, 0, cache.ckind, out.data_ptr(), heads * hd, lse.data_ptr(),
                      ws.data_ptr() if need else 0, need)
    vl.check(L.vgx_paged_attn(gpu.ctx, cache.ref, batch.ref, ctypes.byref(r)))
    with pytest.raises(vl.VgxError, match="length"):
        batch.check()
    for raw, t in ((ws_raw, ws), (out_raw, out), (lse_raw, lse)):
        n = t.numel() * t.element_size()
        assert (raw[:4096] == 0xA5).all() and (raw[4096 + n:] == 0xA5).all()
    want, wl, mag, dots = ref.attend(b, q, heads)
    bound = ref.attn_bound(b, ref.CTYPE[kind], want, mag, dots)
    got = ref.value(out.cpu()).view_as(want)
    kept = [s for s in range(2) if (not max_q or nq[s] <= max_q) and (not max_kv or kv[s] <= max_kv)]
    assert len(kept) == 1
    rows = slice(int(b.qs[kept[0]]), int(b.qs[kept[0] + 1]))
    assert ((got[rows] - want[rows]).abs() <= bound[rows]).all()
    assert torch.isfinite(lse.view(b.ntok, heads)[rows]).all()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_a_step_on_a_side_stream(gpu, kind):
    """The projections, append, attention and the next projection on a side
    stream behind other work of it: use_torch_stream() puts the calls of the
    context there too, and back."""
    from vgx import mmcf
    rng = np.random.default_rng(11)
    heads, kvh, hd, dim = 4, 2, 64, 256

    def mat(r, c):
        w, unit, plane = mmcf.q8_per_row(rng.standard_normal((r, c)).astype(np.float32) * 0.05)
        return gpu.upload(mmcf.Matrix("q8", r, c, (w.view(np.uint8) ^ 0x80).ravel(), unit, True, plane))

    wqkv, wo = mat((heads + 2 * kvh) * hd, dim), mat(dim, heads * hd)
    b = Batch(46, [9, 1, 30], [70, 500, 30], kvh, hd, 16, kind)
    cos, sin = (t.cuda() for t in tables(500, hd))
    given = (torch.randn(b.ntok, dim, generator=b.rng) * 256).to(torch.int16).cuda()

    def step(x):
        cache, batch = make(gpu, b, heads)
        q = cache.append(batch, gpu.gemm(wqkv, x), cos, sin)
        att = cache.attend(batch, q, out=torch.empty(b.ntok, heads * hd, dtype=torch.int16, device="cuda"))[0]
        return gpu.gemm(wo, att, x), batch

    want = step(given)[0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            gpu.use_torch_stream()
            x = torch.zeros_like(given)
            torch.cuda._sleep(20_000_000)
            x.copy_(given)
            got, batch = step(x)
        gpu.use_torch_stream()
        batch.check()
        assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["f16", "q8"])
@pytest.mark.parametrize("page", [5, 16, 64])
@pytest.mark.parametrize("nq, window", [([1, 3, 2], 100), ([1], 600), ([90, 40, 1], 100), ([130, 70], 33), ([7, 9], 1)])
def test_pages_behind_the_window_are_gone(gpu, kind, page, nq, window):
    """Entries of pages that no row sees any more are anything; one of a page
    that the first row still sees is a fault."""
    from vgx import lib as vl
    kv = [n + m for n, m in zip(nq, [700, 333, 1100])]
    b = Batch(47, nq, kv, 2, 64, page, kind)
    full = b.table.clone()
    cache, batch = make(gpu, b, 8)
    q = (2 * b.randn(b.ntok, 8, 64)).to(ref.CTYPE[kind])
    want = cache.attend(batch, q.cuda(), window=window)[0]
    batch.check()
    first = [(m - n - window + 1) // page for n, m in zip(nq, kv)]  # the page of the first key seen
    for gone in (-1, b.pages, 2 ** 31 - 1):
        for s, f in enumerate(first):
            b.table[s, :f] = gone
        cache, batch = make(gpu, b, 8)
        assert torch.equal(cache.attend(batch, q.cuda(), window=window)[0], want)
        batch.check()
    for s, f in enumerate(first):
        b.table.copy_(full)
        b.table[s, f] = -1
        cache, batch = make(gpu, b, 8)
        cache.attend(batch, q.cuda(), window=window)
        with pytest.raises(vl.VgxError, match="page"):
            batch.check()


def test_infinite_values_and_pages_behind_the_window(gpu):
    """The pass that adds them to the rows that see them, over tiles that begin
    before the window."""
    for nq in ([2, 1], [90, 60]):
        b = Batch(48, nq, [n + 500 for n in nq], 2, 64, 16, "bf16")
        for s in range(2):
            pos = 500 - 40
            b.v[int(b.table[s, pos // 16]), :, pos % 16, 7] = math.inf
        cache, batch = make(gpu, b, 4)
        q = torch.randn(b.ntok, 4, 64).bfloat16()
        want = cache.attend(batch, q.cuda(), window=100)[0]
        b.table[:, :(500 - 99) // 16] = -1
        cache, batch = make(gpu, b, 4)
        got = cache.attend(batch, q.cuda(), window=100)[0]
        batch.check()
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and torch.isinf(got).any()


@pytest.mark.parametrize("k_step, v_step", [(0.03, 0.5), (1.0, 1.0 / 128), (2.0 ** -10, 3.0)])
@pytest.mark.parametrize("nq, kv", [([1, 2], [700, 41]), ([1], [6000]), ([90, 70], [300, 70]), ([80, 1], [90, 3000])])
def test_q8_steps_and_scales(gpu, k_step, v_step, nq, kv):
    """Grids of K and V of their own, and a scale: append and attention."""
    heads, kvh, hd = 4, 2, 64
    b = Batch(49, nq, kv, kvh, hd, 16, "q8")
    k, v = b.k.cuda(), b.v.cuda()
    cache = gpu.paged_cache(heads, kvh, hd, "q8", k, v, k_step=k_step, v_step=v_step)
    batch = cache.batch(*b.device(), b.ntok)
    x = b.randn(b.ntok, (heads + 2 * kvh) * hd)
    x[:, heads * hd:] *= torch.cat([torch.full((kvh * hd,), 40 * k_step), torch.full((kvh * hd,), 40 * v_step)])
    q = cache.append(batch, x.cuda())
    for t, new, step in ((k, x[:, heads * hd:(heads + kvh) * hd], k_step), (v, x[:, (heads + kvh) * hd:], v_step)):
        new = new.view(b.ntok, kvh, hd).double()
        for s, (n, m) in enumerate(zip(nq, kv)):
            for r in range(n):
                pos, row = m - n + r, int(b.qs[s]) + r
                got = t[int(b.table[s, pos // 16]), :, pos % 16].cpu().double() * step
                want = new[row].clamp(-128 * step, 127 * step)
                # half a step, and the 32-bit quotient's and sum's rounding of 128 steps
                assert ((got - want).abs() <= step * (0.5 + 256 * 2.0 ** -24)).all()
    b.k, b.v = k.cpu(), v.cpu()
    for scale in (0.0, 0.02 / k_step / hd ** 0.5):
        o, lse = cache.attend(batch, q, scale=scale, lse=True)
        batch.check()
        want, wl, mag, dots = ref.attend(b, q.cpu(), heads, scale or None, 0, k_step, v_step)
        # (the bound's floor for small weights is in V's own grid)
        bound = ref.attn_bound(b, torch.float16, want, mag, dots) + max(kv) * 2.0 ** -25 * 128 * v_step
        assert ((o.cpu().double().view_as(want) - want).abs() <= bound).all()
        tol = dots * (hd + 8) * 2.0 ** -22 + (max(kv) + 32) * 2.0 ** -24 + wl.abs() * 2.0 ** -22
        assert ((lse.cpu().double() - wl).abs() <= tol).all()


@pytest.mark.parametrize("kind, hd", [("bf16", 64), ("q8", 96), ("f16", 112)])
def test_attn_many_sequences_of_chunks(gpu, kind, hd):
    """More sequences than a wave has lanes, of none to 60 rows: tiles are
    counted over all of them; and the same beside single tokens' kernel."""
    rng = np.random.default_rng(6)
    nq = rng.integers(0, 61, 150)
    nq[rng.random(150) < 0.3] = 1
    kv = [int(n) + int(m) for n, m in zip(nq, rng.integers(0, 120, 150))]
    b = Batch(50, nq.tolist(), kv, 1, hd, 16, kind)
    cache, batch = make(gpu, b, 2)
    check_attn(gpu, b, 2, cache=cache, batch=batch)
    check_attn(gpu, b, 2, window=50)


@pytest.mark.parametrize("heads, kvh", [(300, 1), (258, 2), (1024, 4)])
@pytest.mark.parametrize("nq", [[1, 1], [2, 5]])
def test_many_heads(gpu, heads, kvh, nq):
    """More heads a KV head than a tile has columns."""
    b = Batch(51, nq, [40, 200], kvh, 16, 16, "bf16")
    _, cache, batch = check_append(gpu, b, heads, torch.bfloat16, 16, True, True)
    b.k, b.v = cache.k.cpu(), cache.v.cpu()
    check_attn(gpu, b, heads, cache=cache, batch=batch)


@pytest.mark.parametrize("hd", range(16, 257, 16))
@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_every_head_size(gpu, kind, hd):
    for nq, kv in (([1, 3], [50, 33]), ([70, 1], [90, 300])):
        b = Batch(52, nq, kv, 2, hd, 16, kind)
        _, cache, batch = check_append(gpu, b, 6, torch.float16, hd, False, True)
        b.k, b.v = cache.k.cpu(), cache.v.cpu()
        check_attn(gpu, b, 6, cache=cache, batch=batch)
