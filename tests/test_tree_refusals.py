"""What the calls on drafted trees, pages and samples refuse (no GPU needed)."""
import ctypes

import pytest
import torch

from test_paged_refusals import BUF, _binding, _Cpu, batch, cache, query, rows
from vgx import lib as vl

L = vl.load()


def said(call, *args):
    st = call(None, *args)
    return st, vl.load().vgx_last_error().decode()


def ref(x):
    return None if x is None else ctypes.byref(x)


def masks(b=None, parent=BUF, window=0, words=1, depth=BUF, see=BUF):
    return said(L.vgx_tree_masks, ref(b or batch()), parent, window, words, depth, see)


def tree(**kw):
    return vl.Tree(**dict(dict(depth=BUF, see=BUF, words=1), **kw))


def attn(t="", b=None, q=None, c=None):
    return said(L.vgx_paged_attn_tree, ref(c or cache()), ref(b or batch()), ref(q or query()), ref(tree() if t == "" else t))


def accept(b=None, **kw):
    d = dict(parent=BUF, tokens=BUF, chosen=BUF, path=BUF, accepted=BUF, next=BUF)
    d.update(kw)
    return said(L.vgx_tree_accept, ref(b or batch()), *d.values())


def caches(*c):
    return (vl.Paged * len(c))(*c)


def keep(c=None, b=None, n=None, path=BUF, accepted=BUF):
    c = caches(cache()) if c is None else c
    return said(L.vgx_paged_keep, len(c) if n is None else n, c, ref(b or batch()), path, accepted)


def copy(c=None, n=3, ncache=None, src=BUF, dst=BUF, rows=0, fault=0):
    c = caches(cache()) if c is None else c
    return said(L.vgx_paged_copy, len(c) if ncache is None else ncache, c, n, src, dst, rows, fault)


def sample(**kw):
    d = dict(nrows=3, vocab=100, kind=vl.E_F32, logits=BUF, stride=100, u=BUF, temp=0, top_k=0, top_p=0, min_p=0,
             token=BUF, kept=0, prob=0, ws=BUF, ws_bytes=1 << 40)
    d.update(kw)
    return said(L.vgx_sample, ref(vl.Sampling(**d)))


def test_valid_arguments_reach_the_context_check():
    for st, msg in (masks(), attn(), accept(), keep(), copy(), sample(),
                    said(L.vgx_paged_append_tree, ref(cache()), ref(batch()), ref(rows()), BUF)):
        assert st == vl.VGX_EINVAL and msg.endswith("no context"), msg


def bad(got, what, status=vl.VGX_EINVAL):
    assert got[0] == status and what in got[1], got


def test_masks():
    bad(masks(parent=0), "NULL parent")
    bad(masks(depth=0), "NULL parent")
    bad(masks(see=0), "NULL parent")
    bad(masks(words=0), "1 to 16")
    bad(masks(words=17), "1 to 16")
    bad(masks(window=-1), "window")
    bad(masks(batch(ntok=65)), "max_q", vl.VGX_ERANGE)
    bad(masks(batch(ntok=500, max_q=65)), "max_q", vl.VGX_ERANGE)
    assert masks(batch(ntok=500, max_q=64))[1].endswith("no context")
    assert masks(batch(ntok=500), words=8)[1].endswith("no context")
    assert masks(batch(kvlen=0, table=0, table_cols=0))[1].endswith("no context")
    bad(masks(batch(qstart=0)), "qstart")
    bad(masks(batch(nseq=-1)), "nseq")
    bad(masks(batch(ntok=-1)), "ntok")
    bad(masks(batch(max_q=-1)), "bound")
    assert said(L.vgx_tree_masks, None, BUF, 0, 1, BUF, BUF)[0] == vl.VGX_EINVAL


def test_attn():
    bad(attn(None), "NULL tree")
    bad(attn(tree(words=0)), "1 to 16")
    bad(attn(tree(words=17)), "1 to 16")
    bad(attn(tree(see=0)), "masks")
    bad(attn(tree(depth=0), q=query(window=5)), "depths")
    assert attn(tree(depth=0))[1].endswith("no context")
    bad(attn(b=batch(ntok=100, nseq=3)), "max_q", vl.VGX_ERANGE)
    bad(attn(q=query(window=-1)), "window")
    bad(attn(c=cache(kind=vl.E_F32)), "bf16, f16 or q8")
    assert L.vgx_paged_attn_tree_ws(None, ref(cache()), ref(batch()), 0) == 0


def test_append():
    bad(said(L.vgx_paged_append_tree, ref(cache()), ref(batch()), ref(rows()), 0), "depths")


def test_accept():
    for k in ("parent", "tokens", "chosen", "path"):
        bad(accept(**{k: 0}), "NULL parent")
    for k in ("accepted", "next"):
        bad(accept(**{k: 0}), "NULL accepted")
    bad(accept(batch(ntok=1025)), "1024", vl.VGX_ERANGE)
    assert accept(batch(ntok=5000, max_q=1024))[1].endswith("no context")


def test_keep():
    bad(keep(n=0), "no caches")
    bad(keep(c=caches(cache(), cache(k_page=4096))), "differ")
    bad(keep(c=caches(cache(), cache(num_pages=11))), "differ")
    bad(keep(c=caches(cache(), cache(kind=vl.E_F16))), "differ")
    bad(keep(c=caches(cache(), cache(v=0))), "NULL pages")
    bad(keep(c=caches(cache(), cache(v=BUF + 8))), "aligned")
    assert keep(c=caches(cache(), cache(k=2 * BUF, heads=4)))[1].endswith("no context")
    bad(keep(path=0), "NULL path")
    bad(keep(accepted=0), "NULL path")
    bad(keep(b=batch(table=0)), "NULL qstart")


def test_copy():
    bad(copy(ncache=0), "no caches")
    bad(copy(n=-1), "pages outside")
    bad(copy(n=(1 << 20) + 1), "pages outside")
    bad(copy(src=0), "NULL src")
    bad(copy(dst=0), "NULL src")
    bad(copy(c=caches(cache(head_dim=40))), "head_dim")
    big = dict(page_size=1 << 20, k_head=64 << 20, v_head=64 << 20, k_page=128 << 20, v_page=128 << 20)
    assert copy(c=caches(cache(**big)))[1].endswith("no context")
    bad(copy(c=caches(cache(kv_heads=512, heads=512, page_size=1 << 20, k_head=64 << 20, v_head=64 << 20,
                            k_page=1 << 36, v_page=1 << 36))), "too large", vl.VGX_ERANGE)


@pytest.mark.parametrize("kw, what", [
    (dict(nrows=-1), "nrows"), (dict(nrows=65536), "nrows"), (dict(vocab=0), "vocab"),
    (dict(vocab=(1 << 21) + 1, stride=1 << 22), "vocab"), (dict(kind=vl.E_Q8), "f32, bf16"), (dict(kind=0), "f32, bf16"),
    (dict(logits=0), "NULL"), (dict(u=0), "NULL"), (dict(token=0), "NULL"), (dict(stride=99), "stride"),
    (dict(stride=1 << 41), "stride"), (dict(logits=BUF + 2), "aligned"),
    (dict(logits=BUF + 1, kind=vl.E_BF16), "aligned")])
def test_sample(kw, what):
    bad(sample(**kw), what)


def test_sample_workspace():
    kw = dict(vocab=20000, stride=20000)
    need = L.vgx_sample_ws(3, 20000, vl.E_F32)
    assert need > 0
    bad(sample(ws=0, **kw), "workspace")
    bad(sample(ws_bytes=need - 1, **kw), "workspace")
    bad(sample(ws=BUF + 8, **kw), "workspace")
    assert sample(ws_bytes=need, **kw)[1].endswith("no context")
    assert L.vgx_sample_ws(3, 100, vl.E_F32) == 0 and sample(ws=0, ws_bytes=0)[1].endswith("no context")
    assert L.vgx_sample_ws(3, 0, vl.E_F32) == 0 and L.vgx_sample_ws(-1, 10, vl.E_F32) == 0
    assert said(L.vgx_sample, None)[0] == vl.VGX_EINVAL


def test_binding_refuses():
    """What would be read or written past its end, or belongs elsewhere."""
    from vgx import gpu as vg
    c, b = _binding()
    i32 = torch.int32
    for name in ("need_values", "need", "need_rows"):
        setattr(c.gpu, name, lambda *a, f=getattr(vg.GPU, name): f(c.gpu, *a))
    p3, p2 = torch.zeros(3, dtype=i32), torch.zeros(2, dtype=i32)
    with pytest.raises(ValueError, match="parent"):
        b.tree(p2)
    with pytest.raises(ValueError, match="parent"):
        b.tree(p3.long())
    with pytest.raises(ValueError, match="tokens"):
        b.accept(p3, p2, p3)
    with pytest.raises(ValueError, match="chosen"):
        b.accept(p3, p3, torch.zeros(1, dtype=i32).expand(3))
    layers = vg.PagedLayers([c])
    with pytest.raises(ValueError, match="path"):
        layers.keep(b, p2, p2)
    with pytest.raises(ValueError, match="accepted"):
        layers.keep(b, p3, p3)
    with pytest.raises(ValueError, match="dst"):
        layers.copy(p3, p2)
    with pytest.raises(ValueError, match="rows"):
        layers.copy(p3, p3, p2)
    with pytest.raises(ValueError, match="no caches"):
        vg.PagedLayers([])
    other, ob = _binding()
    far = _Cpu()
    far.device = torch.device("cuda", 1)
    other.gpu = far
    with pytest.raises(ValueError, match="several devices"):
        vg.PagedLayers([c, other])
    with pytest.raises(ValueError, match="1024 rows"):
        _binding(ntok=1025)[1].tree(torch.zeros(1025, dtype=i32))
    made = object.__new__(vg.Tree)
    made.batch, made.window = ob, 0
    q = torch.zeros(3, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="another batch"):
        c.attend(b, q, tree=made)
    made.batch = b
    with pytest.raises(ValueError, match="window"):
        c.attend(b, q, window=4, tree=made)
