"""What the paged cache's entry points refuse, each with every other argument
valid (the checks run before the device is touched: no GPU needed)."""
import ctypes

import pytest
import torch

from vgx import lib as vl

BUF = 1 << 20  # stands for a 16-byte aligned device address: nothing here reads it


def cache(**kw):
    d = dict(heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=10, kind=vl.E_BF16, k_step=0.0, v_step=0.0,
             k=BUF, v=BUF, k_page=2048, k_head=1024, k_row=64, v_page=2048, v_head=1024, v_row=64)
    d.update(kw)
    return vl.Paged(**d)


def batch(**kw):
    d = dict(nseq=3, ntok=7, max_q=0, max_kv=0, qstart=BUF, kvlen=BUF, table=BUF, table_cols=4, table_stride=4, fault=0)
    d.update(kw)
    return vl.Ragged(**d)


def rows(**kw):
    d = dict(kind=vl.E_Q16, qkv=BUF, stride=768, cos=BUF, sin=BUF, npos=64, rot=64, rope_half=1, q_norm=BUF, k_norm=BUF,
             eps=1e-5, q=BUF, q_stride=512)
    d.update(kw)
    return vl.PagedRows(**d)


def query(**kw):
    d = dict(q=BUF, q_stride=512, scale=0.0, window=0, out_kind=vl.E_BF16, out=BUF, out_stride=512, lse=0, ws=0,
             ws_bytes=0)
    d.update(kw)
    return vl.PagedQuery(**d)


def said(call, *args):
    st = call(None, *[ctypes.byref(a) if a is not None else None for a in args])
    return st, vl.load().vgx_last_error().decode()


def append(c=None, b=None, r=None):
    return said(vl.load().vgx_paged_append, c or cache(), b or batch(), r or rows())


def attn(c=None, b=None, r=None):
    return said(vl.load().vgx_paged_attn, c or cache(), b or batch(), r or query())


def test_valid_arguments_reach_the_context_check():
    for call in (append, attn):
        st, msg = call()
        assert st == vl.VGX_EINVAL and msg.endswith("no context")


@pytest.mark.parametrize("bad, what", [
    (dict(kind=vl.E_F32), "bf16, f16 or q8"), (dict(kind=vl.E_Q16), "bf16, f16 or q8"),
    (dict(heads=7), "multiple of kv_heads"), (dict(heads=0), "multiple of kv_heads"),
    (dict(kv_heads=-2), "multiple of kv_heads"), (dict(heads=1026), "at most 1024"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=40), "head_dim"), (dict(head_dim=272), "head_dim"),
    (dict(page_size=0), "page_size"), (dict(page_size=(1 << 20) + 1), "page_size"), (dict(num_pages=0), "no pages"),
    (dict(k=0), "NULL pages"), (dict(v=0), "NULL pages"), (dict(v=BUF + 8), "16-byte aligned"),
    (dict(k_row=68), "multiple of 16 bytes"), (dict(v_head=-1024), "negative"),
    (dict(k_row=56), "overlap"), (dict(k_page=1024), "overlap"), (dict(v_head=512), "overlap"),
    (dict(v_page=0), "overlap"), (dict(k_step=float("nan")), "step"), (dict(v_step=-1.0), "step"),
    (dict(k_step=float("inf")), "step"),
])
def test_cache(bad, what):
    for call in (append, attn):
        st, msg = call(c=cache(**bad))
        assert st == vl.VGX_EINVAL and what in msg, msg


@pytest.mark.parametrize("ok", [
    dict(k_page=2048, k_head=64, k_row=128),              # position-major
    dict(num_pages=1, k_page=0), dict(kv_heads=1, v_head=8),
    dict(page_size=1, k_row=0, v_row=0, k_head=64, v_head=64, k_page=128, v_page=128),
    dict(k_page=1 << 30, v_page=1 << 30),
])
def test_cache_layouts_that_are_fine(ok):
    st, msg = append(c=cache(**ok))
    if "kv_heads" in ok:
        assert msg.endswith("no context"), msg
    else:
        assert msg.endswith("no context"), msg


@pytest.mark.parametrize("bad, what, status", [
    (dict(nseq=-1), "nseq", vl.VGX_EINVAL), (dict(ntok=-1), "ntok", vl.VGX_EINVAL),
    (dict(ntok=(1 << 24) + 1), "ntok", vl.VGX_EINVAL), (dict(max_q=-1), "bound", vl.VGX_EINVAL),
    (dict(max_kv=-5), "bound", vl.VGX_EINVAL), (dict(qstart=0), "NULL", vl.VGX_EINVAL),
    (dict(kvlen=0), "NULL", vl.VGX_EINVAL), (dict(table=0), "NULL", vl.VGX_EINVAL),
    (dict(table_cols=0), "columns", vl.VGX_EINVAL), (dict(table_stride=3), "overlap", vl.VGX_EINVAL),
    (dict(table_cols=1 << 28, table_stride=1 << 28), "2^31", vl.VGX_ERANGE),
    (dict(max_kv=65), "max_kv", vl.VGX_ERANGE),
])
def test_batch(bad, what, status):
    for call in (append, attn):
        st, msg = call(b=batch(**bad))
        assert st == status and what in msg, msg


@pytest.mark.parametrize("bad, what", [
    (dict(kind=vl.E_Q8), "f32, bf16, f16 or q16"), (dict(kind=0), "f32, bf16, f16 or q16"),
    (dict(stride=767), "stride"), (dict(stride=760), "stride"), (dict(stride=772), "stride"),
    (dict(rot=24), "rot"), (dict(rot=80), "rot"), (dict(rot=-16), "rot"),
    (dict(cos=0), "table"), (dict(sin=0), "table"), (dict(npos=0), "table"),
    (dict(q_norm=0), "one norm"), (dict(k_norm=0), "one norm"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(q_stride=504), "q_stride"), (dict(q_stride=516), "q_stride"),
    (dict(qkv=0), "NULL qkv"), (dict(qkv=BUF + 2), "aligned"), (dict(q=BUF + 4), "aligned"),
])
def test_append_rows(bad, what):
    st, msg = append(r=rows(**bad))
    assert st == vl.VGX_EINVAL and what in msg, msg


@pytest.mark.parametrize("bad, what", [
    (dict(q_stride=504), "stride"), (dict(out_stride=514), "stride"), (dict(scale=-0.5), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(window=-1), "window"),
    (dict(out_kind=vl.E_F16), "compute type"), (dict(out_kind=vl.E_F32), "compute type"),
    (dict(q=0), "NULL"), (dict(out=0), "NULL"), (dict(q=BUF + 2), "aligned"), (dict(ws=BUF + 4), "aligned"),
])
def test_attn_query(bad, what):
    st, msg = attn(r=query(**bad))
    assert st == vl.VGX_EINVAL and what in msg, msg


def test_null_descriptions():
    L = vl.load()
    for call in (L.vgx_paged_append, L.vgx_paged_attn):
        assert said(call, None, batch(), rows())[0] == vl.VGX_EINVAL
        assert said(call, cache(), None, rows())[0] == vl.VGX_EINVAL
        assert said(call, cache(), batch(), None)[0] == vl.VGX_EINVAL
    assert L.vgx_paged_attn_ws(None, ctypes.byref(cache()), ctypes.byref(batch()), 0) == 0


class _Cpu:
    """What the binding's own checks need of a GPU (no device is touched before them)."""
    device = torch.device("cpu")

    def __init__(self):
        from vgx import gpu as vg
        self.need = lambda *a: vg.GPU.need(self, *a)
        self.need_rows = lambda *a: vg.GPU.need_rows(self, *a)


def _binding(ntok=3, table=None, nseq=2):
    from vgx import gpu as vg
    g = _Cpu()
    k = torch.zeros(6, 2, 16, 32, dtype=torch.bfloat16)
    cache = vg.PagedCache(g, 4, 2, 32, "bf16", k, k.clone())
    i32 = torch.int32
    return cache, cache.batch(torch.arange(nseq + 1, dtype=i32), torch.ones(nseq, dtype=i32),
                              torch.zeros(nseq, 3, dtype=i32) if table is None else table, ntok)


def test_binding_refuses_rows_that_overlap():
    """An expanded tensor holds one row: as many as its shape says would be
    read past its end."""
    cache, batch = _binding()
    row = torch.zeros(1, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        cache.append(batch, row.expand(3, -1))
    with pytest.raises(ValueError, match="rows apart"):
        cache.attend(batch, torch.zeros(1, 4, 32, dtype=torch.bfloat16).expand(3, -1, -1))
    with pytest.raises(ValueError, match="overlap"):
        cache.attend(batch, torch.zeros(1, 128, dtype=torch.bfloat16).expand(3, -1))
    with pytest.raises(ValueError, match="overlap"):
        _binding(table=torch.zeros(1, 3, dtype=torch.int32).expand(2, -1))
    with pytest.raises(ValueError, match="overlap"):
        cache.append(batch, torch.zeros(3 * 256, dtype=torch.bfloat16).as_strided((3, 256), (128, 1)))


def test_binding_refuses_half_a_pair():
    cache, batch = _binding()
    x, t = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(8, 16)
    for kw in (dict(cos=t), dict(sin=t), dict(q_norm=torch.ones(32)), dict(k_norm=torch.ones(32))):
        with pytest.raises(ValueError, match="both"):
            cache.append(batch, x, **kw)
    with pytest.raises(ValueError, match="rot/2"):
        cache.append(batch, x, t[0], t[0])


@pytest.mark.parametrize("step", [2.0 ** -65, 1e-45, 2.0 ** 65, 3e38])
def test_steps_whose_reciprocal_or_range_is_not_finite(step):
    for which in ("k_step", "v_step"):
        st, msg = append(c=cache(kind=vl.E_Q8, **{which: step}))
        assert st == vl.VGX_EINVAL and "step" in msg, msg
        assert append(c=cache(kind=vl.E_Q8, **{which: 2.0 ** -64}))[1].endswith("no context")


def test_binding_refuses_a_batch_of_another_device():
    """Its arrays are read by the cache's device."""
    cache, batch = _binding()
    other = _Cpu()
    other.device = torch.device("cuda", 1)
    batch.gpu = other
    with pytest.raises(ValueError, match="cuda:1"):
        cache.append(batch, torch.zeros(3, 256, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="cuda:1"):
        cache.attend(batch, torch.zeros(3, 128, dtype=torch.bfloat16))


def test_binding_keeps_no_workspace_size_of_a_refused_call():
    """0 bytes, as a refused call has, would leave the next cache's long
    sequences whole."""
    cache, batch = _binding()

    def refuse(call, *args):
        raise vl.VgxError(vl.VGX_EINVAL, "refused")

    cache.gpu.on_current, cache.gpu.ctx = refuse, None
    with pytest.raises(vl.VgxError):
        cache.attend(batch, torch.zeros(3, 128, dtype=torch.bfloat16))
    assert not batch.ws
