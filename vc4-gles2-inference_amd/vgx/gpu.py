"""Host-side mirror of the reference engine's GPU object over libvgx.

`GPU` has the reference's entry points (engine/src/gpu.h:41-633: upload,
matvec / matvec_add, ffn_split_chunked, rmsnorm, attention_block,
kv_rope_write, logits_from) with the same argument meaning; device buffers are
torch tensors on the GPU (plumbing only: every number is computed by libvgx).
"""
import ctypes

import numpy as np
import torch

from . import lib as _l
from .mmcf import Matrix


def _ptr(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


# the handle of torch's current stream on a device (an int)
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _at(t):
    return 0 if t is None else t.data_ptr()


def _np_ptr(a):
    return ctypes.c_void_p(0 if a is None else a.ctypes.data)


class Mat:
    """An uploaded weight matrix (GPU::upload's result)."""

    def __init__(self, gpu, handle, m):
        self.gpu, self.h, self.rows, self.cols, self.kind = gpu, handle, m.rows, m.cols, m.kind

    @property
    def weight_bytes(self):
        return int(_l.load().vgx_mat_weight_bytes(self.h))

    def free(self):
        if self.h:
            _l.load().vgx_mat_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Group:
    """Matrices sharing one input, launched as one kernel (logits tiles)."""

    def __init__(self, gpu, mats):
        L = _l.load()
        arr = (ctypes.c_void_p * len(mats))(*[m.h for m in mats])
        h = ctypes.c_void_p()
        _l.check(L.vgx_group_create(gpu.ctx, len(mats), arr, ctypes.byref(h)))
        self.gpu, self.h, self.mats = gpu, h, list(mats)
        self.rows = int(L.vgx_group_rows(h))

    def gemv(self, x, out=None):
        out = out if out is not None else torch.empty(self.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemv_group(self.gpu.ctx, self.h, _ptr(x), _ptr(out)))
        return out

    def plan(self):
        """(lanes per row, rows per lane) of this group's launch."""
        lpr, ri = ctypes.c_int(), ctypes.c_int()
        _l.check(_l.load().vgx_group_plan_info(self.h, ctypes.byref(lpr), ctypes.byref(ri)))
        return lpr.value, ri.value

    def gemv_f32(self, x, out=None):
        out = out if out is not None else torch.empty(self.rows, dtype=torch.float32, device=x.device)
        _l.check(_l.load().vgx_gemv_group_f32(self.gpu.ctx, self.h, _ptr(x), _ptr(out)))
        return out

    def logits_argmax(self, x, logits=None, token=None):
        logits = logits if logits is not None else torch.empty(self.rows, dtype=torch.int16, device=x.device)
        token = token if token is not None else torch.empty(1, dtype=torch.int32, device=x.device)
        _l.check(_l.load().vgx_logits_argmax(self.gpu.ctx, self.h, _ptr(x), _ptr(logits), _ptr(token)))
        return logits, token

    def gemv_rms(self, x, rms_w, eps, out=None):
        """rmsnorm(x, rms_w, eps) then the group GEMV, one launch."""
        out = out if out is not None else torch.empty(self.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemv_group_rms(self.gpu.ctx, self.h, _ptr(x), _ptr(rms_w), float(eps), _ptr(out)))
        return out

    def logits_argmax_rms(self, x, rms_w, eps, logits=None, token=None):
        """The final norm, the logits pass and the argmax in one launch."""
        logits = logits if logits is not None else torch.empty(self.rows, dtype=torch.int16, device=x.device)
        token = token if token is not None else torch.empty(1, dtype=torch.int32, device=x.device)
        _l.check(_l.load().vgx_logits_argmax_rms(self.gpu.ctx, self.h, _ptr(x), _ptr(rms_w), float(eps),
                                                  _ptr(logits), _ptr(token)))
        return logits, token

    def logits_argmax_step(self, x, rms_w, eps, logits, token, pos, hist, emb, emb_scale, x_next):
        """logits_argmax_rms, then in the reduction launch hist[pos + 1] =
        token, ++pos and the token's q8 embedding row into x_next."""
        vocab, dim = emb.shape
        _l.check(_l.load().vgx_logits_argmax_step(self.gpu.ctx, self.h, _ptr(x), _ptr(rms_w), float(eps),
                                                   _ptr(logits), _ptr(token), _ptr(pos), _ptr(hist),
                                                   int(hist.numel()), _ptr(emb), _ptr(emb_scale), vocab, dim,
                                                   _ptr(x_next)))
        return logits, token

    def free(self):
        if self.h:
            _l.load().vgx_group_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Conv:
    """LFM2 conv-block state and taps (GPU::init_conv / set_conv_kernel)."""

    def __init__(self, gpu, w, layer_is_conv=None):
        L = _l.load()
        self._w = np.ascontiguousarray(w, np.float32)  # [layers][dim][3]
        layers, dim, k = self._w.shape
        self._types = None if layer_is_conv is None else np.ascontiguousarray(layer_is_conv, np.uint8)
        h = ctypes.c_void_p()
        _l.check(L.vgx_conv_create(gpu.ctx, dim, layers, k, _np_ptr(self._w), _np_ptr(self._types),
                                   ctypes.byref(h)))
        self.gpu, self.h, self.dim = gpu, h, dim

    def step(self, layer, bcx, out=None):
        """bcx: (ntok, 3*dim) or (3*dim,) q16; returns y of the same leading shape."""
        n = 1 if bcx.dim() == 1 else bcx.shape[0]
        shape = (self.dim,) if bcx.dim() == 1 else (n, self.dim)
        out = out if out is not None else torch.empty(shape, dtype=torch.int16, device=bcx.device)
        _l.check(_l.load().vgx_conv_step(self.h, layer, n, _ptr(bcx), _ptr(out)))
        return out

    def reset(self):
        _l.check(_l.load().vgx_conv_reset(self.h))

    def state(self, layer):
        buf = np.empty((2, self.dim), np.int16)
        _l.check(_l.load().vgx_conv_state_read(self.h, layer, _np_ptr(buf)))
        return buf

    def set_state(self, layer, st):
        st = np.ascontiguousarray(st, np.int16)
        _l.check(_l.load().vgx_conv_state_write(self.h, layer, _np_ptr(st)))

    def free(self):
        if self.h:
            _l.load().vgx_conv_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Attention:
    """GPU::init_attention's state: KV cache, RoPE table, q/k norm weights."""

    def __init__(self, gpu, dim, heads, kv_heads, head_dim, seq, layers, kv_bits, rope_half, qk_norm,
                 rope_cos, rope_sin, q_norm=None, k_norm=None, layer_is_attn=None, nseq=1):
        L = _l.load()
        self._keep = [np.ascontiguousarray(rope_cos, np.float32), np.ascontiguousarray(rope_sin, np.float32),
                      None if q_norm is None else np.ascontiguousarray(q_norm, np.float32),
                      None if k_norm is None else np.ascontiguousarray(k_norm, np.float32),
                      None if layer_is_attn is None else np.ascontiguousarray(layer_is_attn, np.uint8)]
        d = _l.AttnDesc(dim, heads, kv_heads, head_dim, seq, layers, kv_bits, int(rope_half), int(qk_norm),
                        _np_ptr(self._keep[0]), _np_ptr(self._keep[1]), _np_ptr(self._keep[2]),
                        _np_ptr(self._keep[3]), _np_ptr(self._keep[4]))
        h = ctypes.c_void_p()
        _l.check(L.vgx_attn_create_seqs(gpu.ctx, ctypes.byref(d), nseq, ctypes.byref(h)))
        self.gpu, self.h, self.dim, self.seq, self.nseq = gpu, h, dim, seq, nseq
        self.row_bytes = int(L.vgx_kv_row_bytes(h))
        self.views = []

    def view(self, s):
        """Sequence s's cache as a single-sequence Attention (freed with the parent)."""
        h = ctypes.c_void_p()
        _l.check(_l.load().vgx_attn_seq_view(self.h, s, ctypes.byref(h)))
        v = Attention.__new__(Attention)
        v.gpu, v.h, v.dim, v.seq, v.nseq, v.row_bytes, v.views = self.gpu, h, self.dim, self.seq, 1, self.row_bytes, []
        self.views.append(v)
        return v

    def block_seqs(self, layer, pos, qkv, out=None):
        """Position pos of the sequences 0..n-1 for the n rows of qkv."""
        n = qkv.shape[0]
        out = out if out is not None else torch.empty((n, self.dim), dtype=torch.int16, device=qkv.device)
        _l.check(_l.load().vgx_attn_block_seqs(self.h, layer, pos, n, _ptr(qkv), _ptr(out)))
        return out

    def kv_append(self, layer, pos, qkv):
        _l.check(_l.load().vgx_kv_append(self.h, layer, pos, _ptr(qkv)))

    def decode(self, layer, pos, qkv, out=None):
        out = out if out is not None else torch.empty(self.dim, dtype=torch.int16, device=qkv.device)
        _l.check(_l.load().vgx_attn_decode(self.h, layer, pos, _ptr(qkv), _ptr(out)))
        return out

    def block(self, layer, pos, qkv, out=None):
        out = out if out is not None else torch.empty(self.dim, dtype=torch.int16, device=qkv.device)
        _l.check(_l.load().vgx_attn_block(self.h, layer, pos, _ptr(qkv), _ptr(out)))
        return out

    def block_batch(self, layer, pos0, qkv, out=None):
        """Positions pos0 .. pos0 + n - 1 for the n rows of qkv: the KV rows
        are appended first, then every position attends to its prefix."""
        n = qkv.shape[0]
        out = out if out is not None else torch.empty((n, self.dim), dtype=torch.int16, device=qkv.device)
        L = _l.load()
        _l.check(L.vgx_kv_append_batch(self.h, layer, pos0, n, _ptr(qkv)))
        _l.check(L.vgx_attn_decode_batch(self.h, layer, pos0, n, _ptr(qkv), _ptr(out)))
        return out

    def read_rows(self, layer, row0, nrows):
        buf = np.empty(nrows * self.row_bytes, np.uint8)
        _l.check(_l.load().vgx_kv_read_rows(self.h, layer, row0, nrows, _np_ptr(buf)))
        return buf

    def write_rows(self, layer, row0, data):
        data = np.ascontiguousarray(data, np.uint8)
        _l.check(_l.load().vgx_kv_write_rows(self.h, layer, row0, data.size // self.row_bytes, _np_ptr(data)))

    def free(self):
        for v in getattr(self, "views", []):
            v.free()
        if self.h:
            _l.load().vgx_attn_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


_ELEM = {torch.float32: _l.E_F32, torch.bfloat16: _l.E_BF16, torch.float16: _l.E_F16, torch.int16: _l.E_Q16}
_F32, _I32 = torch.float32, torch.int32
_CACHE = {"bf16": (_l.E_BF16, torch.bfloat16, torch.bfloat16), "f16": (_l.E_F16, torch.float16, torch.float16),
          "q8": (_l.E_Q8, torch.int8, torch.float16)}


def _raise_fault(gpu, fault, who, length):
    torch.cuda.synchronize(gpu.device)
    bits = int(fault.item())
    if bits:
        fault.zero_()
        torch.cuda.synchronize(gpu.device)  # (before another stream's next call can set one)
        what = [w for b, w in ((_l.FAULT_LENGTH, length), (_l.FAULT_PAGE, "a page outside the pool")) if bits & b]
        raise _l.VgxError(_l.VGX_ERANGE, who + ": " + " and ".join(what))


class RaggedBatch:
    """A ragged batch over a paged cache: sequence s has rows qstart[s] ..
    qstart[s+1]-1 of the ntok new ones, kvlen[s] positions counting them, and
    its pages in table[s].  The arrays are read when a call runs, so they may
    change between calls (and between replays of a captured one); max_q and
    max_kv bound one sequence's rows and positions.  check() waits for the
    device (all its streams, whichever the calls ran on) and raises if a call
    met a length or page outside its bounds."""

    def __init__(self, gpu, qstart, kvlen, table, ntok, max_q=0, max_kv=0):
        gpu.need(qstart, torch.int32, 1, "qstart")
        gpu.need(kvlen, torch.int32, 1, "kvlen")
        gpu.need(table, torch.int32, 2, "table")
        nseq = kvlen.shape[0]
        if qstart.shape[0] != nseq + 1 or table.shape[0] != nseq:
            raise ValueError("a batch of %d sequences needs qstart of %d and a table of %d rows"
                             % (nseq, nseq + 1, nseq))
        if ((nseq > 0 and qstart.stride(0) != 1) or (nseq > 1 and kvlen.stride(0) != 1)
                or (table.shape[1] > 1 and table.stride(1) != 1)):
            raise ValueError("qstart, kvlen and a table's rows must be contiguous")
        if nseq > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("a table's rows overlap (an expanded tensor: make it contiguous)")
        self.gpu, self.nseq, self.ntok = gpu, nseq, int(ntok)
        self.fault = torch.zeros(1, dtype=torch.int32, device=gpu.device)
        self._keep = (qstart, kvlen, table)
        self.d = _l.Ragged(nseq, self.ntok, int(max_q), int(max_kv), qstart.data_ptr(), kvlen.data_ptr(),
                           table.data_ptr(), table.shape[1], table.stride(0) if nseq > 1 else table.shape[1],
                           self.fault.data_ptr())
        self.ref = ctypes.byref(self.d)
        self.ws = {}  # workspace bytes by what of a cache and call decides them (PagedCache.attend)

    def tree(self, parent, window=0):
        """The rows as drafted trees: parent[r] is the number of row r's parent
        among its sequence's rows (-1: none)."""
        return Tree(self, parent, window)

    def accept(self, parent, tokens, chosen):
        """The walk down each sequence's tree by the token that each row's
        logits gave: (path: the rows of the way, at qstart[s] + k the k-th,
        -1 behind its end, undefined for rows of no sequence; accepted: rows of
        the way but the first; next: the last one's token)."""
        g = self.gpu
        for t, name in ((parent, "parent"), (tokens, "tokens"), (chosen, "chosen")):
            g.need_values(t, _I32, self.ntok, name)
        path, accepted = torch.empty_like(parent), torch.empty(self.nseq, dtype=_I32, device=g.device)
        nxt = torch.empty_like(accepted)
        g.on_current(_l.load().vgx_tree_accept, self.ref, parent.data_ptr(), tokens.data_ptr(), chosen.data_ptr(),
                     path.data_ptr(), accepted.data_ptr(), nxt.data_ptr())
        return path, accepted, nxt

    def check(self):
        _raise_fault(self.gpu, self.fault, "ragged batch", "a length outside its bounds")


class Tree:
    """A batch's rows as drafted trees: each row's depth and the mask of the
    rows it sees, itself and its ancestors (with a window those inside it), from
    its parent.  Made once for all layers; update() makes them anew from other
    parents, in place (a captured step's)."""

    def __init__(self, batch, parent, window=0):
        g = batch.gpu
        most = min(batch.d.max_q, batch.ntok) or batch.ntok
        self.batch, self.window = batch, int(window)
        self.words = max(1, -(-most // 64))
        if self.words > 16:
            raise ValueError("a tree has at most 1024 rows a sequence: give the batch its bound max_q")
        self.depth = torch.empty(batch.ntok, dtype=_I32, device=g.device)
        self.see = torch.empty((batch.ntok, self.words), dtype=torch.int64, device=g.device)
        self.d = _l.Tree(self.depth.data_ptr(), self.see.data_ptr(), self.words)
        self.ref = ctypes.byref(self.d)
        self.update(parent)

    def update(self, parent):
        g = self.batch.gpu
        g.need_values(parent, _I32, self.batch.ntok, "parent")
        g.on_current(_l.load().vgx_tree_masks, self.batch.ref, parent.data_ptr(), self.window, self.words,
                     self.depth.data_ptr(), self.see.data_ptr())


class PagedLayers:
    """The caches of a model's layers, alike in shape, type and strides, whose
    pages are numbered alike: what moves pages moves them in all of them at
    once."""

    def __init__(self, caches):
        if not caches:
            raise ValueError("no caches")
        self.gpu, self.caches = caches[0].gpu, list(caches)
        if any(c.gpu.device != self.gpu.device for c in caches):
            raise ValueError("the caches are on several devices")
        self.d = (_l.Paged * len(caches))(*[c.d for c in caches])
        self.fault = torch.zeros(1, dtype=_I32, device=self.gpu.device)

    def keep(self, batch, path, accepted):
        """The rows of an accepted path (RaggedBatch.accept) become their
        sequences' next positions: kvlen[s] - rows + 1 + accepted[s] are held
        then."""
        g = self.gpu
        self.caches[0]._same_device(batch)
        g.need_values(path, _I32, batch.ntok, "path")
        g.need_values(accepted, _I32, batch.nseq, "accepted")
        g.on_current(_l.load().vgx_paged_keep, len(self.d), self.d, batch.ref, path.data_ptr(), accepted.data_ptr())

    def copy(self, src, dst, rows=None):
        """Pages dst[i] = pages src[i], of each the first rows[i] positions."""
        g, n = self.gpu, src.shape[0]
        g.need_values(src, _I32, n, "src")
        g.need_values(dst, _I32, n, "dst")
        if rows is not None:
            g.need_values(rows, _I32, n, "rows")
        g.on_current(_l.load().vgx_paged_copy, len(self.d), self.d, n, src.data_ptr(), dst.data_ptr(), _at(rows),
                     self.fault.data_ptr())

    def check(self):
        """Waits for the device and raises if a copy met a page or a number of
        rows outside its bounds (keep's are the batch's)."""
        _raise_fault(self.gpu, self.fault, "paged copy", "a number of rows outside the page")


class PagedCache:
    """One layer's paged KV cache over the caller's tensors k and v, each
    (pages, kv_heads, page_size, head_dim) of any strides whose last is 1 (a
    position-major pool is passed as its transposed view).  kind "bf16",
    "f16" or "q8" (int8, the grids k_step and v_step, 1/16 by default); the
    queries and outputs are bfloat16 for "bf16" and float16 for the others.
    The calls run on torch's current stream (GPU's others on the one set
    last: see GPU)."""

    def __init__(self, gpu, heads, kv_heads, head_dim, kind, k, v, k_step=0.0, v_step=0.0):
        elem, ctype, self.qtype = _CACHE[kind]
        for t, name in ((k, "k"), (v, "v")):
            gpu.need(t, ctype, 4, name)
            if t.shape[1] != kv_heads or t.shape[3] != head_dim or t.stride(3) != 1 or t.shape != k.shape:
                raise ValueError("%s must be (pages, %d, page_size, %d), head vectors contiguous" % (name, kv_heads,
                                                                                                   head_dim))
        self.gpu, self.heads, self.kv_heads, self.head_dim, self.kind = gpu, heads, kv_heads, head_dim, kind
        self.ckind = _ELEM[self.qtype]
        self.k, self.v, self.width = k, v, heads * head_dim
        self.qkv_width, self.norm_shape = (heads + 2 * kv_heads) * head_dim, torch.Size((head_dim,))
        self.d = _l.Paged(heads, kv_heads, head_dim, k.shape[2], k.shape[0], elem, k_step, v_step, k.data_ptr(),
                          v.data_ptr(), *k.stride()[:3], *v.stride()[:3])
        self.ref = ctypes.byref(self.d)

    def batch(self, qstart, kvlen, table, ntok, max_q=0, max_kv=0):
        return RaggedBatch(self.gpu, qstart, kvlen, table, ntok, max_q, max_kv)

    def append(self, batch, qkv, cos=None, sin=None, rope_half=True, q_norm=None, k_norm=None, eps=1e-5, out=None,
               tree=None):
        """The rows qkv (ntok, (heads + 2 kv_heads) * head_dim; float32,
        bfloat16, float16 or q16) normed, rotated (cos, sin: positions x rot/2)
        and written into the cache; returns the queries (ntok, heads, head_dim).
        tree (RaggedBatch.tree): a row is rotated by its depth's position."""
        g = self.gpu
        self._same_device(batch)
        kind = _ELEM.get(qkv.dtype)
        if kind is None:
            raise ValueError("qkv must be float32, bfloat16, float16 or int16 (q16)")
        stride = g.need_rows(qkv, None, batch.ntok, self.qkv_width, "qkv")
        npos = rot = 0
        if (cos is None) != (sin is None) or (q_norm is None) != (k_norm is None):
            raise ValueError("cos and sin, and the norm weights, come both or not at all")
        if cos is not None:
            if cos.dim() != 2:
                raise ValueError("cos and sin must be positions x rot/2")
            npos, half = cos.shape
            rot = 2 * half
            for t in (cos, sin):
                if t.dtype is not _F32 or t.device != g.device or t.shape != cos.shape or not t.is_contiguous():
                    raise ValueError("cos and sin must be contiguous float32 tensors of one shape on %s" % g.device)
        for t in (q_norm, k_norm):
            if t is not None and (t.dtype is not _F32 or t.device != g.device or t.shape != self.norm_shape
                                  or not t.is_contiguous()):
                raise ValueError("a norm weight must be %d contiguous float32 values on %s" % (self.head_dim, g.device))
        if out is None:
            q, qs = torch.empty((batch.ntok, self.heads, self.head_dim), dtype=self.qtype, device=g.device), self.width
        else:
            q, qs = out, self._rows(out, self.qtype, batch.ntok, "out")
        r = _l.PagedRows(kind, qkv.data_ptr(), stride, _at(cos), _at(sin), npos, rot, int(rope_half), _at(q_norm),
                         _at(k_norm), eps, q.data_ptr(), qs)
        if tree is None:
            g.on_current(_l.load().vgx_paged_append, self.ref, batch.ref, ctypes.byref(r))
        else:
            self._same_batch(batch, tree)
            g.on_current(_l.load().vgx_paged_append_tree, self.ref, batch.ref, ctypes.byref(r), tree.d.depth)
        return q

    def attend(self, batch, q, scale=0.0, window=0, out=None, lse=False, tree=None):
        """The attention of the rows q (ntok, heads, head_dim) over their
        sequences: (out (ntok, heads * head_dim), lse (ntok, heads) or None).
        out: a tensor to write, of the compute type or int16 (q16).  tree
        (RaggedBatch.tree, of the same window): of the new rows each sees
        itself and its ancestors."""
        g = self.gpu
        self._same_device(batch)
        qs = self._rows(q, self.qtype, batch.ntok, "q")
        if out is None:
            out, kind, os_ = torch.empty((batch.ntok, self.width), dtype=self.qtype, device=g.device), self.ckind, self.width
        else:
            kind = _l.E_Q16 if out.dtype == torch.int16 else self.ckind
            os_ = self._rows(out, out.dtype if kind == _l.E_Q16 else self.qtype, batch.ntok, "out")
        if tree is not None:
            self._same_batch(batch, tree)
            if tree.window != window:
                raise ValueError("the tree's window is %d, not %d" % (tree.window, window))
        d = self.d
        key = (d.kind, self.heads, self.kv_heads, self.head_dim, d.page_size, d.k_row, d.v_row, window, tree is None)
        need = batch.ws.get(key)
        L = _l.load()
        known = need is not None
        if not known:
            size = L.vgx_paged_attn_ws if tree is None else L.vgx_paged_attn_tree_ws
            need = int(size(g.ctx, self.ref, batch.ref, window))
        ws = torch.empty(need, dtype=torch.uint8, device=g.device) if need else None
        z = torch.empty((batch.ntok, self.heads), dtype=torch.float32, device=g.device) if lse else None
        r = _l.PagedQuery(q.data_ptr(), qs, scale, window, kind, out.data_ptr(), os_, _at(z), _at(ws), need)
        if tree is None:
            g.on_current(L.vgx_paged_attn, self.ref, batch.ref, ctypes.byref(r))
        else:
            g.on_current(L.vgx_paged_attn_tree, self.ref, batch.ref, ctypes.byref(r), tree.ref)
        if not known:  # (a refused call's size is 0)
            batch.ws[key] = need
        return out, z

    def _same_batch(self, batch, tree):
        if tree.batch is not batch:
            raise ValueError("the tree is of another batch")

    def _same_device(self, batch):
        if batch.gpu is not self.gpu and batch.gpu.device != self.gpu.device:
            raise ValueError("the batch is on %s, the cache on %s" % (batch.gpu.device, self.gpu.device))

    def _rows(self, t, dtype, n, name):
        """The stride of n rows of heads x head_dim values, (n, heads, head_dim) or (n, heads * head_dim)."""
        if t.dim() != 3:
            return self.gpu.need_rows(t, dtype, n, self.width, name)
        self.gpu.need(t, dtype, 3, name)
        rows, heads, hd = t.shape
        st = t.stride()
        if (rows < n or heads != self.heads or hd != self.head_dim or st[2] != 1 or (heads > 1 and st[1] != hd)
                or (n > 1 and st[0] < self.width)):
            raise ValueError("%s must be (%d, %d, %d), a row's heads contiguous and its rows apart" % (
                name, n, self.heads, self.head_dim))
        return st[0] if n > 1 else self.width


class GPU:
    """One libvgx context on one device.  It issues on the stream that was
    torch's current one when it was made or use_torch_stream() was last called;
    the calls over a paged cache, sample and draft_verify issue on torch's
    current stream at the call.  Under torch.cuda.stream(...) call use_torch_stream()
    first, and again after, wherever both kinds are mixed: calls on different
    streams are not ordered with one another."""

    def __init__(self, device=0):
        L = _l.load()
        h = ctypes.c_void_p()
        _l.check(L.vgx_ctx_create(device, ctypes.byref(h)))
        self.ctx, self.device = h, torch.device("cuda", device)
        self._get_stream = L.vgx_ctx_stream
        self._verify_ws = {}  # draft_verify's workspace bytes by its sizes
        self.use_torch_stream()

    def use_torch_stream(self):
        """Later calls issue on torch's stream of now."""
        s = torch.cuda.current_stream(self.device).cuda_stream
        _l.check(_l.load().vgx_ctx_set_stream(self.ctx, ctypes.c_void_p(s)))

    def sync(self):
        _l.check(_l.load().vgx_ctx_sync(self.ctx))

    def on_current(self, call, *args):
        """call(ctx, *args) on torch's current stream of this device, where
        its tensors were made; the context's stream is put back after."""
        now, was = _raw_stream(self.device.index), self._get_stream(self.ctx) or 0
        if now == was:
            st = call(self.ctx, *args)
        else:
            L = _l.load()
            _l.check(L.vgx_ctx_set_stream(self.ctx, now))
            st = call(self.ctx, *args)
            L.vgx_ctx_set_stream(self.ctx, was)
        if st:
            _l.check(st)

    def need(self, t, dtype, dims, name):
        """Refuses a tensor of another device, type or number of dimensions."""
        if t.dim() != dims or (dtype is not None and t.dtype is not dtype) or t.device != self.device:
            raise ValueError("%s must be a %d-dimensional %s tensor on %s, not %s on %s" % (
                name, dims, dtype or t.dtype, self.device, t.dtype, t.device))

    def need_rows(self, t, dtype, n, width, name):
        """Refuses all but n rows of width contiguous values; their stride."""
        self.need(t, dtype, 2, name)
        rows, cols = t.shape
        st = t.stride()
        if rows < n or cols != width or (width > 1 and st[1] != 1) or (n > 1 and st[0] < width):
            raise ValueError("%s must be %d rows of %d contiguous values that do not overlap, not %s with strides %s" % (
                name, n, width, tuple(t.shape), st))
        return st[0] if n > 1 else width

    def need_values(self, t, dtype, n, name):
        """Refuses all but n contiguous values."""
        if t.dtype is not dtype or t.device != self.device or t.shape != (n,) or not t.is_contiguous():
            raise ValueError("%s must be %d contiguous %s values on %s" % (name, n, dtype, self.device))

    # -- weights
    def upload(self, m: Matrix):
        keep = [np.ascontiguousarray(m.body, np.uint8)]
        plane = s16 = m16 = None
        if m.plane is not None:
            plane = np.ascontiguousarray(m.plane, np.float32)
        if m.kind == "q4":
            s16 = np.ascontiguousarray(m.s16, np.int16)
            m16 = np.ascontiguousarray(m.m16, np.int16)
        d = _l.WeightDesc(_l.KIND[m.kind], m.rows, m.cols, _np_ptr(keep[0]), keep[0].size, int(m.prebiased),
                          float(m.scale), _np_ptr(plane), _np_ptr(s16), _np_ptr(m16), float(m.scale_mul))
        h = ctypes.c_void_p()
        _l.check(_l.load().vgx_mat_upload(self.ctx, ctypes.byref(d), ctypes.byref(h)))
        return Mat(self, h, m)

    def clone(self, mat):
        h = ctypes.c_void_p()
        _l.check(_l.load().vgx_mat_clone(self.ctx, mat.h, ctypes.byref(h)))
        c = Mat.__new__(Mat)
        c.gpu, c.h, c.rows, c.cols, c.kind = self, h, mat.rows, mat.cols, mat.kind
        return c

    def dequant(self, mat):
        out = torch.empty((mat.rows, mat.cols), dtype=torch.float32, device=self.device)
        _l.check(_l.load().vgx_dequant(self.ctx, mat.h, _ptr(out)))
        return out

    def group(self, mats):
        return Group(self, mats)

    def concat(self, mats):
        """One matrix with the rows of mats in order (q8 or t3, equal cols)."""
        arr = (ctypes.c_void_p * len(mats))(*[m.h for m in mats])
        h = ctypes.c_void_p()
        _l.check(_l.load().vgx_mat_concat(self.ctx, len(mats), arr, ctypes.byref(h)))
        c = Mat.__new__(Mat)
        c.gpu, c.h, c.rows, c.cols, c.kind = self, h, sum(m.rows for m in mats), mats[0].cols, mats[0].kind
        return c

    def argmax_rows(self, v, out=None):
        """The first maximum of each row of a 2-D int16 tensor."""
        out = out if out is not None else torch.empty(v.shape[0], dtype=torch.int32, device=v.device)
        _l.check(_l.load().vgx_argmax_rows(self.ctx, v.shape[0], v.shape[1], _ptr(v), _ptr(out)))
        return out

    def logits_chunks(self, logits, temp):
        """The candidate pass over a q16 logits row: an int32 tensor of
        ceil(n / 16) x 6 chunk records (v1, i1, v2, i2, max, sum on 1/2048)."""
        n = logits.numel()
        out = torch.empty(((n + 15) // 16, 6), dtype=torch.int32, device=logits.device)
        _l.check(_l.load().vgx_logits_chunks(self.ctx, _ptr(logits), n, float(temp), _ptr(out)))
        return out

    # -- GEMV family
    def matvec(self, mat, x, res=None, out=None):
        """matvec_to / matvec_add: y = q16(W.x [+ res])."""
        out = out if out is not None else torch.empty(mat.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemv(self.ctx, mat.h, _ptr(x), _ptr(res), _ptr(out)))
        return out

    def plan(self, mat):
        """(lanes per row, rows per lane) of a GEMV launch over mat."""
        lpr, ri = ctypes.c_int(), ctypes.c_int()
        _l.check(_l.load().vgx_gemv_plan_info(self.ctx, mat.h, ctypes.byref(lpr), ctypes.byref(ri)))
        return lpr.value, ri.value

    def matvec_f32(self, mat, x, out=None):
        out = out if out is not None else torch.empty(mat.rows, dtype=torch.float32, device=x.device)
        _l.check(_l.load().vgx_gemv_f32(self.ctx, mat.h, _ptr(x), _ptr(out)))
        return out

    def matvec_add_split(self, mat, split, x, res, out=None):
        """matvec_add(w2a) then matvec_add(w2b) over the column halves."""
        out = out if out is not None else torch.empty(mat.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemv_add_split(self.ctx, mat.h, split, _ptr(x), _ptr(res), _ptr(out)))
        return out

    def ffn_gate(self, w1, w3, x, hs=0, out=None):
        out = out if out is not None else torch.empty(w1.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_ffn_gate(self.ctx, w1.h, w3.h, _ptr(x), hs, _ptr(out)))
        return out

    def rmsnorm(self, x, w, eps=1e-5, out=None):
        out = out if out is not None else torch.empty_like(x)
        _l.check(_l.load().vgx_rmsnorm(self.ctx, x.numel(), _ptr(x), _ptr(w), float(eps), _ptr(out)))
        return out

    # -- batched prefill: x is (ntok, cols), outputs (ntok, rows)
    def gemm(self, mat, x, res=None, out=None):
        n = x.shape[0]
        out = out if out is not None else torch.empty((n, mat.rows), dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemm(self.ctx, mat.h, n, _ptr(x), _ptr(res), _ptr(out)))
        return out

    def gemm_add_split(self, mat, split, x, res, out=None):
        n = x.shape[0]
        out = out if out is not None else torch.empty((n, mat.rows), dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemm_add_split(self.ctx, mat.h, split, n, _ptr(x), _ptr(res), _ptr(out)))
        return out

    def ffn_gate_batch(self, w1, w3, x, hs=0, out=None):
        n = x.shape[0]
        out = out if out is not None else torch.empty((n, w1.rows), dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_ffn_gate_batch(self.ctx, w1.h, w3.h, n, _ptr(x), hs, _ptr(out)))
        return out

    def gemm_norm(self, mat, x, res, rms_w, eps=1e-5, split=0):
        """gemm (or gemm_add_split when split) and the RMSNorm of the rows it
        wrote: (y, yn)."""
        n = x.shape[0]
        y = torch.empty((n, mat.rows), dtype=torch.int16, device=x.device)
        yn = torch.empty_like(y)
        L = _l.load()
        if split:
            _l.check(L.vgx_gemm_add_split_norm(self.ctx, mat.h, split, n, _ptr(x), _ptr(res), _ptr(y), _ptr(rms_w),
                                               float(eps), _ptr(yn)))
        else:
            _l.check(L.vgx_gemm_norm(self.ctx, mat.h, n, _ptr(x), _ptr(res), _ptr(y), _ptr(rms_w), float(eps),
                                     _ptr(yn)))
        return y, yn

    def gemm_rms(self, mat, x, rms_w, eps=1e-5, res=None, out=None):
        """rmsnorm_batch(x, rms_w, eps) then gemm, one launch."""
        n = x.shape[0]
        out = out if out is not None else torch.empty((n, mat.rows), dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemm_rms(self.ctx, mat.h, n, _ptr(x), _ptr(rms_w), float(eps), _ptr(res), _ptr(out)))
        return out

    def ffn_gate_batch_rms(self, w1, w3, x, rms_w, eps=1e-5, hs=0, out=None):
        """rmsnorm_batch(x, rms_w, eps) then ffn_gate_batch, one launch."""
        n = x.shape[0]
        out = out if out is not None else torch.empty((n, w1.rows), dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_ffn_gate_batch_rms(self.ctx, w1.h, w3.h, n, _ptr(x), _ptr(rms_w), float(eps), hs,
                                                  _ptr(out)))
        return out

    def rmsnorm_batch(self, x, w, eps=1e-5, out=None):
        out = out if out is not None else torch.empty_like(x)
        _l.check(_l.load().vgx_rmsnorm_batch(self.ctx, x.shape[0], x.shape[1], _ptr(x), _ptr(w), float(eps),
                                             _ptr(out)))
        return out

    def embed_q8_batch(self, emb, emb_scale, tokens, out=None):
        vocab, dim = emb.shape
        n = tokens.numel()
        out = out if out is not None else torch.empty((n, dim), dtype=torch.int16, device=emb.device)
        _l.check(_l.load().vgx_embed_q8_batch(self.ctx, _ptr(emb), _ptr(emb_scale), vocab, dim, n, _ptr(tokens),
                                              _ptr(out)))
        return out

    def embed_q8_rms_batch(self, emb, emb_scale, tokens, rms_w, eps=1e-5):
        """(embedding rows, their RMSNorm) of a batch of tokens, one launch."""
        vocab, dim = emb.shape
        n = tokens.numel()
        x = torch.empty((n, dim), dtype=torch.int16, device=emb.device)
        y = torch.empty((n, dim), dtype=torch.int16, device=emb.device)
        _l.check(_l.load().vgx_embed_q8_rms_batch(self.ctx, _ptr(emb), _ptr(emb_scale), vocab, dim, n, _ptr(tokens),
                                                  _ptr(x), _ptr(rms_w), ctypes.c_float(eps), _ptr(y)))
        return x, y

    def matvec_rms(self, mat, x, rms_w, eps=1e-5, res=None, out=None):
        """rmsnorm(x, rms_w, eps) then matvec_add, one launch."""
        out = out if out is not None else torch.empty(mat.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_gemv_rms(self.ctx, mat.h, _ptr(x), _ptr(rms_w), float(eps), _ptr(res), _ptr(out)))
        return out

    def ffn_gate_rms(self, w1, w3, x, rms_w, eps=1e-5, hs=0, out=None):
        """rmsnorm(x, rms_w, eps) then the fused FFN gate, one launch."""
        out = out if out is not None else torch.empty(w1.rows, dtype=torch.int16, device=x.device)
        _l.check(_l.load().vgx_ffn_gate_rms(self.ctx, w1.h, w3.h, _ptr(x), _ptr(rms_w), float(eps), hs, _ptr(out)))
        return out

    def decode_advance(self, pos, token, hist):
        """hist[pos + 1] = token (inside hist), then ++pos; device scalars."""
        _l.check(_l.load().vgx_decode_advance(self.ctx, _ptr(pos), _ptr(token), _ptr(hist), int(hist.numel())))

    def embed_q8(self, emb, emb_scale, token, out=None):
        vocab, dim = emb.shape
        out = out if out is not None else torch.empty(dim, dtype=torch.int16, device=emb.device)
        _l.check(_l.load().vgx_embed_q8(self.ctx, _ptr(emb), _ptr(emb_scale), vocab, dim, _ptr(token), _ptr(out)))
        return out

    def attention(self, **kw):
        return Attention(self, **kw)

    def paged_cache(self, heads, kv_heads, head_dim, kind, k, v, k_step=0.0, v_step=0.0):
        return PagedCache(self, heads, kv_heads, head_dim, kind, k, v, k_step, v_step)

    def paged_layers(self, caches):
        return PagedLayers(caches)

    def sample(self, logits, u, temp=None, top_k=None, top_p=None, min_p=None):
        """A token of each row of logits (rows, vocab; float32, bfloat16,
        float16 or q16) by the random numbers u in [0, 1), after the cuts that
        are given, a value a row: temp (0: greedy), top_k (0: all), top_p (1:
        all), min_p (0: all).  Returns (token, tokens that stay, the token's
        probability among them).  On torch's current stream."""
        kind = _ELEM.get(logits.dtype)
        if kind is None or logits.dim() != 2:
            raise ValueError("logits must be rows of float32, bfloat16, float16 or int16 (q16)")
        n, vocab = logits.shape
        stride = self.need_rows(logits, None, n, vocab, "logits")
        self.need_values(u, _F32, n, "u")
        for t, dtype, name in ((temp, _F32, "temp"), (top_k, _I32, "top_k"), (top_p, _F32, "top_p"),
                               (min_p, _F32, "min_p")):
            if t is not None:
                self.need_values(t, dtype, n, name)
        L, dev = _l.load(), self.device
        need = int(L.vgx_sample_ws(n, vocab, kind))
        token = torch.empty(n, dtype=_I32, device=dev)
        kept, prob = torch.empty_like(token), torch.empty_like(u)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        a = _l.Sampling(n, vocab, kind, logits.data_ptr(), stride, u.data_ptr(), _at(temp), _at(top_k), _at(top_p),
                        _at(min_p), token.data_ptr(), kept.data_ptr(), prob.data_ptr(), _at(ws), need)
        self.on_current(L.vgx_sample, ctypes.byref(a))
        return token, kept, prob

    def draft_verify(self, qstart, tokens, logits, u_accept, u_next, draft=None, temp=None):
        """Drafted tokens against the target's logits (rows, vocab; float32,
        bfloat16, float16 or q16): tokens[r + 1] against row r of its sequence
        (rows qstart[s] .. qstart[s+1]-1).  draft: the logits the drafts were
        drawn from; temp: a temperature a sequence (0: greedy).  Returns
        (accepted drafts and next token of each sequence, the target's
        probability of each drafted token); rows of no sequence have none."""
        nseq, n = qstart.shape[0] - 1, tokens.shape[0]
        if nseq < 0:
            raise ValueError("qstart must hold at least one entry")
        for t, dtype, size, name in ((qstart, _I32, nseq + 1, "qstart"), (tokens, _I32, n, "tokens"),
                                     (u_accept, _F32, n, "u_accept"), (u_next, _F32, nseq, "u_next"),
                                     (temp, _F32, nseq, "temp")):
            if t is not None:
                self.need_values(t, dtype, size, name)
        kind = _ELEM.get(logits.dtype)
        if kind is None or logits.dim() != 2:
            raise ValueError("logits must be rows of float32, bfloat16, float16 or int16 (q16)")
        vocab = logits.shape[1]
        stride = self.need_rows(logits, None, n, vocab, "logits")
        dstride = 0 if draft is None else self.need_rows(draft, logits.dtype, n, vocab, "draft")
        L = _l.load()
        key = (nseq, n, vocab, kind, draft is not None)
        need = self._verify_ws.get(key)
        if need is None:
            if len(self._verify_ws) > 1000:
                self._verify_ws.clear()
            need = self._verify_ws[key] = int(L.vgx_draft_verify_ws(*key))
        dev = self.device
        accepted = torch.empty(nseq, dtype=_I32, device=dev)
        nxt = torch.empty(nseq, dtype=_I32, device=dev)
        prob = torch.empty(n, dtype=_F32, device=dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a = _l.Draft(nseq, n, vocab, qstart.data_ptr(), tokens.data_ptr(), kind, logits.data_ptr(), stride, _at(draft),
                     dstride, _at(temp), u_accept.data_ptr(), u_next.data_ptr(), accepted.data_ptr(), nxt.data_ptr(),
                     prob.data_ptr(), ws.data_ptr(), need)
        self.on_current(L.vgx_draft_verify, ctypes.byref(a))
        return accepted, nxt, prob

    def conv(self, w, layer_is_conv=None):
        return Conv(self, w, layer_is_conv)

    def close(self):
        if self.ctx:
            _l.load().vgx_ctx_destroy(self.ctx)
            self.ctx = None


def quantize_act(v):
    """quantize_act on the host (libvgx's helper)."""
    v = np.ascontiguousarray(v, np.float32).ravel()
    q = np.empty(v.size, np.int16)
    _l.load().vgx_quantize_act(_np_ptr(v), v.size, _np_ptr(q))
    return q


def x_pack_i16_2(v):
    v = np.ascontiguousarray(v, np.float32).ravel()
    out = np.empty(4 * ((v.size + 1) // 2), np.uint8)
    _l.load().vgx_x_pack_i16_2(_np_ptr(v), v.size, _np_ptr(out))
    return out
