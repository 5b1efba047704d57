"""A paged key/value cache: the keys and values of many sequences in one pool of pages that a table names, and what fills and reads it.

For a server that decodes sequences of different lengths together: `append` post-processes and stores new tokens' rows, `attention` is one new token
of every sequence over all of its rows (or a window), `key_bounds` / `select` / `attention_selected` the same over the pages whose
keys promise most, `rows` a cached prefix as f32 rows for decode.causal_attention. The reference keeps one sequence a cache and has no
counterpart. Everything runs through libferric_hip; there is no CPU path.
"""
import ctypes as C

import numpy as np

from . import _lib
from .qmatrix import BF16, F16, F32, Q8_0, DeviceBuffer, Tensor, _arrived, _upload

ALL = (F32, F16, BF16, Q8_0)
NO_PAGE = 0xFFFFFFFF
_VALUE_BYTES = {F32: 4, F16: 2, BF16: 2, Q8_0: 1}


def _buf(t):
    return None if t is None else t.buf


def _at(stream):
    return None if stream is None else stream.handle


class PagedKvCache:
    """Pools [n_pages * page_rows, n_kv * head_dim] of keys and of values (type F32, F16, BF16 or Q8_0: codes and f16 scales as kvquant stores them) and a table
    [n_seq, pages_per_seq] of page numbers: position p of sequence i is row table[i, p / page_rows] * page_rows + p % page_rows. Which page belongs to whom is
    the caller's to decide (set_table)."""

    def __init__(self, ty, page_rows, n_pages, n_kv, head_dim, n_seq, pages_per_seq):
        assert ty in ALL, f"a paged cache holds F32, F16, BF16 or Q8_0, not ggml type {ty}"
        values = n_pages * page_rows * n_kv * head_dim
        pools = [DeviceBuffer(max(values * _VALUE_BYTES[ty], 16)) for _ in range(2)]
        scales = [DeviceBuffer(max(values // 32 * 2, 16)) if ty == Q8_0 else None for _ in range(2)]
        table = DeviceBuffer(max(4 * n_seq * pages_per_seq, 16))
        self._take(ty, page_rows, n_pages, n_kv, head_dim, *pools, *scales, table, n_seq, pages_per_seq)
        self.set_table(np.full((n_seq, pages_per_seq), NO_PAGE, np.uint32))

    @staticmethod
    def wrap(ty, page_rows, n_pages, n_kv, head_dim, k, v, k_scales, v_scales, table, n_seq, pages_per_seq):
        """Over device memory the caller already has (objects with a `ptr`, kept alive here); scales None unless Q8_0."""
        cache = object.__new__(PagedKvCache)
        cache._take(ty, page_rows, n_pages, n_kv, head_dim, k, v, k_scales, v_scales, table, n_seq, pages_per_seq)
        return cache

    def _take(self, ty, page_rows, n_pages, n_kv, head_dim, k, v, k_scales, v_scales, table, n_seq, pages_per_seq):
        _lib.init()
        self.type, self.page_rows, self.n_pages, self.n_kv, self.head_dim = ty, page_rows, n_pages, n_kv, head_dim
        self.k, self.v, self.k_scales, self.v_scales, self.table, self.n_seq, self.pages_per_seq = k, v, k_scales, v_scales, table, n_seq, pages_per_seq
        at = lambda b: None if b is None else getattr(b.ptr, "value", b.ptr)      # noqa: E731
        self._desc = _lib.Paged(ty, page_rows, n_pages, n_kv, head_dim, at(k), at(v), at(k_scales), at(v_scales), at(table), n_seq, pages_per_seq, pages_per_seq)
        self._ref, self._addr = C.byref(self._desc), C.addressof(self._desc)
        self._ws, self._needs, self._rows = {}, {}, n_kv * head_dim

    def set_table(self, pages, stream=None):
        """The whole table from the host, [n_seq, pages_per_seq]; NO_PAGE (or any number past the pool) where a sequence has none."""
        a = np.ascontiguousarray(pages, dtype=np.uint32)
        assert a.shape == (self.n_seq, self.pages_per_seq), f"the table is {[self.n_seq, self.pages_per_seq]}, not {list(a.shape)}"
        if a.nbytes:
            _upload(self.table, a, stream)
            _arrived(a, stream)

    def _workspace(self, n_heads, keys, ws, stream):
        """The caller's workspace, or one kept for the stream, for attention over `keys` keys a sequence (n_heads 0: for select). What was outgrown stays: a graph captured on
        the stream may name it. Graphs that may run at the same time need workspaces of their own."""
        need = self._needs.get((n_heads, keys))
        if need is None:
            lib = _lib.load()
            if len(self._needs) > 1000:               # sizes of lengths that are past
                self._needs.clear()
            need = self._needs[n_heads, keys] = lib.fhip_paged_attention_ws_bytes(self._ref, n_heads, keys) if n_heads else lib.fhip_paged_select_ws_bytes(self._ref, keys)
        if ws is not None:
            assert getattr(ws, "nbytes", need) >= need, f"a workspace of {ws.nbytes} bytes, {need} are needed"
            return ws
        if need == 0:
            return None
        kept = self._ws.setdefault(None if stream is None else stream.handle.value, [])
        if not kept or kept[-1].nbytes < need:
            kept.append(DeviceBuffer(1 << (need - 1).bit_length()))
        return kept[-1]

    def reserve(self, n_heads, max_len, n_select=0, stream=None):
        """Makes the workspace that attention (and, with n_select pages, select and attention_selected) of up to max_len keys takes on this stream, which a capture cannot."""
        self._workspace(n_heads, max_len, None, stream)
        if n_select:
            self._workspace(0, max_len, None, stream)
            self._workspace(n_heads, n_select * self.page_rows, None, stream)

    def append(self, qkv, seqs, positions, n_heads, base, n_rot=None, interleaved=False, eps=1e-6, bias=None, q_norm=None, k_norm=None, freq_scale=None, out=None, stream=None):
        """Post-processes the fused rows qkv [t, (n_heads + 2 n_kv) * head_dim] of t new tokens (bias, head norm, rotation), stores their keys and values, returns their
        queries [t, n_heads * head_dim]. seqs, positions: device u32 Tensors [t]; seqs None: token i is of sequence i."""
        t, width = qkv.shape
        hd = self.head_dim
        assert width == n_heads * hd + 2 * self._rows, f"append: rows of {width} values are not {n_heads} + 2 * {self.n_kv} heads of {hd}"
        assert positions.numel() == t and (t <= self.n_seq if seqs is None else seqs.numel() == t), "append: one position and one sequence a row"
        assert (bias is None or bias.numel() == width) and (q_norm is None or q_norm.numel() == hd) and (k_norm is None or k_norm.numel() == hd), "append: bias or norm of another size"
        if n_rot is None:
            n_rot = hd
        assert freq_scale is None or 2 * freq_scale.numel() >= n_rot, "append: a frequency scale for every pair"
        q = Tensor.empty((t, n_heads * hd)) if out is None else out
        assert q.shape == (t, n_heads * hd), "append: out has another shape"
        _lib.paged_append(self._addr, qkv.buf, _buf(bias), _buf(q_norm), _buf(k_norm), _buf(seqs), positions.buf, _buf(freq_scale), t, n_heads, n_rot, interleaved, eps, base, q.buf,
                          _at(stream))
        return q

    def _query(self, q, lens, n_heads, out):
        assert q.shape == (self.n_seq, n_heads * self.head_dim), f"one query row a sequence: {[self.n_seq, n_heads * self.head_dim]}, not {list(q.shape)}"
        assert lens.numel() == self.n_seq, "one length a sequence"
        if out is None:
            return Tensor.empty(q.shape)
        assert out.shape == q.shape, "out has another shape"
        return out

    def attention(self, q, lens, max_len, n_heads, window=0, softcap=0.0, out=None, ws=None, stream=None):
        """One new token of every sequence, q [n_seq, n_heads * head_dim], over the first lens[i] rows (device u32 Tensor, the new token's own among them; at most
        max_len) or the newest `window` of them. ws: scratch of the caller's in place of the cache's own for the stream; memory that does not say its nbytes is taken at the caller's word."""
        out = self._query(q, lens, n_heads, out)
        _lib.paged_attention(self._addr, q.buf, lens.buf, max_len, n_heads, window, softcap, self._workspace(n_heads, max_len, ws, stream), out.buf, _at(stream))
        return out

    def empty_bounds(self):
        """Room for the pages' key bounds, [n_pages, n_kv, 2, head_dim]; key_bounds fills a page's when its first row is appended."""
        return Tensor.empty((self.n_pages, self.n_kv, 2, self.head_dim))

    def key_bounds(self, lens, max_new, bounds, fresh=None, stream=None):
        """Takes the keys of each sequence's last `fresh` rows (device u32 Tensor; None: max_new) into their pages' bounds, in place."""
        assert lens.numel() == self.n_seq and (fresh is None or fresh.numel() == self.n_seq), "one length a sequence"
        assert bounds.numel() == self.n_pages * self.n_kv * 2 * self.head_dim, "key_bounds: bounds of another size"
        _lib.paged_key_bounds(self._addr, lens.buf, _buf(fresh), max_new, bounds.buf, _at(stream))
        return bounds

    def select(self, q, lens, max_len, bounds, n_heads, n_select, first=1, last=1, out=None, ws=None, stream=None):
        """The n_select pages of every sequence and KV head that promise most, [n_seq, n_kv, n_select] u32, ascending, NO_PAGE behind the last."""
        self._query(q, lens, n_heads, q)
        assert bounds.numel() == self.n_pages * self.n_kv * 2 * self.head_dim, "select: bounds of another size"
        shape = (self.n_seq, self.n_kv, n_select)
        out = Tensor.empty(shape, np.uint32) if out is None else out
        assert out.shape == shape, "select: out has another shape"
        _lib.paged_select(self._addr, q.buf, lens.buf, max_len, bounds.buf, n_heads, n_select, first, last, self._workspace(0, max_len, ws, stream), out.buf,
                          _at(stream))
        return out

    def attention_selected(self, q, lens, selected, n_heads, softcap=0.0, out=None, ws=None, stream=None):
        """attention over the rows of the selected pages [n_seq, n_kv, n] only."""
        out = self._query(q, lens, n_heads, out)
        assert selected.shape[:2] == (self.n_seq, self.n_kv) and len(selected.shape) == 3, "selected is [n_seq, n_kv, n]"
        n = selected.shape[2]
        ws = self._workspace(n_heads, n * self.page_rows, ws, stream)
        _lib.paged_attention_selected(self._addr, q.buf, lens.buf, selected.buf, n, n_heads, softcap, ws, out.buf, _at(stream))
        return out

    def rows(self, seq, row0, rows, out=None, stream=None):
        """Rows row0 .. row0 + rows of sequence seq as f32: (k, v), [rows, n_kv * head_dim] each. Rows of a table entry that names no page are not written: they stay as `out` has
        them, and without `out` hold anything."""
        shape = (rows, self._rows)
        k, v = (Tensor.empty(shape), Tensor.empty(shape)) if out is None else out
        assert k.shape == v.shape == shape, "rows: out has another shape"
        _lib.paged_rows(self._addr, seq, row0, rows, k.buf, v.buf, _at(stream))
        return k, v
