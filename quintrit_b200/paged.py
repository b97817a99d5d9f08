"""A key / value cache in pages and its attention (``quintrit_b200_paged_*``), on torch CUDA tensors.

``PagedCache`` owns the pages of all layers; which of them a sequence has is the caller's page table. ``PagedRows`` describes the new tokens of a
call: their place in packed arrays, the lengths of their sequences and the page tables, all in device memory, so that one object serves every layer
of a step, and a captured graph serves what its tensors hold when it is replayed. Calls are enqueued on the current torch stream of the cache's
device (or the ``stream`` given) and do not wait; ``status()`` reports what they met.
"""
from __future__ import annotations

import ctypes as C

from . import api as _api

F32, F16, BF16, Q8 = 0, 1, 2, 3
_CACHE_TYPES = {"f16": F16, "bf16": BF16, "q8": Q8}
_sz, _vp, _u32, _i32, _f32 = C.c_size_t, C.c_void_p, C.c_uint32, C.c_int32, C.c_float


class _RowsC(C.Structure):
    _fields_ = [("struct_size", _u32), ("sequences", _u32), ("tokens", _u32), ("max_new", _u32), ("max_length", _u32), ("table_stride", _u32), ("d_starts", _vp),
                ("d_lengths", _vp), ("d_table", _vp)]


class _AppendC(C.Structure):
    _fields_ = [("struct_size", _u32), ("type", _i32), ("q_out_type", _i32), ("q_heads", _u32), ("d_q", _vp), ("d_k", _vp), ("d_v", _vp), ("q_token_stride", _sz),
                ("q_head_stride", _sz), ("k_token_stride", _sz), ("k_head_stride", _sz), ("v_token_stride", _sz), ("v_head_stride", _sz), ("d_q_out", _vp),
                ("out_token_stride", _sz), ("out_head_stride", _sz), ("d_q_norm", _vp), ("d_k_norm", _vp), ("norm_eps", _f32), ("d_cos_sin", _vp), ("positions", _u32),
                ("rope_dims", _u32), ("neox", _i32)]


class _AttentionC(C.Structure):
    _fields_ = [("struct_size", _u32), ("q_type", _i32), ("out_type", _i32), ("q_heads", _u32), ("d_q", _vp), ("q_token_stride", _sz), ("q_head_stride", _sz), ("d_out", _vp),
                ("out_token_stride", _sz), ("out_head_stride", _sz), ("scale", _f32), ("cap", _f32), ("window", _u32), ("d_workspace", _vp), ("workspace_bytes", _sz)]


_bound = None


def _lib():
    global _bound
    if _bound is None:
        lib = _api.load_library()
        lib.quintrit_b200_paged_cache_create.argtypes = [_u32] * 6 + [_i32, C.POINTER(_vp)]
        lib.quintrit_b200_paged_cache_free.argtypes = [_vp]
        lib.quintrit_b200_paged_cache_info.argtypes = [_vp, C.POINTER(_sz), C.POINTER(_u32)]
        lib.quintrit_b200_paged_cache_status.argtypes = [_vp]
        lib.quintrit_b200_paged_append_device.argtypes = [_vp, _u32, C.POINTER(_RowsC), C.POINTER(_AppendC), _vp]
        lib.quintrit_b200_paged_read_device.argtypes = [_vp, _u32, C.POINTER(_RowsC), _i32, _vp, _vp, _vp]
        lib.quintrit_b200_paged_attention_workspace.argtypes = [_vp, C.POINTER(_RowsC), _u32, C.POINTER(_sz)]
        lib.quintrit_b200_paged_attention_device.argtypes = [_vp, _u32, C.POINTER(_RowsC), C.POINTER(_AttentionC), _vp]
        _bound = lib
    return _bound


_dtypes = None


def _type_of(t) -> int:
    global _dtypes
    if _dtypes is None:
        import torch

        _dtypes = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
    try:
        return _dtypes[t.dtype]
    except KeyError:
        raise ValueError(f"tensors of heads are float32, float16 or bfloat16, got {t.dtype}") from None


class PagedRows:
    """The new tokens of a call. ``starts`` [sequences + 1], ``lengths`` [sequences] and ``table`` [sequences][pages per sequence] are int32 CUDA tensors
    that stay the caller's to change between calls; sequence s has the packed tokens ``starts[s] .. starts[s + 1] - 1``, the last of them at position
    ``lengths[s] - 1``, and position p lies in page ``table[s][p // page_tokens]``. ``tokens``: rows of the packed arrays; ``max_new``: no sequence has
    more new tokens; ``max_length``: no sequence is longer, as far as is known (it divides the work)."""

    def __init__(self, starts, lengths, table, tokens: int, max_new: int, max_length: int):
        import torch

        for name, t, dim in (("starts", starts, 1), ("lengths", lengths, 1), ("table", table, 2)):
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_cuda or (t.numel() > 1 and t.stride(-1) != 1):
                raise ValueError(f"{name} is a {dim}-dimensional int32 CUDA tensor with consecutive values")
        n = lengths.numel()
        if starts.numel() != n + 1 or table.shape[0] != n:
            raise ValueError(f"{n} lengths go with {n + 1} starts and {n} rows of the table, got {starts.numel()} and {table.shape[0]}")
        if n > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("the rows of the table overlap")
        if not starts.device == lengths.device == table.device:
            raise ValueError("starts, lengths and table lie on different devices")
        self.starts, self.lengths, self.table, self.tokens = starts, lengths, table, tokens
        # (the rows of a table may lie further apart than they are long: what lies between is not the sequence's, but pages beyond a length are never looked at)
        self._c = _RowsC(C.sizeof(_RowsC), n, tokens, max_new, max_length, table.stride(0) if n > 1 else table.shape[1], starts.data_ptr(), lengths.data_ptr(), table.data_ptr())
        self._p = C.byref(self._c)
        self.device = starts.device


class PagedCache:
    """``pages`` pages of ``page_tokens`` positions in each of ``layers`` layers, keys and values of ``kv_heads`` heads of ``head_dim`` values, stored as
    ``dtype`` "f16", "bf16" or "q8" (8-bit codes and a 32-bit scale per position and head)."""

    def __init__(self, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, dtype: str = "f16", device: int = 0):
        self._h = _vp()
        if dtype not in _CACHE_TYPES:
            raise ValueError(f"a paged cache is stored as {', '.join(_CACHE_TYPES)}, got {dtype!r}")
        self._lib = _lib()
        _api._check(self._lib.quintrit_b200_paged_cache_create(device, layers, pages, page_tokens, kv_heads, head_dim, _CACHE_TYPES[dtype], C.byref(self._h)))
        self.layers, self.pages, self.page_tokens, self.kv_heads, self.head_dim, self.dtype, self.device = layers, pages, page_tokens, kv_heads, head_dim, dtype, device

    @property
    def device_bytes(self) -> int:
        n = _sz(0)
        _api._check(self._lib.quintrit_b200_paged_cache_info(self._h, C.byref(n), None))
        return n.value

    def _stream(self, stream):
        if stream is not None:
            return stream
        import torch

        return torch.cuda.current_stream(self.device).cuda_stream

    def _heads(self, name, t, tokens, heads=None):
        if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads) or t.stride(2) != 1:
            raise ValueError(f"{name} is [{tokens}][{'heads' if heads is None else heads}][{self.head_dim}] with the values of a head side by side, got {tuple(t.shape)}, strides {t.stride()}")
        if t.get_device() != self.device:
            raise ValueError(f"{name} is not on the cache's device {self.device}")
        return t

    def _rows(self, rows):
        if rows.device.index != self.device:
            raise ValueError(f"the rows' tensors are not on the cache's device {self.device}")
        return rows

    def append(self, layer: int, rows: PagedRows, q, k, v, *, q_out=None, q_norm=None, k_norm=None, eps: float = 1e-6, cos_sin=None, neox: bool = False, stream=None):
        """Normalises and rotates the new tokens' query and key heads, writes keys and values to the cache and returns the queries (``q_out``, by default new
        and of the queries' type; None if ``q`` is None). ``q_norm`` / ``k_norm``: float32 weights [head_dim]; ``cos_sin``: float32 [positions][rotated values]
        with cos at 2 i and sin at 2 i + 1; ``neox``: pairs (i, i + half) instead of (2 i, 2 i + 1)."""
        import torch

        rows, n = self._rows(rows), rows.tokens
        k, v = self._heads("k", k, n, self.kv_heads), self._heads("v", v, n, self.kv_heads)
        a = _AppendC(C.sizeof(_AppendC))
        a.type = _type_of(k)
        if _type_of(v) != a.type or (q is not None and _type_of(q) != a.type):
            raise ValueError("q, k and v have the same type")
        if q is not None:
            self._heads("q", q, n)
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            self._heads("q_out", q_out, n, q.shape[1])
            a.q_out_type, a.q_heads, a.d_q, a.d_q_out = _type_of(q_out), q.shape[1], q.data_ptr(), q_out.data_ptr()
            a.q_token_stride, a.q_head_stride = q.stride(0), q.stride(1)
            a.out_token_stride, a.out_head_stride = q_out.stride(0), q_out.stride(1)
        else:
            q_out = None
        a.d_k, a.k_token_stride, a.k_head_stride = k.data_ptr(), k.stride(0), k.stride(1)
        a.d_v, a.v_token_stride, a.v_head_stride = v.data_ptr(), v.stride(0), v.stride(1)
        if q_norm is not None or k_norm is not None:
            for w in (q_norm, k_norm):
                if w is not None and (w.dtype != torch.float32 or w.shape != (self.head_dim,) or not w.is_contiguous() or w.get_device() != self.device):
                    raise ValueError(f"norm weights are float32 [{self.head_dim}] on the cache's device")
            a.d_q_norm = None if q_norm is None else q_norm.data_ptr()
            a.d_k_norm = None if k_norm is None else k_norm.data_ptr()
            a.norm_eps = eps
        if cos_sin is not None:
            if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.get_device() != self.device:
                raise ValueError("cos_sin is a contiguous float32 [positions][rotated values] on the cache's device")
            a.d_cos_sin, a.positions, a.rope_dims, a.neox = cos_sin.data_ptr(), cos_sin.shape[0], cos_sin.shape[1], int(neox)
        rc = self._lib.quintrit_b200_paged_append_device(self._h, layer, rows._p, C.byref(a), self._stream(stream))
        if rc != 0:
            _api._check(rc)
        return q_out

    def read(self, layer: int, rows: PagedRows, *, k_out=None, v_out=None, dtype=None, stream=None):
        """The new tokens' rows of the cache, dense: (keys, values), each [tokens][kv_heads][head_dim]. With whole sequences as "new" tokens: all that is cached.
        ``dtype``: of the results where they are not given (default float16)."""
        import torch

        rows, n = self._rows(rows), rows.tokens
        if k_out is None and v_out is None:
            k_out, v_out = (torch.empty((n, self.kv_heads, self.head_dim), dtype=dtype or torch.float16, device=rows.device) for _ in range(2))
        given = [t for t in (k_out, v_out) if t is not None]
        for t in given:
            self._heads("an output", t, n, self.kv_heads)
            if not t.is_contiguous() or t.dtype != given[0].dtype:
                raise ValueError("outputs are contiguous and of one type")
        rc = self._lib.quintrit_b200_paged_read_device(self._h, layer, rows._p, _type_of(given[0]), None if k_out is None else k_out.data_ptr(),
                                                       None if v_out is None else v_out.data_ptr(), self._stream(stream))
        if rc != 0:
            _api._check(rc)
        return k_out, v_out

    def attend_workspace(self, rows: PagedRows, q_heads: int):
        """Scratch memory for ``attend`` on these rows with that many query heads (a uint8 tensor, perhaps empty). Calls that may overlap need one each."""
        import torch

        n = _sz(0)
        _api._check(self._lib.quintrit_b200_paged_attention_workspace(self._h, rows._p, q_heads, C.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=rows.device)

    def attend(self, layer: int, rows: PagedRows, q, *, out=None, scale: float | None = None, cap: float = 0.0, window: int = 0, workspace=None, stream=None):
        """Attention of the new tokens' queries [tokens][query heads][head_dim] over the cached positions up to their own (the last ``window`` of them, if that
        is not 0), scores times ``scale`` (default head_dim ** -0.5), capped to ``cap`` tanh(score / ``cap``) if that is not 0. Returns ``out`` (by default
        new, of the queries' type). ``workspace``: from ``attend_workspace``, by default allocated by torch for this call on its current stream."""
        import torch

        rows, n = self._rows(rows), rows.tokens
        self._heads("q", q, n)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        self._heads("out", out, n, q.shape[1])
        if workspace is None:
            workspace = self.attend_workspace(rows, q.shape[1])
        elif workspace.get_device() != self.device or not workspace.is_contiguous():
            raise ValueError("the workspace is a contiguous tensor on the cache's device")
        a = _AttentionC(C.sizeof(_AttentionC), _type_of(q), _type_of(out), q.shape[1], q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                        self.head_dim ** -0.5 if scale is None else scale, cap, window, workspace.data_ptr(), workspace.numel() * workspace.element_size())
        rc = self._lib.quintrit_b200_paged_attention_device(self._h, layer, rows._p, C.byref(a), self._stream(stream))
        if rc != 0:
            _api._check(rc)
        return out

    def status(self) -> None:
        """Raises ``QuintritError`` if a call that has finished met something out of range since the last time this was asked."""
        _api._check(self._lib.quintrit_b200_paged_cache_status(self._h))

    def free(self) -> None:
        if self._h:
            self._lib.quintrit_b200_paged_cache_free(self._h)
            self._h = _vp()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
