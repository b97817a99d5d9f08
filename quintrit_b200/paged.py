"""A key / value cache in pages and its attention (``quintrit_b200_paged_*``), on torch CUDA tensors.

``PagedCache`` owns the pages of all layers; which of them a sequence has is the caller's page table. ``PagedRows`` describes the new tokens of a
call: their place in packed arrays, the lengths of their sequences and the page tables, all in device memory, so that one object serves every layer
of a step, and a captured graph serves what its tensors hold when it is replayed. Calls are enqueued on the current torch stream of the cache's
device (or the ``stream`` given, the number of a CUDA stream) and do not wait; ``status()`` reports what they met. Results that the caller does not bring
are allocated on the stream that the call runs on: another stream waits for it before it reads them, and tells torch so (``record_stream``) if it may still do so
when they are dropped.
"""
from __future__ import annotations

import ctypes as C
import struct

from . import api as _api

F32, F16, BF16, Q8 = 0, 1, 2, 3
_CACHE_TYPES = {"f16": F16, "bf16": BF16, "q8": Q8}
_sz, _vp, _u32, _i32, _f32 = C.c_size_t, C.c_void_p, C.c_uint32, C.c_int32, C.c_float


class _RowsC(C.Structure):
    _fields_ = [("struct_size", _u32), ("sequences", _u32), ("tokens", _u32), ("max_new", _u32), ("max_length", _u32), ("table_stride", _u32), ("d_starts", _vp),
                ("d_lengths", _vp), ("d_table", _vp), ("table_pages", _u32)]


class _AppendC(C.Structure):
    _fields_ = [("struct_size", _u32), ("type", _i32), ("q_out_type", _i32), ("q_heads", _u32), ("d_q", _vp), ("d_k", _vp), ("d_v", _vp), ("q_token_stride", _sz),
                ("q_head_stride", _sz), ("k_token_stride", _sz), ("k_head_stride", _sz), ("v_token_stride", _sz), ("v_head_stride", _sz), ("d_q_out", _vp),
                ("out_token_stride", _sz), ("out_head_stride", _sz), ("d_q_norm", _vp), ("d_k_norm", _vp), ("norm_eps", _f32), ("d_cos_sin", _vp), ("positions", _u32),
                ("rope_dims", _u32), ("neox", _i32)]


class _AttentionC(C.Structure):
    _fields_ = [("struct_size", _u32), ("q_type", _i32), ("out_type", _i32), ("q_heads", _u32), ("d_q", _vp), ("q_token_stride", _sz), ("q_head_stride", _sz), ("d_out", _vp),
                ("out_token_stride", _sz), ("out_head_stride", _sz), ("scale", _f32), ("cap", _f32), ("window", _u32), ("d_workspace", _vp), ("workspace_bytes", _sz)]


# The same layouts packed in one go: a call's arguments as bytes (a third of the time that filling the structures takes, on a path that a step walks once per layer).
_APPEND = struct.Struct("@IiiIPPPNNNNNNPNNPPfPIIi0P")
_ATTENTION = struct.Struct("@IiiIPNNPNNffIPN")
assert _APPEND.size == C.sizeof(_AppendC) and _ATTENTION.size == C.sizeof(_AttentionC)

_bound = None


def _lib():
    global _bound
    if _bound is None:
        lib = _api.load_library()
        lib.quintrit_b200_paged_cache_create.argtypes = [_u32] * 6 + [_i32, C.POINTER(_vp)]
        lib.quintrit_b200_paged_cache_free.argtypes = [_vp]
        lib.quintrit_b200_paged_cache_info.argtypes = [_vp, C.POINTER(_sz), C.POINTER(_u32)]
        lib.quintrit_b200_paged_cache_status.argtypes = [_vp]
        lib.quintrit_b200_paged_append_device.argtypes = [_vp, _u32, _vp, _vp, _vp]
        lib.quintrit_b200_paged_read_device.argtypes = [_vp, _u32, _vp, _i32, _vp, _vp, _vp]
        lib.quintrit_b200_paged_attention_workspace.argtypes = [_vp, _vp, _u32, C.POINTER(_sz)]
        lib.quintrit_b200_paged_attention_device.argtypes = [_vp, _u32, _vp, _vp, _vp]
        _bound = lib
    return _bound


_dtypes = {}
_torch_stream = None


def _torch():
    """torch, asked for on first use: the rest of the package works without it."""
    global _torch_stream
    import torch

    _dtypes.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    _torch_stream = raw if raw is not None else lambda device: torch.cuda.current_stream(device).cuda_stream
    return torch


def _type_of(t) -> int:
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
        torch = _torch()
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
        if table.shape[1] == 0:
            raise ValueError("a row of the table has one page at least")
        # (the rows of a table may lie further apart than they are long: what lies between is not looked at)
        self._c = _RowsC(C.sizeof(_RowsC), n, tokens, max_new, max_length, table.stride(0) if n > 1 else table.shape[1], starts.data_ptr(), lengths.data_ptr(), table.data_ptr(),
                         table.shape[1])
        self._p = C.addressof(self._c)
        self.device = starts.device
        self._device = starts.get_device()


class PagedCache:
    """``pages`` pages of ``page_tokens`` positions in each of ``layers`` layers, keys and values of ``kv_heads`` heads of ``head_dim`` values, stored as
    ``dtype`` "f16", "bf16" or "q8" (8-bit codes and a 32-bit scale per position and head)."""

    def __init__(self, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, dtype: str = "f16", device: int = 0):
        self._h = _vp()
        if dtype not in _CACHE_TYPES:
            raise ValueError(f"a paged cache is stored as {', '.join(_CACHE_TYPES)}, got {dtype!r}")
        self._lib = _lib()
        self._torch_device = _torch().device("cuda", device)
        _api._check(self._lib.quintrit_b200_paged_cache_create(device, layers, pages, page_tokens, kv_heads, head_dim, _CACHE_TYPES[dtype], C.byref(self._h)))
        self.layers, self.pages, self.page_tokens, self.kv_heads, self.head_dim, self.dtype, self.device = layers, pages, page_tokens, kv_heads, head_dim, dtype, device

    @property
    def device_bytes(self) -> int:
        n = _sz(0)
        _api._check(self._lib.quintrit_b200_paged_cache_info(self._h, C.byref(n), None))
        return n.value

    def _heads(self, name, t, tokens, heads):
        """Checks [tokens][heads][head_dim] (heads None: any number) on this device; returns (type, heads, token stride, head stride)."""
        shape, strides, kind = t.shape, t.stride(), _dtypes.get(t.dtype)
        if len(shape) != 3 or shape[0] != tokens or shape[2] != self.head_dim or (heads is not None and shape[1] != heads) or strides[2] != 1:
            raise ValueError(f"{name} is [{tokens}][{'heads' if heads is None else heads}][{self.head_dim}] with the values of a head side by side, got {tuple(shape)}, strides {strides}")
        if t.get_device() != self.device:
            raise ValueError(f"{name} is not on the cache's device {self.device}")
        if kind is None:
            raise ValueError(f"{name} is float32, float16 or bfloat16, got {t.dtype}")
        return kind, shape[1], strides[0], strides[1]

    def _empty(self, shape, dtype, stream):
        """A new tensor that belongs to the stream that the call runs on: torch's allocator hands memory out, and takes it back, in the order of one stream."""
        torch = _torch()
        if stream is None or stream == _torch_stream(self.device):
            return torch.empty(shape, dtype=dtype, device=self._torch_device)
        own = torch.cuda.ExternalStream(stream, self._torch_device) if stream else torch.cuda.default_stream(self._torch_device)
        with torch.cuda.stream(own):
            return torch.empty(shape, dtype=dtype, device=self._torch_device)

    def _call(self, rc):
        if rc != 0:
            _api._check(rc)

    def _rows(self, rows):
        if rows._device != self.device:
            raise ValueError(f"the rows' tensors are not on the cache's device {self.device}")
        return rows._p

    def append(self, layer: int, rows: PagedRows, q, k, v, *, q_out=None, q_norm=None, k_norm=None, eps: float = 1e-6, cos_sin=None, neox: bool = False, stream=None):
        """Normalises and rotates the new tokens' query and key heads, writes keys and values to the cache and returns the queries (``q_out``, by default new
        and of the queries' type; None if ``q`` is None). ``q_norm`` / ``k_norm``: float32 weights [head_dim]; ``cos_sin``: float32 [positions][rotated values]
        with cos at 2 i and sin at 2 i + 1; ``neox``: pairs (i, i + half) instead of (2 i, 2 i + 1)."""
        at, n = self._rows(rows), rows.tokens
        kind, _, k_token, k_head = self._heads("k", k, n, self.kv_heads)
        v_kind, _, v_token, v_head = self._heads("v", v, n, self.kv_heads)
        q_heads = q_token = q_head = o_token = o_head = q_at = o_at = o_kind = 0
        q_kind = kind
        if q is not None:
            q_kind, q_heads, q_token, q_head = self._heads("q", q, n, None)
            if q_out is None:
                q_out = q.new_empty(q.shape) if stream is None else self._empty(q.shape, q.dtype, stream)
            o_kind, _, o_token, o_head = self._heads("q_out", q_out, n, q_heads)
            q_at, o_at = q.data_ptr(), q_out.data_ptr()
        else:
            q_out = None
        if not kind == v_kind == q_kind:
            raise ValueError("q, k and v have the same type")
        wq = wk = cs = positions = rope = 0
        for w in (q_norm, k_norm):
            if w is not None and (_dtypes.get(w.dtype) != F32 or w.shape != (self.head_dim,) or not w.is_contiguous() or w.get_device() != self.device):
                raise ValueError(f"norm weights are float32 [{self.head_dim}] on the cache's device")
        if q_norm is not None:
            wq = q_norm.data_ptr()
        if k_norm is not None:
            wk = k_norm.data_ptr()
        if cos_sin is not None:
            if _dtypes.get(cos_sin.dtype) != F32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.get_device() != self.device:
                raise ValueError("cos_sin is a contiguous float32 [positions][rotated values] on the cache's device")
            cs, (positions, rope) = cos_sin.data_ptr(), cos_sin.shape
        a = _APPEND.pack(_APPEND.size, kind, o_kind, q_heads, q_at, k.data_ptr(), v.data_ptr(), q_token, q_head, k_token, k_head, v_token, v_head, o_at, o_token, o_head, wq, wk, eps, cs,
                         positions, rope, neox)
        self._call(self._lib.quintrit_b200_paged_append_device(self._h, layer, at, a, _torch_stream(self.device) if stream is None else stream))
        return q_out

    def read(self, layer: int, rows: PagedRows, *, k_out=None, v_out=None, dtype=None, stream=None):
        """The new tokens' rows of the cache, dense: (keys, values), each [tokens][kv_heads][head_dim]. With whole sequences as "new" tokens: all that is cached.
        ``dtype``: of the results where they are not given (default float16)."""
        at, n = self._rows(rows), rows.tokens
        if k_out is None and v_out is None:
            k_out, v_out = (self._empty((n, self.kv_heads, self.head_dim), dtype or _torch().float16, stream) for _ in range(2))
        kind = None
        for t in (k_out, v_out):
            if t is not None:
                t_kind = self._heads("an output", t, n, self.kv_heads)[0]
                if not t.is_contiguous() or (kind is not None and t_kind != kind):
                    raise ValueError("outputs are contiguous and of one type")
                kind = t_kind
        self._call(self._lib.quintrit_b200_paged_read_device(self._h, layer, at, kind, None if k_out is None else k_out.data_ptr(), None if v_out is None else v_out.data_ptr(),
                                                             _torch_stream(self.device) if stream is None else stream))
        return k_out, v_out

    def attend_workspace(self, rows: PagedRows, q_heads: int):
        """Scratch memory for ``attend`` on these rows with that many query heads (a uint8 tensor, perhaps empty). Calls that may overlap need one each."""
        torch, n = _torch(), _sz(0)
        _api._check(self._lib.quintrit_b200_paged_attention_workspace(self._h, self._rows(rows), q_heads, C.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=rows.device)

    def attend(self, layer: int, rows: PagedRows, q, *, out=None, scale: float | None = None, cap: float = 0.0, window: int = 0, workspace=None, stream=None):
        """Attention of the new tokens' queries [tokens][query heads][head_dim] over the cached positions up to their own (the last ``window`` of them, if that
        is not 0), scores times ``scale`` (default head_dim ** -0.5), capped to ``cap`` tanh(score / ``cap``) if that is not 0. Returns ``out`` (by default
        new, of the queries' type). ``workspace``: from ``attend_workspace``, by default allocated by torch for this call on its current stream (a call
        on another ``stream`` brings its own)."""
        at, n = self._rows(rows), rows.tokens
        kind, heads, q_token, q_head = self._heads("q", q, n, None)
        if out is None:
            out = q.new_empty(q.shape) if stream is None else self._empty(q.shape, q.dtype, stream)
        o_kind, _, o_token, o_head = self._heads("out", out, n, heads)
        if not 0 <= window < 2 ** 31:
            raise ValueError(f"window is 0 (none) or the number of visible positions, got {window}")
        if workspace is None:
            workspace = self.attend_workspace(rows, heads)
            if stream is not None and stream != _torch_stream(self.device) and workspace.nbytes:  # torch would hand it out again while the call still runs there
                raise ValueError("a call on another stream than torch's current one brings its workspace")
        elif workspace.get_device() != self.device or not workspace.is_contiguous():
            raise ValueError("the workspace is a contiguous tensor on the cache's device")
        a = _ATTENTION.pack(_ATTENTION.size, kind, o_kind, heads, q.data_ptr(), q_token, q_head, out.data_ptr(), o_token, o_head, self.head_dim ** -0.5 if scale is None else scale, cap,
                            window, workspace.data_ptr(), workspace.nbytes)
        self._call(self._lib.quintrit_b200_paged_attention_device(self._h, layer, at, a, _torch_stream(self.device) if stream is None else stream))
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
