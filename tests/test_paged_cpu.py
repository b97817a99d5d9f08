"""What the paged cache's entry points refuse, without a GPU: a refused call looks at its arguments only, so a handle that owns no memory will do."""
import ctypes as C
import time

import pytest

import quintrit_b200 as q
from quintrit_b200 import paged
from quintrit_b200.paged import BF16, F16, F32, Q8, _AppendC, _AttentionC, _RowsC

NULL, ARG, SHAPE, SMALL, UNSUPPORTED, HANDLE, DEVICE = 1, 2, 3, 4, 6, 14, 15


class _Handle(C.Structure):
    _fields_ = [("magic", C.c_uint32), ("device", C.c_int), ("sm_count", C.c_int), ("layers", C.c_uint32), ("pages", C.c_uint32), ("page_tokens", C.c_uint32), ("kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("type", C.c_int32), ("pointers", C.c_void_p * 5), ("sizes", C.c_size_t * 3)]


def handle(cache_type=F16, layers=2, kv_heads=2, head_dim=64):
    return _Handle(0x51545047, 0, 148, layers, 8, 16, kv_heads, head_dim, cache_type)


def rows(**more):
    r = _RowsC(C.sizeof(_RowsC), 2, 6, 4, 100, 8, 0x1000, 0x2000, 0x3000)
    for k, v in more.items():
        setattr(r, k, v)
    return r


def append(**more):
    a = _AppendC(C.sizeof(_AppendC), F16, F16, 4, 0x10000, 0x20000, 0x30000, 256, 64, 128, 64, 128, 64, 0x40000, 256, 64)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def attention(**more):
    a = _AttentionC(C.sizeof(_AttentionC), F16, F16, 4, 0x10000, 256, 64, 0x20000, 256, 64, 0.125, 0.0, 0, None, 0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def call(name, *args):
    lib = paged._lib()
    rc = getattr(lib, "quintrit_b200_paged_" + name)(*[C.addressof(a) if isinstance(a, C.Structure) else a for a in args])
    assert rc == lib.quintrit_last_error_code() and (rc == 0) == (lib.quintrit_last_error_message() == b"")
    return rc


@pytest.mark.parametrize("args,code", [((0, 1, 16, 1, 64, F16), SHAPE), ((1, 0, 16, 1, 64, F16), SHAPE), ((1, 1, 8, 1, 64, F16), SHAPE), ((1, 1, 48, 1, 64, F16), SHAPE),
                                       ((1, 1, 512, 1, 64, F16), SHAPE), ((1, 1, 16, 0, 64, F16), SHAPE), ((1, 1, 16, 1, 96, F16), UNSUPPORTED), ((1, 1, 16, 1, 0, F16), UNSUPPORTED),
                                       ((1, 1, 16, 1, 64, F32), ARG), ((1, 1, 16, 1, 64, 4), ARG), ((1, 1 << 25, 16, 1, 64, F16), SHAPE)])
def test_create_refuses(args, code):
    h = C.c_void_p(123)
    assert call("cache_create", 0, *args, C.byref(h)) == code
    assert h.value is None


def test_create_without_an_out_pointer_and_handles():
    assert call("cache_create", 0, 1, 1, 16, 1, 64, F16, None) == NULL
    assert call("cache_free", None) == 0
    junk = handle()
    junk.magic = 5
    for h in (None, junk):
        p = None if h is None else C.addressof(h)
        assert call("cache_info", p, None, None) == HANDLE
        assert call("cache_status", p) == HANDLE
        assert call("append_device", p, 0, rows(), append(), None) == HANDLE
        assert call("attention_device", p, 0, rows(), attention(), None) == HANDLE
        assert call("read_device", p, 0, rows(), F16, 0x10000, 0x20000, None) == HANDLE
    assert call("cache_free", C.addressof(junk)) == HANDLE


BAD_ROWS = [(dict(struct_size=8), ARG), (dict(sequences=0), ARG), (dict(sequences=65536), ARG), (dict(tokens=(1 << 24) + 1), ARG), (dict(max_new=0), ARG), (dict(max_new=7), ARG),
            (dict(table_stride=0), ARG), (dict(d_starts=None), NULL), (dict(d_lengths=None), NULL), (dict(d_table=None), NULL), (dict(d_table=0x3002), ARG), (dict(max_length=0xffffffff), ARG)]


@pytest.mark.parametrize("more,code", BAD_ROWS)
def test_row_sets_that_are_refused(more, code):
    h = handle()
    assert call("append_device", h, 0, rows(**more), append(), None) == code
    assert call("attention_device", h, 0, rows(**more), attention(), None) == code
    assert call("read_device", h, 0, rows(**more), F16, 0x10000, 0x20000, None) == code
    n = C.c_size_t(5)
    want = 0 if any(k.startswith("d_") for k in more) else code
    assert call("attention_workspace", h, rows(**more), 4, C.byref(n)) == want
    assert want == 0 or n.value == 0


def test_missing_arguments_and_layers():
    h = handle()
    assert call("append_device", h, 0, None, append(), None) == NULL
    assert call("append_device", h, 0, rows(), None, None) == NULL
    assert call("attention_device", h, 0, rows(), None, None) == NULL
    assert call("attention_workspace", h, rows(), 4, None) == NULL
    for name, args in (("append_device", (append(), None)), ("attention_device", (attention(), None)), ("read_device", (F16, 0x10000, 0x20000, None))):
        assert call(name, h, 2, rows(), *args) == ARG


@pytest.mark.parametrize("more,code", [(dict(struct_size=16), ARG), (dict(type=Q8), ARG), (dict(q_out_type=Q8), ARG), (dict(q_out_type=-1), ARG), (dict(q_heads=0), SHAPE), (dict(d_k=None), NULL),
                                       (dict(d_v=None), NULL), (dict(d_q_out=None), NULL), (dict(d_q=0x10008), ARG), (dict(d_k=0x20004), ARG), (dict(d_v=0x30002), ARG),
                                       (dict(q_token_stride=255), ARG), (dict(k_head_stride=60), ARG), (dict(v_token_stride=4), ARG), (dict(out_head_stride=1), ARG),
                                       (dict(d_q_norm=0x50004, norm_eps=1e-5), ARG), (dict(d_k_norm=0x50000, norm_eps=-1.0), ARG), (dict(d_k_norm=0x50000, norm_eps=float("nan")), ARG),
                                       (dict(d_cos_sin=0x60000, positions=10, rope_dims=0), ARG), (dict(d_cos_sin=0x60000, positions=10, rope_dims=33), ARG),
                                       (dict(d_cos_sin=0x60000, positions=10, rope_dims=66), ARG), (dict(d_cos_sin=0x60000, positions=0, rope_dims=64), ARG),
                                       (dict(d_q_out=0x10000, q_out_type=BF16), ARG), (dict(d_q_out=0x10000, out_token_stride=512), ARG)])
def test_append_refuses(more, code):
    assert call("append_device", handle(), 0, rows(), append(**more), None) == code


@pytest.mark.parametrize("more,code", [(dict(struct_size=16), ARG), (dict(q_type=BF16), ARG), (dict(q_type=Q8), ARG), (dict(out_type=Q8), ARG), (dict(q_heads=0), SHAPE), (dict(q_heads=3), SHAPE),
                                       (dict(d_q=None), NULL), (dict(d_out=None), NULL), (dict(d_q=0x10004), ARG), (dict(q_head_stride=65), ARG), (dict(out_token_stride=3), ARG),
                                       (dict(scale=float("inf")), ARG), (dict(cap=-1.0), ARG), (dict(cap=float("nan")), ARG), (dict(window=1 << 31), ARG)])
def test_attention_refuses(more, code):
    assert call("attention_device", handle(), 0, rows(), attention(**more), None) == code


def test_attention_needs_its_workspace():
    h, r, n = handle(), rows(max_length=100000), C.c_size_t(0)
    assert call("attention_workspace", h, r, 4, C.byref(n)) == 0 and n.value > 0 and n.value % 16 == 0
    assert call("attention_workspace", h, r, 3, C.byref(C.c_size_t(0))) == SHAPE
    assert call("attention_device", h, 0, r, attention(), None) == NULL
    assert call("attention_device", h, 0, r, attention(d_workspace=0x100000, workspace_bytes=64), None) == SMALL
    assert call("attention_device", h, 0, r, attention(d_workspace=0x100004, workspace_bytes=n.value), None) == ARG


def test_read_refuses():
    h = handle()
    assert call("read_device", h, 0, rows(), Q8, 0x10000, 0x20000, None) == ARG
    assert call("read_device", h, 0, rows(), F16, None, None, None) == NULL
    assert call("read_device", h, 0, rows(), F16, 0x10004, None, None) == ARG
    assert call("read_device", h, 0, rows(), F32, None, 0x20008, None) == ARG


def test_calls_without_tokens_do_nothing():
    h, r = handle(), rows(tokens=0, max_new=0)
    assert call("append_device", h, 0, r, append(d_k=None), None) == 0
    assert call("attention_device", h, 0, r, attention(d_q=None), None) == 0
    assert call("read_device", h, 0, r, F16, None, None, None) == 0


def test_no_cache_type_of_another_name():
    with pytest.raises(ValueError):
        paged.PagedCache(1, 1, 16, 1, 64, "f32")


def test_paged_batches_refuse_what_is_no_batch():
    lib = q.load_library()
    out = C.c_void_p(5)
    assert lib.quintrit_b200_batch_create_paged(None, 1, 1, 16, F16, None) == NULL
    assert lib.quintrit_b200_batch_create_paged(None, 1, 1, 16, F16, C.byref(out)) == HANDLE and not out.value
    assert lib.quintrit_b200_batch_pages(None, None, None, None) == HANDLE
    assert lib.quintrit_b200_batch_read_cache(None, 0, 0, None, 0, None, 0) == HANDLE


def test_tables_with_room_between_their_rows():
    """table_pages came later than the rest: a caller without it is served as before."""
    h, n = handle(), C.c_size_t(0)
    for more, code in ((dict(table_pages=9), ARG), (dict(table_pages=8), 0), (dict(table_pages=1), 0), (dict(struct_size=_RowsC.table_pages.offset, table_pages=9), 0),
                       (dict(struct_size=_RowsC.table_pages.offset - 1), ARG)):
        assert call("attention_workspace", h, rows(**more), 4, C.byref(n)) == code


@pytest.mark.parametrize("head_dim,kv_heads,q_heads,new,sequences", [(64, 1, 4, 60, 1), (128, 4, 32, 257, 2), (256, 4, 12, 200, 1)])
def test_a_call_is_planned_in_no_time_whatever_length_is_announced(head_dim, kv_heads, q_heads, new, sequences):
    h, n = handle(head_dim=head_dim, kv_heads=kv_heads), C.c_size_t(0)
    r = rows(sequences=sequences, tokens=new + sequences - 1, max_new=new, max_length=0x7fff0000, table_stride=1 << 23)
    t = time.perf_counter()
    for _ in range(20):
        assert call("attention_workspace", h, r, q_heads, C.byref(n)) == 0 and n.value > 0
    assert time.perf_counter() - t < 0.5


def test_more_rows_than_can_be_counted_are_refused():
    h = handle(kv_heads=1)
    for tokens, q_heads in ((1 << 24, 128), ((1 << 24) - 1, 128), (1 << 15, 65536)):
        assert call("attention_device", h, 0, rows(tokens=tokens, max_new=tokens), attention(q_heads=q_heads, q_token_stride=64 * q_heads, out_token_stride=64 * q_heads), None) == SHAPE
