"""The C entries of the paged KV cache and of adjusted logits refuse what they cannot take before anything is launched."""
import ctypes as C

import pytest

BAD_ARG, BAD_SHAPE, UNSUPPORTED = 1, 4, 9
AT = 1 << 24


class Pages(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("pages", "n_kv_heads", "page_size", "head_dim", "dtype")] + [("k", C.c_void_p), ("v", C.c_void_p)]


class Table(C.Structure):
    _fields_ = [("entries", C.c_void_p), ("sequences", C.c_int32), ("width", C.c_int32), ("stride", C.c_int64)]


class Rows(C.Structure):
    _fields_ = [("at", C.c_void_p), ("token_stride", C.c_int64), ("head_stride", C.c_int64)]


class Adjust(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("dtype", "biases", "masks")] + [("width", C.c_int64)]
    _fields_ += [(n, C.c_void_p) for n in ("logits", "out", "next")]
    _fields_ += [(n, C.c_int64) for n in ("logits_stride", "out_stride", "tokens_stride", "bias_ids_stride", "bias_stride", "mask_stride")]
    _fields_ += [(n, C.c_void_p) for n in ("tokens", "length", "prompt", "repetition", "presence", "frequency", "bias_ids", "bias", "mask", "mask_rows")]


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real: only where nothing can be launched")
    from cherryq_b200 import _cabi
    L = _cabi.lib()
    L.cq_pages_attend_workspace_bytes.restype = C.c_size_t
    return L


def pages(**o):
    return Pages(**{**dict(pages=7, n_kv_heads=2, page_size=16, head_dim=128, dtype=0, k=1 << 26, v=1 << 27), **o})


def table(**o):
    return Table(**{**dict(entries=AT, sequences=3, width=5, stride=5), **o})


def rows(**o):
    return Rows(**{**dict(at=AT, token_stride=512, head_stride=128), **o})


def ref(x):
    return None if x is None else C.byref(x)


def write(lib, p=None, t=None, q=rows(), q_out=AT, k=rows(), v=rows(), cos=None, sin=None, pos=None, table_rows=0, first=AT, starts=None, n=6, heads=4):
    return lib.cq_pages_write(ref(p or pages()), ref(t or table()), ref(q), C.c_void_p(q_out), ref(k), ref(v), C.c_void_p(cos), C.c_void_p(sin),
                              C.c_void_p(pos), table_rows, C.c_void_p(first), C.c_void_p(starts), n, heads, None)


def read(lib, p=None, t=None, first=AT, count=4, k=AT, v=AT):
    return lib.cq_pages_read(ref(p or pages()), ref(t or table()), C.c_void_p(first), count, C.c_void_p(k), C.c_void_p(v), None)


def attend(lib, p=None, t=None, q=rows(), length=AT, out=AT, heads=4, window=0, sinks=0, scale=1.0, ws=AT):
    return lib.cq_pages_attend(ref(p or pages()), ref(t or table()), ref(q), C.c_void_p(length), C.c_void_p(out), heads, window, sinks, C.c_float(scale),
                               C.c_void_p(ws), None)


def step(lib, p=None, t=None, q=rows(), k=rows(), v=rows(), cos=None, sin=None, pos=None, table_rows=0, length=AT, out=AT, heads=4, window=0, sinks=0,
         scale=1.0, ws=AT):
    return lib.cq_pages_step(ref(p or pages()), ref(t or table()), ref(q), ref(k), ref(v), C.c_void_p(cos), C.c_void_p(sin), C.c_void_p(pos), table_rows,
                             C.c_void_p(length), C.c_void_p(out), heads, window, sinks, C.c_float(scale), C.c_void_p(ws), None)


@pytest.mark.parametrize("field,value,code", [
    ("pages", 0, BAD_SHAPE), ("pages", -1, BAD_SHAPE), ("n_kv_heads", 0, BAD_SHAPE), ("n_kv_heads", 16384, BAD_SHAPE), ("page_size", 8, BAD_SHAPE),
    ("page_size", 48, BAD_SHAPE), ("page_size", 512, BAD_SHAPE), ("head_dim", 96, UNSUPPORTED), ("head_dim", 256, UNSUPPORTED), ("dtype", 1, UNSUPPORTED),
    ("k", None, BAD_ARG), ("v", None, BAD_ARG), ("k", (1 << 26) + 8, BAD_ARG), ("v", 1 << 26, BAD_ARG), ("v", (1 << 26) + 7 * 2 * 16 * 256 - 16, BAD_ARG),
])
def test_pool_fields(lib, field, value, code):
    p = pages(**{field: value})
    assert lib.cq_pages_check(C.byref(p)) == code and lib.cq_pages_check(None) == BAD_ARG
    for call in (write, read, attend, step):
        assert call(lib, p) == code
    assert lib.cq_pages_attend_workspace_bytes(C.byref(p), C.byref(table()), 4, 0, 0) == 0


def test_pools_start_on_32_bytes(lib):
    for field in ("k", "v"):
        p = pages()
        setattr(p, field, getattr(p, field) + 16)
        assert lib.cq_pages_check(C.byref(p)) == BAD_ARG
        setattr(p, field, getattr(p, field) + 16)
        assert lib.cq_pages_check(C.byref(p)) == 0


@pytest.mark.parametrize("field,value,code", [
    ("entries", None, BAD_ARG), ("entries", AT + 2, BAD_ARG), ("stride", -1, BAD_ARG), ("sequences", 0, BAD_SHAPE), ("sequences", 65536, BAD_SHAPE),
    ("width", 0, BAD_SHAPE), ("width", (1 << 26) + 1, BAD_SHAPE),
])
def test_table_fields(lib, field, value, code):
    t = table(**{field: value})
    for call in (write, read, attend, step):
        assert call(lib, None, t) == code


@pytest.mark.parametrize("bad", [dict(at=None), dict(at=AT + 8), dict(token_stride=-8), dict(head_stride=-128), dict(token_stride=4), dict(head_stride=130)])
def test_rows_fields(lib, bad):
    r = rows(**bad)
    assert attend(lib, q=r) == step(lib, q=r) == step(lib, k=r) == step(lib, v=r) == write(lib, q=r) == write(lib, k=r) == write(lib, v=r) == BAD_ARG


def test_calls(lib):
    assert lib.cq_pages_check(C.byref(pages())) == 0
    assert lib.cq_pages_check(C.byref(pages(v=(1 << 26) + 7 * 2 * 16 * 256))) == 0         # side by side is apart
    for call in (attend, step):
        for bad in (dict(q=None), dict(length=None), dict(out=None), dict(out=AT + 8), dict(ws=AT + 8), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
                    dict(scale=-1.0), dict(scale=float("nan")), dict(length=AT + 4)):
            assert call(lib, **bad) == BAD_ARG, bad
        assert call(lib, heads=0) == call(lib, heads=3) == BAD_SHAPE
        assert call(lib) not in (0, BAD_ARG, BAD_SHAPE, UNSUPPORTED)                      # (no device to launch on)
    for bad in (dict(k=None), dict(v=None), dict(cos=AT), dict(cos=AT, sin=AT, pos=AT, table_rows=0), dict(cos=AT, pos=AT, table_rows=4),
                dict(cos=AT, sin=AT, pos=AT + 4, table_rows=4), dict(cos=AT + 2, sin=AT, pos=AT, table_rows=4)):
        assert step(lib, **bad) == BAD_ARG and write(lib, **bad) == BAD_ARG, bad
    for bad in (dict(first=None), dict(first=AT + 4), dict(starts=AT + 4), dict(n=0), dict(heads=-1), dict(q=None), dict(q_out=None), dict(q_out=AT + 8)):
        assert write(lib, **bad) == BAD_ARG, bad
    assert write(lib, n=7) == BAD_SHAPE                                                    # not the same for three sequences
    for bad in (dict(first=None), dict(first=AT + 4), dict(count=0), dict(k=None), dict(v=AT + 8)):
        assert read(lib, **bad) == BAD_ARG, bad
    assert write(lib, q=None, q_out=None, heads=0) not in (0, BAD_ARG, BAD_SHAPE, UNSUPPORTED)
    # a long table is cut into ranges, whose sums need room
    t = table(width=4096)
    assert lib.cq_pages_attend_workspace_bytes(C.byref(pages()), C.byref(t), 4, 0, 0) > 0 and attend(lib, None, t, ws=None) == BAD_ARG


def adjust(**o):
    f = dict(dtype=0, logits=AT, out=AT + (1 << 20), next=AT + (2 << 20), logits_stride=1000, out_stride=1000)
    full = dict(tokens=AT, tokens_stride=9, width=9, bias_ids=AT, bias=AT, biases=3, bias_ids_stride=3, bias_stride=3, mask=AT, masks=2, mask_stride=32)
    return Adjust(**{**f, **full, **o})


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), BAD_ARG), (dict(out=None), BAD_ARG), (dict(next=None), BAD_ARG), (dict(dtype=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED),
    (dict(logits=AT + 1), BAD_ARG), (dict(dtype=1, out=AT + (1 << 20) + 2), BAD_ARG), (dict(logits_stride=-1), BAD_ARG), (dict(out_stride=999), BAD_ARG),
    (dict(width=-1), BAD_ARG), (dict(width=1 << 31), BAD_SHAPE), (dict(tokens=None, length=AT), BAD_ARG), (dict(tokens=None, repetition=AT), BAD_ARG),
    (dict(tokens_stride=-1), BAD_ARG), (dict(biases=-1), BAD_ARG), (dict(bias=None), BAD_ARG), (dict(bias_ids=None), BAD_ARG), (dict(bias_stride=-1), BAD_ARG),
    (dict(tokens=AT + 4), BAD_ARG), (dict(prompt=AT + 4), BAD_ARG), (dict(next=AT + 4), BAD_ARG), (dict(mask=AT + 2), BAD_ARG), (dict(presence=AT + 1), BAD_ARG),
    (dict(masks=1), BAD_ARG), (dict(masks=0, mask_rows=AT), BAD_ARG), (dict(mask=None, mask_rows=AT), BAD_ARG), (dict(mask_stride=-1), BAD_ARG),
    # out over logits in part, one row further, and with another stride
    (dict(out=AT + 2), BAD_ARG), (dict(out=AT + 2000), BAD_ARG), (dict(out=AT - 3998), BAD_ARG), (dict(out=AT, out_stride=1001), BAD_ARG),
])
def test_adjust_fields(lib, change, code):
    assert lib.cq_adjust_logits(C.byref(adjust(**change)), 2, 1000, None) == code


def test_adjust_calls(lib):
    assert lib.cq_adjust_logits(None, 2, 1000, None) == BAD_ARG
    for rows_, vocab in ((0, 1000), (65536, 1000), (2, 0), (2, (1 << 30) + 1)):
        assert lib.cq_adjust_logits(C.byref(adjust()), rows_, vocab, None) == BAD_SHAPE
    for fine in (dict(), dict(out=AT), dict(out=AT + 4000), dict(mask_rows=AT, masks=1), dict(tokens=None), dict(biases=0, bias=None, bias_ids=None)):
        assert lib.cq_adjust_logits(C.byref(adjust(**fine)), 2, 1000, None) not in (0, BAD_ARG, BAD_SHAPE, UNSUPPORTED)      # (no device to launch on)
