"""The C entries of the 4-bit KV cache and of prompt attention refuse what they cannot take before anything is launched."""
import ctypes as C

import pytest

BAD_ARG, BAD_SHAPE, UNSUPPORTED = 1, 4, 9


class Cache(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("sequences", "n_kv_heads", "slots", "head_dim", "group")]
    _fields_ += [(n, C.c_void_p) for n in ("k_codes", "k_scales", "v_codes", "v_scales")]


class Prompt(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("sequences", "queries", "keys", "n_heads", "n_kv_heads", "head_dim", "window", "sinks")]
    _fields_ += [(n, C.c_int64 * 3) for n in ("q_strides", "k_strides", "v_strides")] + [("scale", C.c_float)]


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real: only where nothing can be launched")
    from cherryq_b200 import _cabi
    L = _cabi.lib()
    L.cq_kv4_evict_workspace_bytes.restype = L.cq_kv4_attend_workspace_bytes.restype = C.c_size_t
    return L


def cache(**o):
    f = dict(sequences=2, n_kv_heads=2, slots=64, head_dim=128, group=32, k_codes=1 << 20, k_scales=1 << 21, v_codes=1 << 22, v_scales=1 << 23)
    f.update(o)
    return Cache(**f)


@pytest.mark.parametrize("field,value,code", [
    ("sequences", 0, BAD_SHAPE), ("sequences", 65536, BAD_SHAPE), ("n_kv_heads", 0, BAD_SHAPE), ("slots", 0, BAD_SHAPE), ("slots", 40, BAD_SHAPE),
    ("head_dim", 96, UNSUPPORTED), ("head_dim", 256, UNSUPPORTED), ("group", 128, UNSUPPORTED), ("group", 16, UNSUPPORTED),
    ("k_codes", None, BAD_ARG), ("v_scales", None, BAD_ARG), ("k_scales", (1 << 21) + 8, BAD_ARG), ("v_codes", (1 << 22) + 4, BAD_ARG),
])
def test_cache_fields(lib, field, value, code):
    c = cache(**{field: value})
    assert lib.cq_kv4_check(C.byref(c)) == code
    at = C.c_void_p(1 << 24)
    assert lib.cq_kv4_read(C.byref(c), at, 1, at, at, None) == code
    assert lib.cq_kv4_attend(C.byref(c), at, at, at, 4, 0, 0, C.c_float(1.0), None, None, at, None) == code
    assert lib.cq_kv4_evict(C.byref(c), C.byref(cache()), at, at, at, at, 8, 0, 0, at, at, None) == code
    assert lib.cq_kv4_evict_workspace_bytes(C.byref(c), 8) == 0 and lib.cq_kv4_attend_workspace_bytes(C.byref(c), 4, 0, 0, 1) == 0


def test_cache_calls(lib):
    c, at, odd = cache(), C.c_void_p(1 << 24), C.c_void_p((1 << 24) + 8)
    assert lib.cq_kv4_check(C.byref(c)) == 0 and lib.cq_kv4_check(None) == BAD_ARG
    f = C.c_float(1.0)
    attend = lambda q=at, n=at, out=at, heads=4, window=0, sinks=0, w=None, wo=None, ws=at: lib.cq_kv4_attend(
        C.byref(c), q, n, out, heads, window, sinks, f, w, wo, ws, None)
    for bad in (dict(q=None), dict(n=None), dict(out=None), dict(w=at, wo=at, ws=None), dict(window=-1), dict(sinks=-1), dict(w=at), dict(wo=at), dict(q=odd), dict(out=odd)):
        assert attend(**bad) == BAD_ARG, bad
    assert attend(heads=0) == BAD_SHAPE and attend(heads=3) == BAD_SHAPE
    write = lambda q=at, qo=at, k=at, v=at, cos=None, sin=None, pos=None, rows=0, first=at, tokens=1, heads=4: lib.cq_kv4_write(
        C.byref(c), q, qo, k, v, cos, sin, pos, rows, first, tokens, heads, None)
    for bad in (dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(first=None), dict(tokens=0), dict(heads=-1), dict(k=odd), dict(cos=at),
                dict(cos=at, sin=at, pos=at, rows=0)):
        assert write(**bad) == BAD_ARG, bad
    assert lib.cq_kv4_read(C.byref(c), at, 0, at, at, None) == BAD_ARG and lib.cq_kv4_read(C.byref(c), at, 1, odd, at, None) == BAD_ARG
    to = cache(k_codes=5 << 20, k_scales=6 << 20, v_codes=7 << 20, v_scales=9 << 20)
    evict = lambda to=to, keep=8, sinks=0, recent=0, w=at, ws=at: lib.cq_kv4_evict(C.byref(c), C.byref(to), w, at, at, at, keep, sinks, recent, at, ws, None)
    for bad in (dict(keep=0), dict(keep=65), dict(sinks=-1), dict(recent=-1), dict(w=None), dict(to=c, ws=None),
                dict(to=cache(k_scales=6 << 20)), dict(to=cache(slots=32))):
        assert evict(**bad) == BAD_ARG, bad
    for bad in (cache(sequences=1), cache(n_kv_heads=4), cache(head_dim=64), cache(group=64)):
        assert evict(to=bad) == BAD_SHAPE
    assert lib.cq_kv4_evict_workspace_bytes(C.byref(c), 8) == 2 * 2 * 8 * 2 * (64 + 16)


def prompt(**o):
    f = dict(sequences=1, queries=8, keys=16, n_heads=4, n_kv_heads=2, head_dim=64, window=0, sinks=0, scale=0.125)
    strides = o.pop("strides", (1024, 256, 64))
    f.update(o)
    s = (C.c_int64 * 3)(*strides)
    return Prompt(q_strides=s, k_strides=s, v_strides=s, **f)


@pytest.mark.parametrize("change,code", [
    (dict(sequences=0), BAD_SHAPE), (dict(queries=0), BAD_SHAPE), (dict(queries=17), BAD_SHAPE), (dict(n_heads=3), BAD_SHAPE), (dict(n_kv_heads=0), BAD_SHAPE),
    (dict(head_dim=96), UNSUPPORTED), (dict(window=-1), BAD_ARG), (dict(sinks=-1), BAD_ARG), (dict(strides=(1024, 260, 64)), BAD_ARG),
])
def test_prompt_fields(lib, change, code):
    s, at = prompt(**change), C.c_void_p(1 << 24)
    assert lib.cq_attn_prefill(C.byref(s), at, at, at, None, at, at, at, None, None) == code
    assert lib.cq_attn_prefill_weights(C.byref(s), at, at, at, None, 4, at, at, None, None) == code


def test_prompt_calls(lib):
    s, at, odd = prompt(), C.c_void_p(1 << 24), C.c_void_p((1 << 24) + 2)
    for a in ((None, at, at, None, at, at), (at, None, at, None, at, at), (at, at, None, None, at, at), (odd, at, at, None, at, at),
              (at, at, odd, None, at, at), (at, at, at, None, None, at), (at, at, at, None, at, None)):
        assert lib.cq_attn_prefill(C.byref(s), *a, at, None, None) == BAD_ARG
    for a in ((None, at, at, None, 4, at), (at, at, None, None, 4, at), (at, at, at, None, 0, at), (at, at, at, None, 4, None)):
        assert lib.cq_attn_prefill_weights(C.byref(s), *a, at, None, None) == BAD_ARG


def test_evict_into_memory_of_its_own(lib):
    """Another cache, and the results, must share no memory with what is read: codes of 16384 bytes, scales of 4096, weights of 1024."""
    c, at = cache(), lambda n: C.c_void_p((1 << 28) + n)

    def evict(to, w=at(0), left=at(1 << 16), n=at(2 << 16), now=at(3 << 16), kept=at(4 << 16)):
        return lib.cq_kv4_evict(C.byref(c), C.byref(to), w, left, n, now, 8, 0, 0, kept, at(5 << 16), None)
    apart = dict(k_codes=5 << 20, k_scales=6 << 20, v_codes=7 << 20, v_scales=9 << 20)
    for field, address in (("k_codes", (1 << 20) + 16384 - 16), ("k_codes", (1 << 20) - 16384 + 16), ("v_codes", (1 << 20) + 64), ("k_scales", (1 << 22) + 16),
                           ("v_scales", (1 << 23) + 4096 - 16), ("v_scales", (1 << 21) - 4096 + 16)):
        assert evict(cache(**{**apart, field: address})) == BAD_ARG, (field, hex(address))
    to = cache(**apart)
    for bad in (dict(left=at(0)), dict(left=at(1020)), dict(left=at(-124)), dict(now=at(2 << 16)), dict(now=at((2 << 16) + 8)), dict(now=at((2 << 16) - 8)),
                dict(kept=at(0)), dict(kept=at(2 << 16))):
        assert evict(to, **bad) == BAD_ARG, bad
    # side by side is apart, and in place is in place
    for fine in (cache(**{**apart, "k_codes": (1 << 20) + 16384}), cache(**{**apart, "v_scales": (1 << 21) - 4096}), c):
        assert evict(fine, left=at(1024)) not in (0, BAD_ARG, BAD_SHAPE, UNSUPPORTED)      # (no device to launch on)


def test_weights_over_themselves_or_apart(lib):
    """weights_out is weights or shares no memory with it (1024 bytes each)."""
    c, at = cache(), C.c_void_p(1 << 24)
    for off in (16, -16, 1008, -1008):
        wo = C.c_void_p((1 << 25) + off)
        assert lib.cq_kv4_attend(C.byref(c), at, at, at, 4, 0, 0, C.c_float(1.0), C.c_void_p(1 << 25), wo, at, None) == BAD_ARG
        assert lib.cq_kv4_step(C.byref(c), at, at, at, None, None, None, 0, at, at, 4, 0, 0, C.c_float(1.0), C.c_void_p(1 << 25), wo, at, None) == BAD_ARG
    for off in (0, 1024, -1024):
        rc = lib.cq_kv4_attend(C.byref(c), at, at, at, 4, 0, 0, C.c_float(1.0), C.c_void_p(1 << 25), C.c_void_p((1 << 25) + off), at, None)
        assert rc not in (0, BAD_ARG, BAD_SHAPE, UNSUPPORTED)          # (no device to launch on)
