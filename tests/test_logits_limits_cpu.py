"""The C entry of adjusted logits refuses more entries a row than its kernel's 32-bit indices step through."""
import ctypes as C

import pytest

from test_pages_cpu import BAD_SHAPE, UNSUPPORTED, BAD_ARG, adjust, lib  # noqa: F401


@pytest.mark.parametrize("change", [dict(biases=1 << 30), dict(biases=2 ** 31 - 1), dict(width=1 << 30), dict(width=2 ** 40)])
def test_more_than_indices_hold(lib, change):  # noqa: F811
    assert lib.cq_adjust_logits(C.byref(adjust(**change)), 2, 1000, None) == BAD_SHAPE


@pytest.mark.parametrize("change", [dict(biases=(1 << 30) - 1), dict(width=(1 << 30) - 1)])
def test_as_many_as_they_hold(lib, change):  # noqa: F811
    assert lib.cq_adjust_logits(C.byref(adjust(**change)), 2, 1000, None) not in (0, BAD_ARG, BAD_SHAPE, UNSUPPORTED)      # (no device to launch on)
