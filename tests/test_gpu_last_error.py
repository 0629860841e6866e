"""The last failed call's message lasts until the next call that is not a
release: the binding's garbage collector may release objects in between."""

import ctypes as C

import pytest

import emeans_b200 as eb

pytestmark = pytest.mark.gpu


def test_releases_keep_the_last_errors_message(engine):
    lib = eb.load()
    other = eb.Engine(0)
    buf, plan = engine.zeros_f32(8), eb.AdamW(engine, [])
    out = C.c_void_p()
    assert lib.eb_buf_alloc(engine.h, 99, 4, C.byref(out)) == eb.INVALID_ARGUMENT
    assert lib.eb_last_error() == b"unknown dtype"
    buf.free()
    plan.free()
    other.close()
    assert lib.eb_last_error() == b"unknown dtype"
    engine.sync()
    assert lib.eb_last_error() == b""
