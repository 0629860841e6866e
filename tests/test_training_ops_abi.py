"""The training operators' entry points on CPU: argument checks that need no
device answer with an error status before any CUDA call."""

import ctypes as C

import numpy as np
import pytest

import emeans_b200 as eb


def test_null_arguments_are_refused():
    lib = eb.load()
    out = C.c_void_p()
    for rc in (lib.eb_layer_norm(None, None, 1, 1, 0, None, None, 1e-5, None, 0, None, None),
               lib.eb_layer_norm_backward(None, None, 0, None, 0, 1, 1, None, None, None, None, 0,
                                          None, None),
               lib.eb_linear_ce(None, None, 1, 1, 0, None, 1, 0, None, 1.0, None, None),
               lib.eb_linear_ce_backward(None, None, 1, 1, 0, None, 1, 0, None, 1.0, None, None,
                                         None, 0, None, 0),
               lib.eb_adamw_create(None, None, 0, C.byref(out)),
               lib.eb_adamw_step(None, None, 1e-3, 1, 0.9, 0.999, 1e-8, 1.0),
               lib.eb_engine_create_on(0, None, None)):
        assert rc == eb.INVALID_ARGUMENT
        assert b"null" in lib.eb_last_error()
    assert lib.eb_adamw_destroy(None, None) == eb.OK


def test_host_types_of_the_buffer_types():
    """What a read returns and a write takes for each buffer type: the types
    numpy lacks travel as bits of the same size."""
    sizes = {eb.F32: 4, eb.U32: 4, eb.BF16: 2, eb.F16: 2, eb.F8: 1}
    assert {k: np.dtype(v).itemsize for k, v in eb._HOST.items()} == sizes


def test_view_of_another_element_size_is_refused():
    class FakeBuffer:
        ptr = 4096
        dtype = eb.BF16

        def __len__(self):
            return 64

    with pytest.raises(eb.EngineError) as err:
        eb.Engine.view(None, FakeBuffer(), 0, 8, eb.F32)
    assert err.value.code == eb.INVALID_ARGUMENT
