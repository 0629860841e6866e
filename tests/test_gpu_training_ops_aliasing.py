"""The training operators refuse outputs that share memory with one another or
with their inputs, in part or whole (nothing is launched), and still take what
may be shared: y over x, dx over dy, and buffers that touch end to end."""

import pytest

import emeans_b200 as eb
from tests.test_gpu_training_ops import refused

pytestmark = pytest.mark.gpu

ROWS, D = 8, 16  # 128 elements


def room(eng, n=512, dtype=eb.F32):
    """A buffer and views of it."""
    b = eng.zeros(dtype, n)
    return lambda at, length: eng.view(b, at, length, dtype)


def test_layer_norm_outputs_apart(engine):
    at = room(engine)
    z = engine.zeros_f32
    x, y, s, w, b, mean, rstd = at(0, 128), z(128), at(128, 16), at(144, 16), z(16), z(8), z(8)
    ok = dict(x=x, rows=ROWS, d=D, weight=w, bias=b, y=y, mean=mean, rstd=rstd)

    def call(**kw):
        return lambda: engine.layer_norm(**{**ok, **kw})

    for kw in (dict(mean=at(120, 8)), dict(rstd=at(0, 8)), dict(mean=at(148, 8)),
               dict(rstd=engine.view(b, 8, 8, eb.F32)), dict(mean=engine.view(y, 4, 8, eb.F32)),
               dict(mean=mean, rstd=mean), dict(y=at(132, 128)),
               dict(mean=s, rstd=at(132, 8))):
        refused(call(**kw), "overlaps")
    call()()
    call(y=x)()                     # in place
    call(mean=at(128, 8), rstd=at(136, 8))()  # end to end with x, w and each other
    engine.sync()


def test_layer_norm_backward_outputs_apart(engine):
    at = room(engine)
    z = engine.zeros_f32
    x, dy, dx, w, mean, rstd = at(0, 128), at(128, 128), z(128), at(256, 16), z(8), z(8)
    ok = dict(dy=dy, x=x, rows=ROWS, d=D, weight=w, mean=mean, rstd=rstd, dx=dx, dweight=z(16),
              dbias=z(16))

    def call(**kw):
        return lambda: engine.layer_norm_backward(**{**ok, **kw})

    for kw in (dict(dweight=at(4, 16)), dict(dbias=at(240, 16)), dict(dweight=w),
               dict(dbias=at(260, 16)), dict(dweight=ok["dbias"]), dict(dbias=engine.view(dx, 100, 28, eb.F32)),
               dict(dweight=engine.view(ok["dbias"], 4, 12, eb.F32), d=12, rows=1),
               dict(dx=at(260, 128)), dict(mean=engine.view(dx, 8, 8, eb.F32)),
               dict(dx=at(136, 128)), dict(dweight=rstd, d=8, rows=8)):
        refused(call(**kw), "overlaps")
    call()()
    call(dx=dy)()                   # in place
    call(dweight=at(272, 16), dbias=at(288, 16))()
    engine.sync()
