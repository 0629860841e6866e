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


def test_adamw_buffers_apart(engine):
    """Of one tensor and of several: no buffer is written twice, in part either,
    and no gradient lies over one that is written. Gradients may be shared."""
    n = 300
    z = engine.zeros

    def tensor(**kw):
        return eb.AdamWTensor(**{**dict(p=z(eb.F32, n), g=z(eb.F32, n), m=z(eb.F32, n),
                                        v=z(eb.F32, n)), **kw})

    at = room(engine, 2000)
    byte = room(engine, 4000, eb.F8)
    eight = dict(m=byte(0, n), v=byte(320, n), m_scale=at(0, 2), v_scale=at(4, 2))
    a = tensor(p=at(0, n))
    for ts, why in (([tensor(p=at(0, n), m=at(200, n))], "written twice"),
                    ([a, tensor(v=at(296, n))], "written twice"),
                    ([a, tensor(p=at(0, n))], "written twice"),
                    ([tensor(p=at(0, n), g=at(0, n))], "g overlaps"),
                    ([a, tensor(g=at(100, n))], "g overlaps"),
                    ([tensor(g=at(100, n)), a], "g overlaps"),
                    ([tensor(g=at(296, n)), a], "g overlaps"),
                    ([tensor(**{**eight, "v": byte(288, n)})], "written twice"),
                    ([tensor(**{**eight, "m_scale": at(4, 2)})], "written twice"),
                    ([tensor(**eight), tensor(g=at(0, n))], "g overlaps")):
        refused(lambda: eb.AdamW(engine, ts), why)
    one = z(eb.F32, n)
    plan = eb.AdamW(engine, [tensor(p=at(0, n), m=at(300, n), v=at(600, n), g=one), tensor(g=one),
                             tensor(**{**eight, "m_scale": at(1200, 2), "v_scale": at(1204, 2)})])
    plan.step(lr=1e-3, step=1)
    engine.sync()
