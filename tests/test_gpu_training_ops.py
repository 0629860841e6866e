"""The training operators on the B200 against plain 64-bit formulas.

Layer norm, the linear cross entropy and AdamW, each over types, sizes from
one element up, odd sizes, row strides and the inputs where it can go wrong.
Tolerances are elementwise bounds of the rounding that the operators are
allowed (FP32 sums, one rounding of the output, and the stated rounding of P),
computed in 64 bits from the inputs.
"""

import math

import numpy as np
import pytest
import torch

import emeans_b200 as eb

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24  # half an ulp of f32 at 1 (24 significant bits; bf16 has 8, f16 11)
HALF_ULP = {torch.float32: U32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = {torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}


@pytest.fixture(scope="module")
def eng():
    e = eb.Engine(0, stream=torch.cuda.current_stream().cuda_stream)
    yield e
    e.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def strided(x, ld, fill=math.nan):
    """x (rows x d) in a flat tensor with rows `ld` apart, and the view of the rows."""
    rows, d = x.shape
    flat = torch.full((max(rows * ld, 1),), fill, device="cuda", dtype=x.dtype)
    view = flat[:rows * ld].view(rows, ld)[:, :d]
    view.copy_(x)
    return flat, view


def wrap(e, t):
    return None if t is None else e.wrap(t)


def within(got, want, tol, what):
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], tol.expand_as(want)[bad][:4])


# ---------------------------------------------------------------- layer norm

NORM_SHAPES = [(1, 1), (3, 2), (9, 5), (33, 64), (2, 768), (501, 768), (70, 387), (40, 1024),
               (19, 1027), (5, 2048), (3, 4096), (4, 4099), (3, 16384), (2, 16386), (2, 20001)]


def norm_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / ((x - mean).square().mean(1, keepdim=True) + eps).sqrt()
    u = (x - mean) * rstd
    return mean, rstd, u, u * w + b


def norm_sums(d):
    """Roundings a value meets in a sum over d elements: a thread's own
    (32, or d / 512 for the longest rows), five shuffles, 16 warps, and a few
    operations around them."""
    return max(32, math.ceil(d / 512)) + 5 + 16 + 8


@pytest.mark.parametrize("pad", [0, 3, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,d", NORM_SHAPES)
def test_layer_norm_forward(eng, rows, d, dtype, pad):
    g = gen(rows * 31 + d)
    x = (randn(g, rows, d) * 2.0 + 3.0 * randn(g, rows, 1)).to(dtype)
    wt = dtype if pad == 3 else torch.float32
    w, b = (1 + 0.2 * randn(g, d)).to(wt), randn(g, d).to(wt)
    flat, xv = strided(x, d + pad)
    yflat, yv = strided(torch.zeros_like(x), d + pad, fill=7.0)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    eng.layer_norm(wrap(eng, flat), rows, d, wrap(eng, w), wrap(eng, b), wrap(eng, yflat),
                   eps=1e-5, mean=wrap(eng, mean), rstd=wrap(eng, rstd), ldx=d + pad, ldy=d + pad)
    eng.sync()
    m, r, u, want = norm_reference(xv, w.double(), b.double(), 1e-5)
    q = norm_sums(d) * 2 * U32
    spread = xv.double().abs().amax(1, keepdim=True)
    within(mean[:, None], m, q * spread, "mean")
    # The variance is a sum of squares of deviations, each off by the mean's error.
    rel = q + 2 * q * spread * r
    within(rstd[:, None], r, r * rel, "rstd")
    tol = w.double().abs() * (u.abs() * rel + q * spread * r) + 4 * U32 * (u * w).abs()
    within(yv, want, tol + HALF_ULP[dtype] * (want.abs() + tol) + 2 * U32 * want.abs() + TINY[dtype],
           "y")
    if pad:
        gap = yflat.view(rows, d + pad)[:, d:]
        assert (gap == 7.0).all(), "elements between the rows were written"


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,d", NORM_SHAPES + [(3000, 100), (2000, 1024)])
def test_layer_norm_backward(eng, rows, d, dtype):
    g = gen(rows * 17 + d)
    pad = 8 if rows % 2 else 1
    x = (randn(g, rows, d) + randn(g, rows, 1)).to(dtype)
    dy = randn(g, rows, d).to(dtype)
    w = (1 + 0.2 * randn(g, d)).to(dtype)
    mean = x.float().mean(1)
    rstd = ((x.float() - mean[:, None]).square().mean(1) + 1e-5).rsqrt()
    xf, xv = strided(x, d + pad)
    df, dv = strided(dy, d + 2 * pad)
    of, ov = strided(torch.zeros_like(x), d, fill=0.0)
    dw, db = torch.empty(d, device="cuda"), torch.empty(d, device="cuda", dtype=dtype)
    eng.layer_norm_backward(wrap(eng, df), wrap(eng, xf), rows, d, wrap(eng, w), wrap(eng, mean),
                            wrap(eng, rstd), wrap(eng, of), wrap(eng, dw), wrap(eng, db),
                            lddy=d + 2 * pad, ldx=d + pad)
    eng.sync()
    X, G, W = x.double(), dy.double(), w.double()
    M, R = mean.double()[:, None], rstd.double()[:, None]
    u, h = (X - M) * R, G * W
    want = R * (h - h.mean(1, keepdim=True) - u * (h * u).mean(1, keepdim=True))
    eu = 3 * U32 * (X.abs() + M.abs()) * R  # error of u
    q = norm_sums(d) * 2 * U32
    e1 = q * h.abs().mean(1, keepdim=True)
    e2 = q * (h * u).abs().mean(1, keepdim=True) + (h.abs() * eu).mean(1, keepdim=True)
    c2 = (h * u).mean(1, keepdim=True).abs()
    tol = R * (e1 + u.abs() * e2 + eu * (c2 + e2)
               + 6 * U32 * (h.abs() + h.mean(1, keepdim=True).abs() + u.abs() * c2))
    within(ov, want, tol + HALF_ULP[dtype] * (want.abs() + tol) + TINY[dtype], "dx")
    sums = (rows + 8) * U32
    wdw, wdb = (G * u).sum(0), G.sum(0)
    within(dw, wdw, sums * (G * u).abs().sum(0) + (G.abs() * eu).sum(0) + U32 * wdw.abs(), "dweight")
    tdb = sums * G.abs().sum(0)
    within(db, wdb, tdb + HALF_ULP[dtype] * (wdb.abs() + tdb) + TINY[dtype], "dbias")


def test_layer_norm_gradient_is_the_difference_quotient(eng):
    """dx, dweight and dbias of sum(dy y) against central differences of the
    64-bit forward formula (step 1e-5: truncation 1e-10, cancellation 1e-11
    relative to values of order 1; f32 rounding of the result dominates)."""
    rows, d = 5, 12
    g = gen(4)
    x, dy, w, b = randn(g, rows, d), randn(g, rows, d), 1 + 0.3 * randn(g, d), randn(g, d)
    mean, rstd, y = (torch.empty(s, device="cuda") for s in (rows, rows, (rows, d)))
    dx, dw, db = torch.empty(rows, d, device="cuda"), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    eng.layer_norm(wrap(eng, x), rows, d, wrap(eng, w), wrap(eng, b), wrap(eng, y), eps=1e-5,
                   mean=wrap(eng, mean), rstd=wrap(eng, rstd))
    eng.layer_norm_backward(wrap(eng, dy), wrap(eng, x), rows, d, wrap(eng, w), wrap(eng, mean),
                            wrap(eng, rstd), wrap(eng, dx), wrap(eng, dw), wrap(eng, db))
    eng.sync()

    def f(x, w, b):
        return float((norm_reference(x, w, b, 1e-5)[3] * dy.double()).sum())

    X, W, B = x.double(), w.double(), b.double()
    for got, var, at in ((dx, X, 0), (dw, W, 1), (db, B, 2)):
        for i in range(var.numel()):
            args = [X, W, B]
            lo, hi = var.clone(), var.clone()
            lo.view(-1)[i] -= 1e-5
            hi.view(-1)[i] += 1e-5
            args[at] = hi
            up = f(*args)
            args[at] = lo
            want = (up - f(*args)) / 2e-5
            assert abs(float(got.view(-1)[i]) - want) <= 2e-5 * (1 + abs(want))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_layer_norm_in_place_without_weights_and_non_finite_rows(eng, dtype):
    rows, d = 6, 96
    x = randn(gen(2), rows, d).to(dtype)
    x[1, 3], x[3, 5], x[4] = math.inf, math.nan, 2.0
    want = norm_reference(x, torch.ones(d, device="cuda").double(), 0.0, 1e-5)[3]
    buf = wrap(eng, x)
    eng.layer_norm(buf, rows, d, None, None, buf)
    eng.sync()
    keep = [0, 2, 5]
    tol = 60 * U32 * 8 + HALF_ULP[dtype] * want[keep].abs()
    within(x[keep], want[keep], tol, "finite rows")
    assert x[1].isnan().all() and x[3].isnan().all()
    assert (x[4] == 0).all(), "a constant row has no spread: zeros"


def test_layer_norm_of_no_rows_zeroes_the_weight_gradients(eng):
    d = 40
    z = torch.empty(0, device="cuda")
    dw, db = torch.ones(d, device="cuda"), torch.ones(d, device="cuda")
    e = eng.zeros_f32(0)
    eng.layer_norm(e, 0, d, None, None, eng.zeros_f32(0))
    eng.layer_norm_backward(e, e, 0, d, None, e, e, None, wrap(eng, dw), wrap(eng, db))
    eng.sync()
    assert z.numel() == 0 and (dw == 0).all() and (db == 0).all()


def test_layer_norm_sums_are_the_same_bits_on_every_call(eng):
    rows, d = 5003, 192
    g = gen(9)
    x, dy = randn(g, rows, d), randn(g, rows, d)
    mean, rstd = x.mean(1), torch.ones(rows, device="cuda")
    outs = []
    for _ in range(2):
        dx, dw, db = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
        eng.layer_norm_backward(wrap(eng, dy), wrap(eng, x), rows, d, None, wrap(eng, mean),
                                wrap(eng, rstd), wrap(eng, dx), wrap(eng, dw), wrap(eng, db))
        eng.sync()
        outs.append((dx, dw, db))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ---------------------------------------------------------------- linear cross entropy

CE_SHAPES = [(1, 1, 1), (1, 2, 4), (2, 3, 5), (5, 49, 11), (1, 300, 64), (130, 257, 70),
             (128, 256, 64), (257, 513, 72), (300, 1000, 384), (64, 5000, 200), (1000, 32, 64),
             (3000, 40, 33)]


class Ce:
    """One problem, its 64-bit values and the bounds on each output."""

    def __init__(self, n, k, d, dtype, seed, scale=1.3, ignored=0.1, lean=4.0, per_row=True):
        g = gen(seed)
        self.n, self.k, self.d, self.scale, self.dtype = n, k, d, scale, dtype
        w = randn(g, k, d)
        w = w / w.norm(dim=1, keepdim=True)
        t = torch.randint(0, k, (n,), generator=g, device="cuda")
        x = randn(g, n, d) + lean * torch.rand(n, 1, generator=g, device="cuda") * w[t]
        drop = torch.rand(n, generator=g, device="cuda") < ignored
        self.x, self.w = x.to(dtype), w.to(dtype)
        self.t = torch.where(drop, torch.full_like(t, eb.IGNORE), t)
        self.dloss = randn(g, n) if per_row else torch.full((1,), 1.0 / n, device="cuda")

    def run(self, e, pad=0, dx=True, dw=True, dxt=None, dwt=None):
        n, k, d = self.n, self.k, self.d
        xf, _ = strided(self.x, d + pad)
        wf, _ = strided(self.w, d + 2 * pad)
        loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        tb = wrap(e, self.t.to(torch.uint32))
        xb, wb, lb = wrap(e, xf), wrap(e, wf), wrap(e, lse)
        e.linear_cross_entropy(xb, n, d, wb, k, tb, wrap(e, loss), lb, scale=self.scale,
                               ldx=d + pad, ldw=d + 2 * pad)
        gx = strided(torch.zeros(n, d, device="cuda", dtype=dxt or self.dtype), d + pad, 5.0) if dx else None
        gw = strided(torch.zeros(k, d, device="cuda", dtype=dwt or self.dtype), d + pad, 5.0) if dw else None
        e.linear_cross_entropy_backward(
            xb, n, d, wb, k, tb, lb, wrap(e, self.dloss), wrap(e, gx[0]) if dx else None,
            wrap(e, gw[0]) if dw else None, scale=self.scale, ldx=d + pad, ldw=d + 2 * pad,
            lddx=d + pad, lddw=d + pad)
        e.sync()
        for q in (gx, gw):
            if q is not None and pad:
                assert (q[0].view(-1, d + pad)[:, d:] == 5.0).all(), "between the rows"
        return loss, lse, gx and gx[1], gw and gw[1]

    def check(self, got):
        loss, lse, dx, dw = got
        X, W, s = self.x.double(), self.w.double(), self.scale
        live = self.t != eb.IGNORE
        t = torch.where(live, self.t, torch.zeros_like(self.t))[:, None]
        Z = s * (X @ W.T)
        L = torch.logsumexp(Z, 1)
        # A score: its products (two-term operands drop 3 2^-22 of them and
        # keep 2^-38 of the largest element), FP32 sums cut at every step.
        two = self.dtype == torch.float32
        cross = X.abs() @ W.abs().T
        ez = s * ((self.d / 4 + 8) * 2.0 ** -23 * cross)
        if two:
            ez = ez + s * 3 * 2.0 ** -22 * cross + s * 2.0 ** -38 * (
                float(X.abs().max()) * W.abs().sum(1)[None, :] + float(W.abs().max()) * X.abs().sum(1)[:, None])
        el = ez.amax(1) + 2.0 ** -20 + 6 * 2.0 ** -23 * (L.abs() + Z.abs().amax(1))
        within(lse, L, el, "lse")
        zt = Z.gather(1, t)[:, 0]
        want = torch.where(live, L - zt, torch.zeros_like(L))
        within(loss, want, torch.where(live, el + ez.gather(1, t)[:, 0] + 4 * 2.0 ** -23 * zt.abs(),
                                       torch.zeros_like(L)), "loss")
        g = torch.where(live, self.dloss.double().expand(self.n), torch.zeros_like(L)) * s
        p = torch.exp(Z - L[:, None])
        hot = torch.zeros_like(p).scatter_(1, t, 1.0)
        P = g[:, None] * (p - hot)
        gm = float(self.dloss.abs().max()) * s
        keep = {torch.float32: 2.0 ** -21, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}[self.dtype]
        least = {torch.float32: 2.0 ** -37, torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -37}[self.dtype]
        eP = g[:, None].abs() * p * (ez + 2 * el[:, None] + 2.0 ** -20) + P.abs() * keep + gm * least
        eP[~live] = 0
        eP = eP + g[:, None].abs() * 2.0 ** -23 * hot
        for out, A, B, eA, what in ((dx, P, W, eP, "dx"), (dw, P.T, X, eP.T, "dw")):
            if out is None:
                continue
            want = A @ B
            depth = A.shape[1] / 4 + 40
            tol = eA @ B.abs() + (depth * 2.0 ** -23 + (2.0 ** -20 if two else 0)) * (A.abs() @ B.abs())
            if two:
                tol = tol + 2.0 ** -38 * float(B.abs().max()) * A.abs().sum(1, keepdim=True)
            ulp = HALF_ULP[out.dtype]
            within(out, want, tol + ulp * (want.abs() + tol) + TINY[out.dtype], what)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", CE_SHAPES)
def test_linear_cross_entropy(eng, n, k, d, dtype):
    c = Ce(n, k, d, dtype, n + k + d, per_row=(n + k) % 2 == 0)
    c.check(c.run(eng))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("pad", [1, 8])
def test_linear_cross_entropy_row_strides(eng, dtype, pad):
    c = Ce(77, 301, 40, dtype, pad)
    c.check(c.run(eng, pad=pad))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=NAMES.get)
def test_linear_cross_entropy_f32_gradients_of_16_bit_inputs(eng, dtype):
    c = Ce(200, 500, 64, dtype, 5)
    c.check(c.run(eng, dxt=torch.float32, dwt=torch.float32))


def test_linear_cross_entropy_one_gradient_at_a_time(eng):
    c = Ce(90, 400, 48, torch.bfloat16, 6)
    both = c.run(eng)
    assert torch.equal(c.run(eng, dw=False)[2], both[2])
    assert torch.equal(c.run(eng, dx=False)[3], both[3])


@pytest.mark.parametrize("n,k,d,dtype", [(40000, 8000, 16, torch.bfloat16),
                                         (66000, 4096, 8, torch.bfloat16),
                                         (20000, 9000, 12, torch.float32)])
def test_linear_cross_entropy_in_pieces(eng, n, k, d, dtype):
    """More of P than the scratch holds: several pieces of the prototypes, and
    of the rows."""
    c = Ce(n, k, d, dtype, 11, per_row=False)
    c.check(c.run(eng))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_linear_cross_entropy_long_sums(eng, dtype):
    """dw sums over many rows of one sign: the chains of the tensor cores' cut
    sums would show."""
    c = Ce(16384, 8, 24, dtype, 12, ignored=0.0, per_row=False)
    c.x = c.x.abs()
    c.check(c.run(eng))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_linear_cross_entropy_ignored_rows(eng, dtype):
    c = Ce(150, 70, 32, dtype, 13, ignored=0.0)
    c.t[::3] = eb.IGNORE
    got = c.run(eng)
    c.check(got)
    assert (got[2][::3] == 0).all() and (got[0][::3] == 0).all()
    c.t[:] = eb.IGNORE
    loss, lse, dx, dw = c.run(eng)
    assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all() and lse.isfinite().all()


def test_linear_cross_entropy_zero_and_extreme_loss_gradients(eng):
    c = Ce(60, 50, 16, torch.float32, 14)
    c.dloss = torch.zeros(60, device="cuda")
    _, _, dx, dw = c.run(eng)
    assert (dx == 0).all() and (dw == 0).all()
    c.dloss = 1e-30 * randn(gen(1), 60)
    c.check(c.run(eng))
    c.dloss = 1e20 * randn(gen(1), 60)
    c.check(c.run(eng))
    c.dloss = -torch.ones(1, device="cuda")
    c.check(c.run(eng))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_linear_cross_entropy_large_scores(eng, dtype):
    """Scores of several hundred: exponentials far below the type's range, and
    rows whose target has no weight left."""
    c = Ce(100, 130, 64, dtype, 15, scale=40.0)
    c.check(c.run(eng))


def test_linear_cross_entropy_non_finite_row_stays_its_own(eng):
    for dtype in TYPES:
        c = Ce(140, 90, 32, dtype, 16, ignored=0.0)
        clean = c.run(eng)
        c.x[7, 3] = math.nan
        c.x[9, 1] = math.inf
        c.t[7] = eb.IGNORE
        loss, lse, dx, _ = c.run(eng)
        keep = torch.ones(140, dtype=torch.bool, device="cuda")
        keep[7] = keep[9] = False
        assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep])
        assert torch.equal(dx[keep], clean[2][keep])
        assert lse[7].isnan() and lse[9].isnan() and loss[9].isnan() and dx[9].isnan().any()
        assert loss[7] == 0


def test_linear_cross_entropy_of_no_rows(eng):
    w, dw = randn(gen(1), 9, 8), torch.ones(9, 8, device="cuda")
    e = eng.zeros_f32(0)
    t = eng.zeros_u32(0)
    eng.linear_cross_entropy(e, 0, 8, wrap(eng, w), 9, t, eng.zeros_f32(0), eng.zeros_f32(0))
    eng.linear_cross_entropy_backward(e, 0, 8, wrap(eng, w), 9, t, eng.zeros_f32(0),
                                      eng.zeros_f32(1), None, wrap(eng, dw))
    eng.sync()
    assert (dw == 0).all()


def test_linear_cross_entropy_target_out_of_range_is_reported(eng):
    c = Ce(40, 30, 16, torch.float32, 17, ignored=0.0)
    loss, lse = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    t = c.t.clone()
    t[5] = 30
    eng.linear_cross_entropy(wrap(eng, c.x), 40, 16, wrap(eng, c.w), 30,
                             wrap(eng, t.to(torch.uint32)), wrap(eng, loss), wrap(eng, lse))
    with pytest.raises(eb.EngineError) as err:
        eng.sync()
    assert err.value.code == eb.INVALID_ARGUMENT
    assert loss[5] == 0
    eng.sync()  # reported once


def test_linear_cross_entropy_is_the_same_bits_on_every_call(eng):
    c = Ce(700, 900, 128, torch.bfloat16, 18)
    a, b = c.run(eng), c.run(eng)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_linear_cross_entropy_gradient_is_the_difference_quotient(eng):
    """Central differences of the 64-bit loss (step 1e-5) against f32 gradients
    of order 1."""
    c = Ce(6, 7, 5, torch.float32, 19, ignored=0.2)
    _, _, dx, dw = c.run(eng)
    live = c.t != eb.IGNORE
    t = torch.where(live, c.t, torch.zeros_like(c.t))[:, None]

    def f(x, w):
        z = c.scale * (x @ w.T)
        loss = torch.logsumexp(z, 1) - z.gather(1, t)[:, 0]
        return float((loss * live * c.dloss.double()).sum())

    X, W = c.x.double(), c.w.double()
    for got, var, at in ((dx, X, 0), (dw, W, 1)):
        for i in range(var.numel()):
            pair = []
            for sign in (1e-5, -1e-5):
                v = var.clone()
                v.view(-1)[i] += sign
                pair.append(f(*((v, W) if at == 0 else (X, v))))
            want = (pair[0] - pair[1]) / 2e-5
            assert abs(float(got.reshape(-1)[i]) - want) <= 3e-5 * (1 + abs(want))


# ---------------------------------------------------------------- AdamW

HYPER = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8)


def plain_step(p, g, m, v, step, wd, gs=np.float32(1)):
    """The step in f32, each operation rounded by itself."""
    f = np.float32
    b1, b2, lr, eps = HYPER["beta1"], HYPER["beta2"], HYPER["lr"], HYPER["eps"]
    with np.errstate(over="ignore", invalid="ignore"):
        g = g * gs
        m = m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * g) * f(1 - b2)
        root = np.sqrt(v)
        size, fix = f(lr / (1 - b1 ** step)), f(1 / math.sqrt(1 - b2 ** step))
        p = p * f(1 - lr * wd) - m / (root * fix + f(eps)) * size
    return p, m, v, root


def bf16(a):
    return torch.from_numpy(a).to(torch.bfloat16)


def test_adamw_is_bitwise_the_rounded_formula_over_a_mixed_plan(eng):
    """f32 and bf16 parameters and gradients, lengths around the vector and
    piece sizes, an empty tensor, bf16 copies: three steps, each bit."""
    rng = np.random.default_rng(3)
    specs = [(n, pt, gt, cp) for n in (1, 3, 4, 255, 2047, 2048, 2049, 10001)
             for pt, gt, cp in (("f", "f", False), ("f", "b", True), ("b", "b", False), ("b", "f", True))]
    specs.append((0, "f", "f", False))
    ts, tensors = [], []
    for i, (n, pt, gt, cp) in enumerate(specs):
        d = {"p": rng.standard_normal(n).astype(np.float32), "g": rng.standard_normal(n).astype(np.float32),
             "m": 0.1 * rng.standard_normal(n).astype(np.float32),
             "v": (0.01 * rng.standard_normal(n).astype(np.float32)) ** 2, "wd": 0.01 * (i % 3), "pt": pt}
        if pt == "b":
            d["p"] = bf16(d["p"]).float().numpy()
        if gt == "b":
            d["g"] = bf16(d["g"]).float().numpy()
        d["dev"] = {q: torch.from_numpy(d[q]).cuda() for q in "pgmv"}
        if pt == "b":
            d["dev"]["p"] = d["dev"]["p"].to(torch.bfloat16)
        if gt == "b":
            d["dev"]["g"] = d["dev"]["g"].to(torch.bfloat16)
        d["copy"] = torch.zeros(n, device="cuda", dtype=torch.bfloat16) if cp else None
        tensors.append(d)
        hold = {q: (eng.wrap(t) if n else eng.zeros(eb.F32, 0)) for q, t in d["dev"].items()}
        ts.append(eb.AdamWTensor(**hold, copy=wrap(eng, d["copy"]) if n else None, weight_decay=d["wd"]))
    plan = eb.AdamW(eng, ts)
    launches = eng.stats()["kernel_launches"]
    for step in (1, 2, 3):
        plan.step(step=step, grad_scale=0.5, **HYPER)
        for d in tensors:
            p, d["m"], d["v"], _ = plain_step(d["p"], d["g"], d["m"], d["v"], step, d["wd"], np.float32(0.5))
            d["p"] = bf16(p).float().numpy() if d["pt"] == "b" else p
            d["new"] = p
    eng.sync()
    assert eng.stats()["kernel_launches"] == launches + 3
    for d in tensors:
        assert np.array_equal(d["dev"]["p"].float().cpu().numpy(), d["p"])
        assert np.array_equal(d["dev"]["m"].cpu().numpy(), d["m"])
        assert np.array_equal(d["dev"]["v"].cpu().numpy(), d["v"])
        if d["copy"] is not None:
            assert torch.equal(d["copy"].cpu(), bf16(d["new"]))


def test_adamw_against_64_bits(eng):
    """One step from zero states: p moves by lr (1 + a few roundings), and the
    moments are (1 - beta) g and g^2."""
    n = 4097
    rng = np.random.default_rng(5)
    p, g = rng.standard_normal(n).astype(np.float32), rng.standard_normal(n).astype(np.float32)
    dp, dg = torch.from_numpy(p).cuda(), torch.from_numpy(g).cuda()
    st = eb.AdamW.states(eng, n)
    eb.AdamW(eng, [eb.AdamWTensor(p=eng.wrap(dp), g=eng.wrap(dg), **st, weight_decay=0.1)]).step(
        step=1, **HYPER)
    eng.sync()
    P, G = p.astype(np.float64), g.astype(np.float64)
    want = P * (1 - HYPER["lr"] * 0.1) - HYPER["lr"] * G / (np.abs(G) + HYPER["eps"])
    assert np.all(np.abs(dp.cpu().numpy() - want) <= 2 * U32 * np.abs(P) + 16 * U32 * HYPER["lr"] + U32 * np.abs(want))
    assert np.all(np.abs(st["m"].read() - (1 - HYPER["beta1"]) * G) <= 4 * U32 * np.abs(G))
    assert np.all(np.abs(st["v"].read() - (1 - HYPER["beta2"]) * G * G) <= 6 * U32 * G * G)


def quantise(v, root):
    """Codes and scales of the 8-bit states, 256 elements a scale."""
    f = np.float32
    n = v.size
    pad = np.zeros(-(-n // 256) * 256, f)
    pad[:n] = v
    b = pad.reshape(-1, 256)
    scale = np.abs(b).max(1) * f(1 / 448)
    inv = np.where(scale > 0, f(1) / np.where(scale > 0, scale, f(1)), f(0)).astype(f)
    q = torch.from_numpy(np.clip(b * inv[:, None], -448, 448)).to(torch.float8_e4m3fn)
    if root:
        least = torch.full(q.shape, 2.0 ** -9)
        qf = q.float()
        q = torch.where(torch.from_numpy(b > 0), torch.maximum(qf, least), qf).to(torch.float8_e4m3fn)
    return q.reshape(-1)[:n], scale


@pytest.mark.parametrize("n", [1, 7, 255, 256, 257, 2048, 2049, 30011])
def test_adamw_8_bit_states(eng, n):
    """Three steps of 8-bit states from zero, each bit: codes, scales and
    parameters follow the rounded formula on the decoded states."""
    f = np.float32
    rng = np.random.default_rng(n)
    p = rng.standard_normal(n).astype(f)
    g = (rng.standard_normal(n) * 10.0 ** rng.uniform(-6, 2, n)).astype(f)
    g[::5] = 0
    g[:min(n, 256)] *= f(1e-9) if n > 300 else f(1)
    dp, dg = torch.from_numpy(p).cuda(), torch.from_numpy(g).cuda()
    copy = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    st = eb.AdamW.states(eng, n, eight_bit=True)
    plan = eb.AdamW(eng, [eb.AdamWTensor(p=eng.wrap(dp), g=eng.wrap(dg), copy=eng.wrap(copy), **st,
                                         weight_decay=0.02)])
    m, v = np.zeros(n, f), np.zeros(n, f)
    for step in (1, 2, 3):
        plan.step(step=step, **HYPER)
        p, m, v, root = plain_step(p, g, m, v, step, 0.02)
        qm, sm = quantise(m, False)
        qr, sr = quantise(root, True)
        eng.sync()
        assert np.array_equal(st["m"].read(), qm.view(torch.uint8).numpy())
        assert np.array_equal(st["v"].read(), qr.view(torch.uint8).numpy())
        assert np.array_equal(st["m_scale"].read(), sm) and np.array_equal(st["v_scale"].read(), sr)
        assert np.array_equal(dp.cpu().numpy(), p)
        assert torch.equal(copy.cpu(), bf16(p))
        each = np.repeat(sm, 256)[:n]
        m = qm.float().numpy() * each
        v = (qr.float().numpy() * np.repeat(sr, 256)[:n]) ** 2
        assert np.all((qr.float().numpy() > 0) == (root > 0)), "a root above zero stays above zero"


def test_adamw_8_bit_block_with_a_non_finite_gradient(eng):
    n = 700
    g = randn(gen(1), n)
    g[300] = math.inf
    p = randn(gen(2), n)
    st = eb.AdamW.states(eng, n, eight_bit=True)
    before = p.clone()
    eb.AdamW(eng, [eb.AdamWTensor(p=eng.wrap(p), g=eng.wrap(g), **st)]).step(step=1, **HYPER)
    eng.sync()
    ms = st["m_scale"].read()
    assert np.isfinite(ms[0]) and np.isnan(ms[1]) and np.isfinite(ms[2])
    assert p[300].isnan() and p[:256].isfinite().all() and p[512:].isfinite().all()
    assert (p[:256] != before[:256]).any()


def test_adamw_empty_plan(eng):
    eb.AdamW(eng, []).step(step=1, **HYPER)
    eng.sync()


# ---------------------------------------------------------------- streams and refusals

def test_operators_on_the_callers_stream(eng):
    """An engine on a torch stream runs in order with torch's work there: the
    rows are written, normalised and read back with no wait in between."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        e = eb.Engine(0, stream=side.cuda_stream)
        x = torch.empty(4000, 512, device="cuda")
        y = torch.empty_like(x)
        xb, yb = e.wrap(x), e.wrap(y)
        for i in range(5):
            x.normal_(mean=float(i)).mul_(1.0 + i)
            e.layer_norm(xb, 4000, 512, None, None, yb)
            got = y.clone()
            want = torch.nn.functional.layer_norm(x.double(), (512,))
            assert float((got.double() - want).abs().max()) < 1e-4
        assert e.stream() == side.cuda_stream
        e.sync()
        xb.free(), yb.free()
        e.close()
    side.synchronize()


def refused(fn, match):
    with pytest.raises(eb.EngineError, match=match) as err:
        fn()
    assert err.value.code == eb.INVALID_ARGUMENT


def test_layer_norm_refusals(eng):
    z = eng.zeros
    x, y, w, s = z(eb.F32, 64), z(eb.F32, 64), z(eb.F32, 8), z(eb.F32, 8)
    h = z(eb.BF16, 64)
    refused(lambda: eng.layer_norm(x, 8, 8, w, None, h), "one type")
    refused(lambda: eng.layer_norm(z(eb.U32, 64), 8, 8, w, None, y), "f32, bf16 or f16")
    refused(lambda: eng.layer_norm(x, 9, 8, w, None, y), "too short")
    refused(lambda: eng.layer_norm(x, 8, 8, w, None, y, ldx=9), "too short")
    refused(lambda: eng.layer_norm(x, 8, 8, w, None, y, ldx=7), "shorter than a row")
    refused(lambda: eng.layer_norm(x, 8, 0, w, None, y), "d must be positive")
    refused(lambda: eng.layer_norm(x, 2**63, 8, w, None, y), "too short")
    refused(lambda: eng.layer_norm(x, 8, 8, z(eb.F32, 7), None, y), "d elements")
    refused(lambda: eng.layer_norm(x, 8, 8, z(eb.BF16, 8), None, y), "weight and bias")
    refused(lambda: eng.layer_norm(h, 8, 8, z(eb.BF16, 8), w, z(eb.BF16, 64)), "one type")
    refused(lambda: eng.layer_norm(x, 8, 8, w, None, y, mean=z(eb.F32, 7)), "one element a row")
    refused(lambda: eng.layer_norm(x, 8, 8, w, None, y, eps=-1.0), "eps")
    refused(lambda: eng.layer_norm(x, 4, 8, w, None, eng.view(x, 16, 32, eb.F32)), "overlaps")
    refused(lambda: eng.layer_norm_backward(h, x, 8, 8, w, s, s, y), "one type")
    refused(lambda: eng.layer_norm_backward(y, x, 8, 8, w, s, z(eb.F32, 7), None), "one element a row")
    refused(lambda: eng.layer_norm_backward(y, x, 8, 8, w, s, s, x), "overlaps")
    refused(lambda: eng.layer_norm_backward(y, x, 8, 8, w, s, s, None, z(eb.F16, 8)), "dweight")


def test_linear_cross_entropy_refusals(eng):
    z = eng.zeros
    x, w, t, a, b = z(eb.F32, 64), z(eb.F32, 40), z(eb.U32, 8), z(eb.F32, 8), z(eb.F32, 8)
    ok = dict(x=x, n=8, d=8, w=w, k=5, targets=t, loss=a, lse=b)

    def call(**kw):
        return lambda: eng.linear_cross_entropy(**{**ok, **kw})

    refused(call(w=z(eb.BF16, 40)), "one type")
    refused(call(targets=a), "u32")
    refused(call(targets=z(eb.U32, 7)), "one element a row")
    refused(call(loss=z(eb.F32, 7)), "one element a row")
    refused(call(k=6), "too short")
    refused(call(k=0), "k must be positive")
    refused(call(scale=0.0), "scale")
    refused(call(scale=math.inf), "scale")
    refused(call(lse=a), "overlaps")
    refused(call(ldw=7), "shorter than a row")
    back = dict(x=x, n=8, d=8, w=w, k=5, targets=t, lse=b, dloss=z(eb.F32, 1), dx=z(eb.F32, 64),
                dw=z(eb.F32, 40))

    def grad(**kw):
        return lambda: eng.linear_cross_entropy_backward(**{**back, **kw})

    refused(grad(dloss=z(eb.F32, 2)), "dloss")
    refused(grad(dx=x), "overlaps")
    refused(grad(dx=z(eb.BF16, 64)), "x's type or f32|f32 or of x's type")
    refused(grad(dw=z(eb.F32, 39)), "too short")


def test_adamw_refusals(eng):
    z = eng.zeros

    def plan(**kw):
        t = dict(p=z(eb.F32, 300), g=z(eb.F32, 300), m=z(eb.F32, 300), v=z(eb.F32, 300))
        t.update(kw)
        return lambda: eb.AdamW(eng, [eb.AdamWTensor(**t)])

    refused(plan(p=z(eb.F16, 300)), "f32 or bf16")
    refused(plan(g=z(eb.F32, 299)), "one length")
    refused(plan(m=z(eb.F8, 300)), "f32 buffers")
    refused(plan(m_scale=z(eb.F32, 2)), "given together")
    refused(plan(m=z(eb.F8, 300), v=z(eb.F8, 300), m_scale=z(eb.F32, 1), v_scale=z(eb.F32, 2)),
            "each 256")
    refused(plan(copy=z(eb.F32, 300)), "copy")
    p = z(eb.F32, 300)
    refused(plan(p=p, m=p), "written twice")
    refused(plan(weight_decay=math.nan), "weight_decay")
    ok = plan()()
    refused(lambda: ok.step(step=0, lr=1e-3), "step")
    refused(lambda: ok.step(step=1, lr=math.nan), "lr")
    refused(lambda: ok.step(step=1, lr=1e-3, beta1=1.0), "betas")
    refused(lambda: ok.step(step=1, lr=1e-3, eps=-1.0), "eps")
