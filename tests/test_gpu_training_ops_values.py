"""The training operators over the whole range of values that their types hold:
rows, prototypes, features and loss gradients that lie orders of magnitude
apart, very large and very small ones, against 64-bit formulas with bounds of
each row's own size."""

import math

import pytest
import torch

import emeans_b200 as eb
from tests.test_gpu_training_ops import (HALF_ULP, NAMES, TINY, TYPES, U32, gen, randn, within,
                                         wrap)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = eb.Engine(0, stream=torch.cuda.current_stream().cuda_stream)
    yield e
    e.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=NAMES.get)
@pytest.mark.parametrize("d", [1, 3, 70, 387, 700, 1023, 5000])
def test_layer_norm_backward_of_large_rows_without_spread(eng, d, dtype):
    """Rows of 1e37 alike: x - mean is 0, whatever their mean times rstd is, so
    dx = rstd (h - avg h) and dweight = 0. The bound: the sum of h and its
    mean (at most 64 roundings a thread and its group), and four more."""
    rows = 5
    g = gen(d)
    x = torch.full((rows, d), 1e37, device="cuda", dtype=dtype)
    dy, w = randn(g, rows, d).to(dtype), 1 + 0.2 * randn(g, d)
    mean, rstd = x[:, 0].float().clone(), torch.full((rows,), 316.0, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    eng.layer_norm_backward(wrap(eng, dy), wrap(eng, x), rows, d, wrap(eng, w), wrap(eng, mean),
                            wrap(eng, rstd), wrap(eng, dx), wrap(eng, dw), wrap(eng, db))
    eng.sync()
    h = dy.double() * w.double()
    want = 316.0 * (h - h.mean(1, keepdim=True))
    tol = 316.0 * (64 * 2 * U32 * h.abs().mean(1, keepdim=True) + 8 * U32 * h.abs())
    within(dx, want, tol + HALF_ULP[dtype] * (want.abs() + tol), "dx")
    assert (dw == 0).all()
    within(db, dy.double().sum(0), rows * 2 * U32 * dy.double().abs().sum(0), "dbias")


# ---------------------------------------------------------------- linear cross entropy


class Values:
    """One problem, run through the engine and in 64 bits, and the bounds of
    each output by the row's own size (`check`)."""

    def __init__(self, n, k, d, dtype, seed, ignored=0.1, scale=1.0):
        g = gen(seed)
        self.n, self.k, self.d, self.scale, self.dtype = n, k, d, scale, dtype
        self.x, self.w = randn(g, n, d), 0.3 * randn(g, k, d)
        t = torch.randint(0, k, (n,), generator=g, device="cuda")
        drop = torch.rand(n, generator=g, device="cuda") < ignored
        drop[3] = True
        self.t = torch.where(drop, torch.full_like(t, eb.IGNORE), t)
        self.dloss = randn(g, n)
        self.rand = torch.rand(n, generator=g, device="cuda")

    def run(self, e, outs=None):
        """loss, lse, dx and dw; dx and dw of `outs`' type, or x's."""
        n, k, d = self.n, self.k, self.d
        self.x, self.w = self.x.to(self.dtype), self.w.to(self.dtype)
        loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        dx = torch.empty(n, d, device="cuda", dtype=outs or self.dtype)
        dw = torch.empty(k, d, device="cuda", dtype=outs or self.dtype)
        xb, wb, tb, lb = wrap(e, self.x), wrap(e, self.w), wrap(e, self.t.to(torch.uint32)), wrap(e, lse)
        e.linear_cross_entropy(xb, n, d, wb, k, tb, wrap(e, loss), lb, scale=self.scale)
        e.linear_cross_entropy_backward(xb, n, d, wb, k, tb, lb, wrap(e, self.dloss), wrap(e, dx),
                                        wrap(e, dw), scale=self.scale)
        e.sync()
        return loss, lse, dx, dw

    def check(self, got, floor=True):
        """Against 64 bits. (Without `floor`: f32's terms leave nothing out.) A score is off by its products' roundings (2^-22
        each for f32's terms) and sums (cut, at most d / 4 + 8 of them), and
        by 2^-26 of its row's and its prototype's largest element for each of
        the other's (what the terms of f32 may leave out). P: the scores'
        errors, the exponential's, its own rounding (`keep`) and 2^-25 of the
        row's loss gradient. The gradients: P's error through the other
        operand, the products and sums again, and 2^-26 of each row's largest
        element for each weight."""
        loss, lse, dx, dw = got
        X, W, s = self.x.double(), self.w.double(), self.scale
        live = self.t != eb.IGNORE
        t = torch.where(live, self.t, torch.zeros_like(self.t))[:, None]
        f32 = self.dtype == torch.float32
        Z = s * (X @ W.T)
        cross = X.abs() @ W.abs().T
        top_x, top_w = X.abs().amax(1, keepdim=True), W.abs().amax(1, keepdim=True)
        ez = s * cross * ((self.d / 4 + 8) * 2.0 ** -23 + (3 * 2.0 ** -22 if f32 else 0))
        if f32 and floor:
            ez = ez + s * 2.0 ** -26 * (top_x * W.abs().sum(1)[None, :] + top_w.T * X.abs().sum(1, keepdim=True))
        L = torch.logsumexp(Z, 1)
        el = ez.amax(1) + 2.0 ** -20 + 6 * 2.0 ** -23 * (L.abs() + Z.abs().amax(1))
        within(lse, L, el, "lse")
        zt = Z.gather(1, t)[:, 0]
        within(loss, torch.where(live, L - zt, 0 * L),
               torch.where(live, el + ez.gather(1, t)[:, 0] + 4 * 2.0 ** -23 * zt.abs(), 0 * L), "loss")
        g = torch.where(live, self.dloss.double().expand(self.n), 0 * L)[:, None] * s
        p = torch.exp(Z - L[:, None])
        hot = torch.zeros_like(p).scatter_(1, t, 1.0)
        P = g * (p - hot)
        keep = {torch.float32: 2.0 ** -21, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -10}[self.dtype]
        least = 2.0 ** -25 if floor else 2.0 ** -100
        eP = g.abs() * (p * (ez + 2 * el[:, None] + 2.0 ** -20) + 2.0 ** -23 * hot + least) + P.abs() * keep
        for out, A, B, eA, top, what in ((dx, P, W, eP, top_w, "dx"), (dw, P.T, X, eP.T, top_x, "dw")):
            want = A @ B
            tol = eA @ B.abs() + ((A.shape[1] / 4 + 40) * 2.0 ** -23 + (2.0 ** -20 if f32 else 0)) * (A.abs() @ B.abs())
            if f32 and floor:
                tol = tol + 2.0 ** -26 * (A.abs() @ top)
            tol = tol + HALF_ULP[out.dtype] * (want.abs() + tol) + TINY[out.dtype]
            most = float(torch.finfo(out.dtype).max)
            assert out[want.abs() - tol > 1.001 * most].isinf().all(), what  # past the type
            fits = want.abs() + tol <= most
            within(out[fits], want[fits], tol[fits], what)


# Shapes of each kind of tile (pairs, single CTAs, narrow ones), off 16 bytes too.
SHAPES = [(300, 200, 130), (40, 3000, 72), (700, 1100, 264), (129, 70, 40)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", SHAPES)
def test_loss_gradient_of_a_row_without_a_target_is_not_used(eng, n, k, d, dtype):
    """Whatever an ignored row's loss gradient holds, every output is the same."""
    c = Values(n, k, d, dtype, 1)
    clean = c.run(eng)
    c.check(clean)
    for value in (1e30, -3e38, math.inf, math.nan, 0.0):
        c.dloss[3] = value
        for a, b in zip(c.run(eng), clean):
            assert torch.equal(a, b)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", SHAPES + [(50, 30, 20), (9, 300, 65)])
def test_one_non_finite_loss_gradient_leaves_ignored_rows_at_zero(eng, n, k, d, dtype, value):
    c = Values(n, k, d, dtype, 2)
    c.dloss = torch.full((1,), value, device="cuda")
    _, _, dx, dw = c.run(eng)
    none = c.t == eb.IGNORE
    assert none.any() and (dx[none] == 0).all()
    assert not dx[~none].isfinite().any() and not dw.isfinite().any()


@pytest.mark.parametrize("sizes", [(1e-25, 1e-25, 1.0, 1.0), (1e-33, 1e-30, 1.0, 1.0),
                                   (1e15, 1e-25, 1e10, 1e-5), (1e-25, 1e15, 1e10, 1e5),
                                   (1e-20, 1e-18, 1e38, 1e-30), (1e17, 1e18, 1e-35, 1.0)], ids=str)
@pytest.mark.parametrize("n,k,d", SHAPES)
def test_rows_and_prototypes_of_any_size(eng, n, k, d, sizes):
    """f32 rows, prototypes, scale and loss gradients whose products stay in
    range though those of some factors leave it."""
    c = Values(n, k, d, torch.float32, 3)
    c.x, c.w, c.scale, c.dloss = c.x * sizes[0], c.w * sizes[1], sizes[2], c.dloss * sizes[3]
    c.check(c.run(eng))


def masked_row(c):
    c.x[3] = 1e30  # ignored


def small_rows(c):
    c.x[5::7] *= 1e-9
    c.x[6] *= 1e-20


def small_prototypes(c):
    c.w[5::7] *= 1e-9
    c.w[6] *= 1e-20


def features_apart(c):
    c.x[:, 5], c.w[:, 5] = c.x[:, 5] * 1e9, c.w[:, 5] * 1e-9
    c.x[:, 7], c.w[:, 7] = c.x[:, 7] * 1e-12, c.w[:, 7] * 1e10


def loss_gradients_apart(c):
    c.dloss = c.dloss.sign() * 10.0 ** (-12 * c.rand)


def loss_gradients_far_apart(c):
    c.dloss = c.dloss.sign() * 10.0 ** (-50 * c.rand + 20)


def one_row(c):
    """A single element that is not 0 in a row and in a column."""
    c.x[9] = 0
    c.x[9, 2] = 1e-15
    c.w[:, 4] = 0
    c.w[11, 4] = 1e-15


@pytest.mark.parametrize("edit", [masked_row, small_rows, small_prototypes, features_apart,
                                  loss_gradients_apart, loss_gradients_far_apart, one_row],
                         ids=lambda f: f.__name__)
@pytest.mark.parametrize("n,k,d", SHAPES + [(20, 5000, 520), (257, 513, 1100), (3000, 1000, 392)])
def test_f32_values_orders_of_magnitude_apart(eng, n, k, d, edit):
    """What lies far below the largest of its matrix keeps its own 22 bits: rows,
    prototypes and features, and gradients of rows of little weight."""
    c = Values(n, k, d, torch.float32, 4)
    edit(c)
    got = c.run(eng)
    c.check(got, floor=False)
    for a, b in zip(c.run(eng), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n,k,d", SHAPES)
def test_f32_non_finite_rows_beside_values_apart(eng, n, k, d):
    """In three terms as in two: a row with a NaN or an infinity stays its own."""
    c = Values(n, k, d, torch.float32, 5, ignored=0.0)
    small_rows(c)
    clean = c.run(eng)
    c.x[7, 3], c.x[9, 1] = math.nan, math.inf
    c.t[7] = eb.IGNORE
    loss, lse, dx, _ = c.run(eng)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[7] = keep[9] = False
    assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(lse[keep], clean[1][keep])
    assert torch.equal(dx[keep], clean[2][keep])
    assert lse[7].isnan() and lse[9].isnan() and loss[9].isnan() and dx[9].isnan().any()
    assert loss[7] == 0 and (dx[7] == 0).all()


def sparse(c):
    """Most elements 0, whole columns too: no block of rows sees every column."""
    c.x = torch.where(c.x > 1.0, c.x, 0 * c.x)
    c.x[:, 2::9] = 0
    c.w[:, 1::5] = 0
    c.w[20:, 3::7] = 0


def sparse_and_apart(c):
    sparse(c)
    c.x[8, 0], c.w[8, 0] = 1e9, 1e-9
    c.x[9:, 0] = 0


def sparse_rows(c):
    """The prototypes' columns are all there."""
    w = c.w.clone()
    sparse(c)
    c.w = w


def sparse_range(c):
    """Columns of zeros in one range of columns alone (of 1,024), and a far
    smaller one there."""
    c.x[:, :2] = 0
    c.w[:, 1] *= 1e-6


@pytest.mark.parametrize("edit,floor", [(sparse, True), (sparse_and_apart, False), (sparse_rows, True),
                                        (sparse_range, False)], ids=lambda v: getattr(v, "__name__", ""))
@pytest.mark.parametrize("n,k,d", SHAPES + [(257, 513, 2100), (3000, 1000, 392), (70, 900, 60)])
def test_f32_columns_of_zeros(eng, n, k, d, edit, floor):
    c = Values(n, k, d, torch.float32, 6)
    edit(c)
    c.check(c.run(eng), floor)


def test_f32_calls_leave_nothing_for_the_next(eng):
    """What one call finds in its rows is not there in the next one's."""
    c = Values(300, 200, 130, torch.float32, 7)
    clean = c.run(eng)
    big = Values(300, 200, 130, torch.float32, 8)
    big.x, big.dloss = big.x * 1e20, big.dloss * 1e-20
    small_prototypes(big)
    big.run(eng)
    wider = Values(40, 300, 1500, torch.float32, 9)
    wider.check(wider.run(eng))
    for a, b in zip(c.run(eng), clean):
        assert torch.equal(a, b)


@pytest.mark.parametrize("size", [1e3, 1e5, 1e9])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", SHAPES + [(257, 513, 1100), (300, 4000, 800), (9, 300, 65), (50, 30, 20)])
def test_rows_of_very_large_scores(eng, n, k, d, dtype, size):
    """Rows far longer than the rest, whose softmax is one prototype's: their
    gradient is g scale (w of the best - w of the target), though the last bit
    of their scores is many units; the other rows' is as ever."""
    c = Values(n, k, d, dtype, 10, ignored=0.0)
    c.t[3] = 0
    big = torch.arange(0, n, 7, device="cuda")
    c.x[big] *= size if dtype != torch.float16 else min(size, 1e4)
    loss, lse, dx, dw = c.run(eng)
    # Rows of 1e3 stay within what two FP16 terms hold, and f16's P has its floor.
    c.check((loss, lse, dx, dw), floor=size == 1e3 or dtype == torch.float16)
    X, W = c.x[big].double(), c.w.double()
    z = X @ W.T
    two = z.topk(2, 1).values
    # A best score that no rounding of the scores can bring near another.
    near = (2.0 ** -20 + d * 2.0 ** -24) * (X.abs() @ W.abs().T).amax(1)
    clear = two[:, 0] - two[:, 1] > 100.0 + 4 * near
    assert size < 1e5 or clear.sum() >= len(big) // 2
    rows = big[clear]
    g = c.dloss[rows].double()[:, None]
    want = g * (W[z[clear].argmax(1)] - W[c.t[rows]])
    tol = g.abs() * 2.0 ** -19 * (W[z[clear].argmax(1)].abs() + W[c.t[rows]].abs())
    keep = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -9}[dtype]
    tol = tol + keep * g.abs() * (W[z[clear].argmax(1)].abs() + W[c.t[rows]].abs())
    within(dx[rows], want, tol + HALF_ULP[dtype] * want.abs() + 2.0 ** -24, "dx of the clear rows")


# ---------------------------------------------------------------- long sums, and f32 gradients


def uniform_rows(n, k, d, dtype, seed):
    """Positive rows whose scores are all near 0, and one target: every other
    prototype's gradient is g scale / k times the sum of the rows."""
    c = Values(n, k, d, dtype, seed, ignored=0.0, scale=1e-6)
    c.x, c.t, c.dloss = c.x.abs(), torch.zeros_like(c.t), torch.full((1,), 1.0, device="cuda")
    return c


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", [(16384, 96, 80), (70000, 100, 72)])
def test_f32_gradients_of_long_one_signed_sums(eng, n, k, d, dtype):
    """Sums of one sign over many rows, in f32: the tensor cores cut their sums
    (2^-24 a step of 16 rows at worst, 2^-26 in the mean), which one chain over the rows
    would show (two-term sums 1.8e-5), and P alike in all rows, whose rounding to 16
    bits would (2e-3). P is off by the last bits of the log-sum (2^-22) and of the
    exponent (2^-22) and by the exponential (2^-22): 1e-6 at most, alike in all
    rows; chains of 128 rows by 24 cut steps of three products (2^-26 each: 4e-7),
    and the rounded additions of their sums by at most 2^-24 a chain of a split
    (600: 3.6e-5 at worst, but of either sign: 25 times 2^-24). 4e-6, and 2e-6 in the mean."""
    c = uniform_rows(n, k, d, dtype, 11)
    _, _, dx, dw = c.run(eng, outs=torch.float32)
    X, W = c.x.double(), c.w.double()
    p = torch.softmax(c.scale * (X @ W.T), 1)
    p[:, 0] -= 1
    want = c.scale * (p.T @ X)
    off = ((dw.double() - want) / want)[1:]
    assert float(off.abs().max()) <= 4e-6 and float(off.mean().abs()) <= 2e-6
    want = c.scale * (p @ W)
    assert float((dx.double() - want).abs().max() / want.abs().max()) <= 4e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", SHAPES + [(257, 513, 1100), (3000, 1000, 392), (20000, 9000, 16)])
def test_f32_gradients_of_16_bit_rows_keep_p(eng, n, k, d, dtype):
    """Rows' gradients in f32, against 64 bits of the same 16-bit inputs: FP32's
    own error (5e-6 of a row's norm at 2,000 products; P in bf16 or f16 alone is 2e-3
    or 2e-4 off), whichever of the two is wanted in f32."""
    c = Values(n, k, d, dtype, 12)
    got = c.run(eng, outs=torch.float32)
    X, W = c.x.double(), c.w.double()
    live = c.t != eb.IGNORE
    t = torch.where(live, c.t, 0 * c.t)[:, None]
    p = torch.softmax(X @ W.T, 1).scatter_add(1, t, -torch.ones_like(t, dtype=torch.float64))
    p = p * torch.where(live, c.dloss.double(), 0.0)[:, None]
    for out, want in ((got[2], p @ W), (got[3], p.T @ X)):
        norm = want.norm(dim=1)
        some = norm > 1e-3 * norm.max()
        off = (out.double() - want).norm(dim=1)[some] / norm[some]
        assert float(off.max()) <= 3e-5 and float(off.median()) <= 5e-6
    e, lse = eng, got[1]
    dw = torch.empty(k, d, device="cuda")
    dx = torch.empty(n, d, device="cuda", dtype=dtype)
    e.linear_cross_entropy_backward(wrap(e, c.x), n, d, wrap(e, c.w), k, wrap(e, c.t.to(torch.uint32)),
                                    wrap(e, lse), wrap(e, c.dloss), wrap(e, dx), wrap(e, dw))
    e.sync()
    assert torch.equal(dw, got[3]) and torch.equal(dx, got[2].to(dtype))


def test_linear_cross_entropy_passes_hold_the_scratch(eng):
    """Tiles of 128 columns and fewer leave more half tiles: the rows go in more
    passes (two launches each), not in more than 256 MB of their sums."""
    n, k, d = 640, 3490000, 900
    e = eb.Engine(0, stream=torch.cuda.current_stream().cuda_stream)
    x, w = torch.zeros(n, d, device="cuda"), torch.zeros(k, d, device="cuda")
    t = torch.zeros(n, device="cuda", dtype=torch.int32)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    before = e.stats()["kernel_launches"]
    e.linear_cross_entropy(e.wrap(x), n, d, e.wrap(w), k, e.wrap(t), e.wrap(loss), e.wrap(lse))
    e.sync()
    launches = e.stats()["kernel_launches"] - before
    assert launches >= 2 + 2 * 2
    assert float((lse - math.log(k)).abs().max()) < 1e-5 and torch.equal(loss, lse)
    e.close()


@pytest.mark.parametrize("size", [1e3, 1e5, 1e9])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", SHAPES + [(257, 513, 1100), (9, 300, 65), (4, 5000, 41), (50, 30, 20)])
def test_rows_of_very_large_scores_under_a_scale(eng, n, k, d, dtype, size):
    """The same with a scale that scores are rounded by: a score less its row's
    log-sum is 0 or less, never the rounding of a product."""
    c = Values(n, k, d, dtype, 13, ignored=0.0, scale=1.3)
    c.t[:] = torch.arange(n, device="cuda") % k
    big = torch.arange(0, n, 2, device="cuda")
    c.x[big] *= size if dtype != torch.float16 else min(size, 1e4)
    c.dloss = 1e-3 * c.dloss
    loss, lse, dx, dw = c.run(eng)
    c.check((loss, lse, dx, dw), floor=size == 1e3 or dtype == torch.float16)
    X, W = c.x[big].double(), c.w.double()
    z = c.scale * (X @ W.T)
    two = z.topk(2, 1).values
    near = c.scale * (2.0 ** -20 + d * 2.0 ** -24) * (X.abs() @ W.abs().T).amax(1)
    clear = two[:, 0] - two[:, 1] > 100.0 + 4 * near
    assert size < 1e5 or clear.sum() >= len(big) // 2
    rows = big[clear]
    g = c.scale * c.dloss[rows].double()[:, None]
    best = W[z[clear].argmax(1)]
    want = g * (best - W[c.t[rows]])
    keep = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -9}[dtype]
    tol = (2.0 ** -19 + keep) * g.abs() * (best.abs() + W[c.t[rows]].abs())
    # P of f16 and of two terms leaves out 2^-38 of the largest loss gradient.
    tol = tol + 2.0 ** -36 * float(c.dloss.abs().max()) * W.abs().sum(0)
    within(dx[rows], want, tol + HALF_ULP[dtype] * want.abs() + 2 * TINY[dtype], "dx of the clear rows")
