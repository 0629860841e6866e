"""The training operators at sizes that take several passes or pieces, checked
on slices that 64-bit formulas can afford, and shapes at the edges of their
kernels' variants."""

import math

import pytest
import torch

import emeans_b200 as eb
from tests.test_gpu_training_ops import (HALF_ULP, NAMES, TYPES, Ce, gen, randn, strided,
                                         test_layer_norm_backward as norm_backward,
                                         test_layer_norm_forward as norm_forward, within, wrap)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    e = eb.Engine(0, stream=torch.cuda.current_stream().cuda_stream)
    yield e
    e.close()


def score_error(c, rows, cols):
    """Ce.check's bound on the scores of some rows and columns."""
    X, W, s = c.x[rows].double(), c.w[cols].double(), c.scale
    cross = X.abs() @ W.abs().T
    ez = s * ((c.d / 4 + 8) * 2.0 ** -23 * cross)
    if c.dtype == torch.float32:
        ez = ez + s * 3 * 2.0 ** -22 * cross + s * 2.0 ** -38 * (
            float(c.x.abs().max()) * W.abs().sum(1)[None, :] +
            float(c.w.abs().max()) * X.abs().sum(1)[:, None])
    return X, W, ez


def test_linear_cross_entropy_forward_in_row_passes(eng):
    """More half tiles than the scratch keeps: rows in two passes."""
    n, k, d = 70000, 40000, 8
    c = Ce(n, k, d, torch.bfloat16, 21, per_row=False)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    eng.linear_cross_entropy(wrap(eng, c.x), n, d, wrap(eng, c.w), k,
                             wrap(eng, c.t.to(torch.uint32)), wrap(eng, loss), wrap(eng, lse),
                             scale=c.scale)
    eng.sync()
    cols = torch.arange(k, device="cuda")
    for rows in (torch.arange(300, device="cuda"), torch.arange(66300, 67100, device="cuda"),
                 torch.arange(n - 300, n, device="cuda")):
        X, W, ez = score_error(c, rows, cols)
        Z = c.scale * (X @ W.T)
        L = torch.logsumexp(Z, 1)
        el = ez.amax(1) + 2.0 ** -20 + 6 * 2.0 ** -23 * (L.abs() + Z.abs().amax(1))
        within(lse[rows], L, el, "lse")
        t = c.t[rows]
        live = t != eb.IGNORE
        zt = Z.gather(1, torch.where(live, t, 0 * t)[:, None])[:, 0]
        within(loss[rows], torch.where(live, L - zt, 0 * L), 2 * el + 2.0 ** -21 * zt.abs(), "loss")


def test_linear_cross_entropy_pieces_of_both_sides(eng):
    """So many rows and prototypes that P is cut both ways: rows of dx and of dw
    against their own sums over everything."""
    n, k, d = 70000, 66000, 4
    c = Ce(n, k, d, torch.float32, 22, per_row=False)
    c.dloss = torch.full((1,), 1.0, device="cuda")
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    dx, dw = torch.empty(n, d, device="cuda"), torch.empty(k, d, device="cuda")
    tb = wrap(eng, c.t.to(torch.uint32))
    eng.linear_cross_entropy(wrap(eng, c.x), n, d, wrap(eng, c.w), k, tb, wrap(eng, loss),
                             wrap(eng, lse), scale=c.scale)
    eng.linear_cross_entropy_backward(wrap(eng, c.x), n, d, wrap(eng, c.w), k, tb, wrap(eng, lse),
                                      wrap(eng, c.dloss), wrap(eng, dx), wrap(eng, dw),
                                      scale=c.scale)
    eng.sync()
    everyone = {0: torch.arange(n, device="cuda"), 1: torch.arange(k, device="cuda")}
    for rows, cols in ((torch.tensor([0, 5, 65535, 65536, n - 1], device="cuda"), everyone[1]),
                       (everyone[0], torch.tensor([0, 7, 2047, 2048, 65000, k - 1], device="cuda"))):
        X, W, ez = score_error(c, rows, cols)
        L = lse[rows].double()
        live = (c.t[rows] != eb.IGNORE)[:, None]
        hot = (c.t[rows][:, None] == cols[None, :]).double()
        p = torch.exp(c.scale * (X @ W.T) - L[:, None])
        P = torch.where(live, c.scale * (p - hot), 0 * p)
        eP = torch.where(live, c.scale * p * (ez + 2.0 ** -20 + 2.0 ** -22 * L[:, None].abs()), 0 * p)
        eP = eP + P.abs() * 2.0 ** -21 + c.scale * (2.0 ** -37 + 2.0 ** -23 * hot)
        if len(rows) < len(cols):
            got, A, B, eA = dx[rows], P, W, eP
        else:
            got, A, B, eA = dw[cols], P.T, X, eP.T
        # Chains of 128 products, and one rounded sum of each chain and piece.
        tol = eA @ B.abs() + (2.0 ** -20 + 600 * 2.0 ** -23) * (A.abs() @ B.abs()) + \
            2.0 ** -38 * float(B.abs().max()) * A.abs().sum(1, keepdim=True)
        within(got, A @ B, tol, "dx" if len(rows) < len(cols) else "dw")


# Rows that fill 4, 8, 16 and 32 packs of 16 bytes and one element to either
# side, several packs a lane, and whole blocks a row.
EDGE_WIDTHS = [15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 255, 257, 511, 513, 769, 1023, 1025,
               4097, 8191, 8192, 8193]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("d", EDGE_WIDTHS)
def test_layer_norm_widths(eng, d, dtype):
    rows = 600 if d < 300 else 37
    for pad in (0, 3, 8):
        norm_forward(eng, rows, d, dtype, pad)
    norm_backward(eng, rows, d, dtype)
    norm_backward(eng, rows + 1, d, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("d", [768, 776, 1023, 1025, 1536, 1544, 2049, 3079, 4104, 6144, 6150])
def test_layer_norm_of_several_warps_a_row(eng, d, dtype):
    """Both sides of each change of the group that holds a row."""
    for rows, pad in ((37, 0), (37, 3), (1201, 8)):
        norm_forward(eng, rows, d, dtype, pad)
    norm_backward(eng, 37, d, dtype)
    norm_backward(eng, 1201, d, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_layer_norm_rows_aligned_apart(eng, dtype):
    """Row strides of the tensors that leave their rows aligned differently:
    element by element."""
    rows, d = 41, 70
    x = randn(gen(3), rows, d).to(dtype)
    xf, _ = strided(x, d + 1)
    y, yv = strided(torch.zeros_like(x), d + 2, fill=7.0)
    eng.layer_norm(wrap(eng, xf), rows, d, None, None, wrap(eng, y), ldx=d + 1, ldy=d + 2)
    eng.sync()
    X = x.double()
    c = X - X.mean(1, keepdim=True)
    want = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt()
    within(yv, want, 60 * 2.0 ** -23 * 8 + HALF_ULP[dtype] * want.abs(), "y")
    assert (y.view(rows, d + 2)[:, d:] == 7.0).all()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 4735, 4737])
@pytest.mark.parametrize("k,d", [(64, 64), (65, 64), (64, 65), (1, 64), (63, 3)])
def test_linear_cross_entropy_around_the_small_kernels_limits(eng, n, k, d):
    c = Ce(n, k, d, torch.float32, n + k + d, per_row=n % 2 == 0)
    c.check(c.run(eng))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n", [1, 8, 127, 128, 129])
def test_linear_cross_entropy_few_rows(eng, n, dtype):
    """One CTA a tile up to 128 rows, a pair past them; tiles of several widths."""
    for k in (1000, 40000):
        c = Ce(n, k, 72, dtype, n + k, per_row=False)
        c.check(c.run(eng))


@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("k,d", [(1, 65), (3, 93), (127, 31), (700, 1), (4097, 333), (31, 1024),
                                 (9000, 1023), (500, 1025)])
def test_linear_cross_entropy_few_f32_rows(eng, n, k, d):
    """Rows up to 16 of 32 bits, to both sides of the widest, with row strides."""
    for pad in (0, 3):
        c = Ce(n, k, d, torch.float32, n + k + d, per_row=n % 2 == 0, ignored=0.3)
        c.check(c.run(eng, pad=pad))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=NAMES.get)
@pytest.mark.parametrize("n,k,d", [(1, 3, 93), (4, 700, 1), (5, 4097, 333), (8, 129, 66), (9, 31, 1023),
                                   (16, 9000, 420), (16, 500, 1025)])
def test_linear_cross_entropy_few_16_bit_rows_off_alignment(eng, n, k, d, dtype):
    for pad in (0, 3):
        c = Ce(n, k, d, dtype, n + k + d, per_row=n % 2 == 0)
        c.check(c.run(eng, pad=pad))
    c.check(c.run(eng, dxt=torch.float32, dwt=torch.float32))


def test_linear_cross_entropy_few_f32_rows_one_gradient_and_bits(eng):
    c = Ce(7, 1003, 129, torch.float32, 5)
    both, again = c.run(eng), c.run(eng)
    for a, b in zip(both, again):
        assert torch.equal(a, b)
    assert torch.equal(c.run(eng, dw=False)[2], both[2])
    assert torch.equal(c.run(eng, dx=False)[3], both[3])


def test_linear_cross_entropy_few_f32_rows_non_finite(eng):
    """A row without a gradient stays at zero whatever it holds; another row's
    infinities reach its own loss only."""
    c = Ce(6, 300, 70, torch.float32, 9, ignored=0.0)
    c.t[2] = eb.IGNORE
    c.x[2, 3], c.x[4, 5] = math.nan, math.inf
    loss, lse, dx, dw = c.run(eng)
    assert loss[2] == 0 and (dx[2] == 0).all()
    assert not torch.isfinite(loss[4])
    rest = [0, 1, 3, 5]
    X, W = c.x.double()[rest], c.w.double()
    Z = c.scale * (X @ W.T)
    want = torch.logsumexp(Z, 1) - Z.gather(1, c.t[rest][:, None])[:, 0]
    tol = 2.0 ** -19 * (1 + Z.abs().amax(1)) + (c.d / 4 + 8) * 2.0 ** -22 * c.scale * (
        X.abs() @ W.abs().T).amax(1)
    within(loss[rest], want, tol, "loss")


def test_linear_cross_entropy_long_rows(eng):
    """Scores of 16-bit rows past 768 columns, summed in chains: FP32's own
    error, well inside Ce.check's bound for one chain."""
    c = Ce(64, 500, 3000, torch.bfloat16, 30, lean=30.0, scale=0.2)
    got = c.run(eng)
    c.check(got)
    z = c.scale * (c.x.double() @ c.w.double().T)
    assert float((got[1].double() - torch.logsumexp(z, 1)).abs().max()) <= \
        2.0 ** -20 * (1 + float(z.abs().max()))
