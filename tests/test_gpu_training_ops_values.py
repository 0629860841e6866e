"""The training operators over the whole range of values that their types hold:
rows, prototypes, features and loss gradients that lie orders of magnitude
apart, very large and very small ones, against 64-bit formulas with bounds of
each row's own size."""

import math

import pytest
import torch

import emeans_b200 as eb
from tests.test_gpu_training_ops import HALF_ULP, NAMES, TYPES, U32, gen, randn, within, wrap

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
