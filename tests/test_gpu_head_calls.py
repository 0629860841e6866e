"""The cluster head's calls in other orders and with other inputs than a run of
steps: losses between calls, batches of no rows, rows of another width."""

import numpy as np
import pytest

import emeans_b200 as eb
from emeans_b200.head import ClusterHead

pytestmark = pytest.mark.gpu

D, K = 24, 9


def batch(n, seed):
    rng = np.random.default_rng(seed)
    return rng.standard_normal((n, D)).astype(np.float32), rng.integers(0, K, n).astype(np.uint32)


def test_last_loss_is_the_last_steps_whatever_is_called_after_it(engine):
    head = ClusterHead(engine, D, K, seed=1)
    with pytest.raises(RuntimeError, match="no step"):
        head.last_loss()
    x, labels = batch(100, 1)
    labels[::9] = eb.IGNORE
    before = head.evaluate(x, labels)
    head.step(x, labels, lr=1e-2)
    assert head.last_loss() == before
    head.evaluate(x[:90], np.zeros(90, np.uint32))  # fewer rows, in the same buffers
    assert head.last_loss() == before
    head.evaluate(*batch(300, 2))  # more rows, in new ones
    assert head.last_loss() == before
    head.predict(batch(500, 3)[0])
    assert head.last_loss() == before
    head.step(x[:40], labels[:40], lr=1e-2)
    assert head.last_loss() != before


def test_batches_of_no_rows(engine):
    """No loss, no predictions, and a step whose gradients are zero: the first
    moments stay zero and the weights take the decay alone."""
    head = ClusterHead(engine, D, K, seed=2, weight_decay=0.5)
    x, labels = batch(0, 1)
    w = head.w.read()
    assert head.evaluate(x, labels) == 0.0 and head.predict(x).shape == (0,)
    head.step(x, labels, lr=1e-2)
    assert head.last_loss() == 0.0
    keep = np.float32(1.0 - 1e-2 * 0.5)
    assert np.array_equal(head.w.read(), w * keep) and np.array_equal(head.weight.read(), np.ones(D))


def test_rows_of_another_width_are_refused(engine):
    head = ClusterHead(engine, D, K)
    for x in (np.zeros((10, 2 * D), np.float32), np.zeros((3 * D, 1), np.float32)):
        with pytest.raises(ValueError, match="rows of"):
            head.step(x, np.zeros(x.size // D, np.uint32), lr=1e-3)
    for x in (np.zeros(5 * D + 1, np.float32), engine.zeros_f32(5 * D + 1)):
        with pytest.raises(ValueError, match="not rows of"):
            head.evaluate(x, np.zeros(5, np.uint32))
    assert np.isfinite(head.evaluate(np.zeros(5 * D, np.float32), np.zeros(5, np.uint32)))
