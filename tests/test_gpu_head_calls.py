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
