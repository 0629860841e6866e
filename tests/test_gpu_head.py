"""The cluster head: the training operators run together on the engine."""

import numpy as np
import pytest
import torch

import emeans_b200 as eb
from emeans_b200.head import ClusterHead
from tests.helpers import mixture

pytestmark = pytest.mark.gpu


def plain_head(x, labels, w0, scale, lr, steps, batch):
    """The same head in plain 64-bit torch: its loss and its rows' predictions."""
    d = x.shape[1]
    X, T = torch.from_numpy(x).double(), torch.from_numpy(labels.astype(np.int64))
    w = torch.from_numpy(w0).double().requires_grad_()
    g, b = torch.ones(d).double().requires_grad_(), torch.zeros(d).double().requires_grad_()
    opt = torch.optim.AdamW([{"params": [g, b], "weight_decay": 0.0},
                             {"params": [w], "weight_decay": 0.01}], lr=lr, eps=1e-8)

    def scores(rows):
        return scale * torch.nn.functional.layer_norm(rows, (d,), g, b) @ w.T

    for i in range(steps):
        lo = i % (4000 // batch) * batch
        loss = torch.nn.functional.cross_entropy(scores(X[lo:lo + batch]), T[lo:lo + batch])
        opt.zero_grad()
        loss.backward()
        opt.step()
    with torch.no_grad():
        z = scores(X)
        return (float(torch.nn.functional.cross_entropy(z[:4000], T[:4000])),
                z.argmax(1).numpy().astype(np.uint32))


@pytest.mark.parametrize("eight_bit", [False, True])
def test_head_learns_the_engines_own_labels(engine, eight_bit):
    """A head trained on a clustering's labels gives them back on held-out
    rows as well as the same head trained in 64 bits does (8-bit moments: to a
    few hundredths of the loss)."""
    n, d, k = 6000, 32, 12
    x = mixture(n, d, k, 0.2, False, 3)
    tr = engine.train(x[:4000], eb.Config(d=d, k=k, seed=5))
    labels, _ = engine.assign(x, d, tr.centroids, eb.L2)
    head = ClusterHead(engine, d, k, eight_bit=eight_bit, seed=1)
    loss, want = plain_head(x, labels, head.w.read().reshape(k, d), head.scale, 3e-2, 60, 1000)
    first = head.evaluate(x[:4000], labels[:4000])
    for i in range(60):
        lo = i % 4 * 1000
        head.step(x[lo:lo + 1000], labels[lo:lo + 1000], lr=3e-2)
    last = head.evaluate(x[:4000], labels[:4000])
    assert last < 0.5 * first and abs(last - loss) <= 0.05 * first
    agreed, plain = np.mean(head.predict(x[4000:]) == labels[4000:]), np.mean(want[4000:] == labels[4000:])
    assert agreed >= plain - 0.01


def test_head_steps_follow_a_64_bit_run(engine):
    """Five steps against the same steps in 64 bits. Adam divides by the
    gradient's own size, so where a first gradient is near zero its sign may
    differ: those elements move by lr a step either way, and are few."""
    n, d, k, lr = 300, 24, 17, 1e-2
    rng = np.random.default_rng(2)
    x = rng.standard_normal((n, d)).astype(np.float32)
    labels = rng.integers(0, k, n).astype(np.uint32)
    labels[::7] = eb.IGNORE
    head = ClusterHead(engine, d, k, seed=4, weight_decay=0.05)
    X = torch.from_numpy(x).double()
    w = torch.from_numpy(head.w.read().reshape(k, d)).double().requires_grad_()
    g, b = torch.ones(d).double().requires_grad_(), torch.zeros(d).double().requires_grad_()
    keep = torch.from_numpy(labels != eb.IGNORE)
    t = torch.from_numpy(labels.astype(np.int64))[keep]
    opt = torch.optim.AdamW([{"params": [g, b], "weight_decay": 0.0},
                             {"params": [w], "weight_decay": 0.05}], lr=lr, eps=1e-8)
    for _ in range(5):
        head.step(x, labels, lr)
        y = torch.nn.functional.layer_norm(X, (d,), g, b)
        loss = torch.nn.functional.cross_entropy(head.scale * y[keep] @ w.T, t)
        assert abs(head.last_loss() - float(loss)) < 1e-4
        opt.zero_grad()
        loss.backward()
        opt.step()
    off = np.abs(head.w.read().reshape(k, d) - w.detach().numpy())
    assert off.max() <= 2 * 5 * lr and np.mean(off > 1e-4) < 0.01
    assert np.mean(np.abs(head.weight.read() - g.detach().numpy()) > 1e-4) < 0.1


def test_head_refusals(engine):
    with pytest.raises(ValueError, match="k x d"):
        ClusterHead(engine, 8, 4, prototypes=np.zeros((3, 8)))
    head = ClusterHead(engine, 8, 4)
    with pytest.raises(ValueError, match="one label per row"):
        head.step(np.zeros((5, 8), np.float32), np.zeros(4, np.uint32), lr=1e-3)
