"""A cluster head: a softmax classifier over embedding rows, trained on labels.

The engine's ``assign`` labels rows by their nearest centroid. A head learns
those labels (or any others) by gradient: rows are layer-normalised and scored
against one prototype per cluster, and the norm's weights and the prototypes
take AdamW steps on the cross entropy. Started from the centroids it refines a
clustering; over another encoder's rows of the same items it carries the
clustering over to that encoder.

Run as ``python -m emeans_b200.head`` it clusters generated rows and trains a
head on the labels.
"""

from __future__ import annotations

import math
from typing import Optional

import numpy as np

import emeans_b200 as eb


class ClusterHead:
    """Layer norm, k prototypes and their AdamW states on one engine.

    Weights are f32 on the engine; ``eight_bit`` keeps the moments in 8 bits.
    ``prototypes`` (k x d) starts the head, for one from centroids; without it
    they are drawn at random. ``scale`` multiplies the scores (1 / temperature).
    """

    def __init__(self, engine: eb.Engine, d: int, k: int, prototypes=None,
                 scale: Optional[float] = None, weight_decay: float = 0.01,
                 eight_bit: bool = False, seed: int = 0):
        self.engine, self.d, self.k = engine, int(d), int(k)
        self.scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
        if prototypes is None:
            prototypes = np.random.default_rng(seed).standard_normal((k, d))
        prototypes = np.asarray(prototypes, np.float32)
        if prototypes.shape != (k, d):
            raise ValueError("prototypes must be k x d")
        self.weight = engine.upload_f32(np.ones(d, np.float32))
        self.bias = engine.zeros_f32(d)
        self.w = engine.upload_f32(prototypes)
        self.dweight, self.dbias = engine.zeros_f32(d), engine.zeros_f32(d)
        self.dw = engine.zeros_f32(k * d)

        def tensor(p, g, decay):
            states = eb.AdamW.states(engine, len(p), eight_bit)
            return eb.AdamWTensor(p=p, g=g, weight_decay=decay, **states)

        self.optimizer = eb.AdamW(engine, [tensor(self.weight, self.dweight, 0.0),
                                           tensor(self.bias, self.dbias, 0.0),
                                           tensor(self.w, self.dw, weight_decay)])
        self.dloss = engine.zeros_f32(1)
        self.steps = 0
        self._rows = -1
        self._last = None  # (losses, rows, labelled rows) of the last step

    def _room(self, n: int):
        """Per-row buffers for batches of up to n rows."""
        if n <= self._rows:
            return
        e, f = self.engine, self.engine.zeros_f32
        self.mean, self.rstd, self.lse = f(n), f(n), f(n)
        self.y, self.dy = f(n * self.d), f(n * self.d)
        # Losses of the steps and of other calls apart: ``last_loss`` reads the
        # former whatever was called in between.
        self.step_loss, self.loss = f(n), f(n)
        self.targets = e.zeros_u32(n)
        self._rows = n

    def _forward(self, x: eb.Buffer, n: int, labels, loss: str):
        labels = np.ascontiguousarray(labels, np.uint32)
        if labels.shape != (n,):
            raise ValueError("one label per row")
        self._room(n)
        e, d, loss = self.engine, self.d, getattr(self, loss)
        self.targets.write(0, labels)
        e.layer_norm(x, n, d, self.weight, self.bias, self.y, mean=self.mean, rstd=self.rstd)
        e.linear_cross_entropy(self.y, n, d, self.w, self.k, self.targets, loss, self.lse,
                               scale=self.scale)
        return loss, n, int((labels != eb.IGNORE).sum())

    def _buffer(self, x):
        """x on the engine, and its rows."""
        if not isinstance(x, eb.Buffer):
            x = np.asarray(x, np.float32)
            if x.ndim > 1 and x.shape[-1] != self.d:
                raise ValueError(f"rows of {x.shape[-1]} elements, the head's have {self.d}")
            x = self.engine.upload_f32(x)
        if len(x) % self.d:
            raise ValueError(f"{len(x)} elements are not rows of {self.d}")
        return x, len(x) // self.d

    @staticmethod
    def _mean(loss: eb.Buffer, n: int, kept: int) -> float:
        return float(loss.read(0, n).sum(dtype=np.float64)) / max(kept, 1)

    def step(self, x, labels, lr: float, beta1: float = 0.9, beta2: float = 0.999) -> None:
        """One gradient step on the mean loss of rows x (an f32 Buffer or host
        array, n x d) with ``labels`` (n; ``IGNORE`` for rows without one).
        Queued on the engine's stream; ``last_loss`` waits for it."""
        x, n = self._buffer(x)
        self._last = self._forward(x, n, labels, "step_loss")
        kept = self._last[2]
        e, d = self.engine, self.d
        self.dloss.write(0, [1.0 / max(kept, 1)])
        e.linear_cross_entropy_backward(self.y, n, d, self.w, self.k, self.targets, self.lse,
                                        self.dloss, self.dy, self.dw, scale=self.scale)
        e.layer_norm_backward(self.dy, x, n, d, self.weight, self.mean, self.rstd, None,
                              self.dweight, self.dbias)
        self.steps += 1
        self.optimizer.step(lr, self.steps, beta1=beta1, beta2=beta2)

    def last_loss(self) -> float:
        """The mean loss of the last ``step``'s labelled rows, before it."""
        if self._last is None:
            raise RuntimeError("no step has been taken")
        return self._mean(*self._last)

    def evaluate(self, x, labels) -> float:
        """The mean loss of rows x."""
        x, n = self._buffer(x)
        return self._mean(*self._forward(x, n, labels, "loss"))

    def predict(self, x) -> np.ndarray:
        """The best-scoring prototype of each row: the exact top-1 of the
        normalised rows against the prototypes."""
        x, n = self._buffer(x)
        self._room(n)
        e = self.engine
        e.layer_norm(x, n, self.d, self.weight, self.bias, self.y)
        labels, scores = e.zeros_u32(n), e.zeros_f32(n)
        e.top1(self.y, self.d, None, range(0, n), self.w, None, self.k, eb.IP, labels, scores)
        return labels.read()


def main():
    rng = np.random.default_rng(0)
    n, d, k = 20000, 64, 32
    means = rng.standard_normal((k, d))
    x = (means[rng.integers(0, k, n)] + 0.4 * rng.standard_normal((n, d))).astype(np.float32)
    with eb.Engine(0) as e:
        trained = e.train(x, eb.Config(d=d, k=k, seed=7))
        labels = np.asarray(trained.labels, np.uint32)
        head = ClusterHead(e, d, k)
        batch = 2000
        for epoch in range(10):
            order = rng.permutation(n)
            for at in range(0, n, batch):
                rows = order[at:at + batch]
                head.step(x[rows], labels[rows], lr=0.1)
            print(f"epoch {epoch}: loss {head.evaluate(x, labels):.4f}, "
                  f"agreement {np.mean(head.predict(x) == labels):.4f}")


if __name__ == "__main__":
    main()
