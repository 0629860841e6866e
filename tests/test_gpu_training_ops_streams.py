"""The cross entropy and AdamW on the caller's streams: in order with the
caller's own work there with no wait in between, and two engines at once on two
streams, each with its own scratch."""

import pytest
import torch

import emeans_b200 as eb
from tests.test_gpu_training_ops import gen, randn

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, 300, 200, 130), (torch.bfloat16, 500, 700, 264), (torch.float32, 8, 900, 72),
         (torch.float32, 100, 40, 32)]


class Step:
    """Buffers of one loss, its gradients and an AdamW step of the prototypes."""

    def __init__(self, e, dtype, n, k, d):
        self.e, self.n, self.k, self.d = e, n, k, d
        f = dict(device="cuda")
        self.x, self.dx = torch.empty(n, d, dtype=dtype, **f), torch.empty(n, d, dtype=dtype, **f)
        self.p, self.w = torch.empty(k, d, **f), torch.empty(k, d, dtype=dtype, **f)
        self.dw = torch.empty(k, d, dtype=dtype, **f)
        self.m, self.v = torch.empty(k, d, **f), torch.empty(k, d, **f)
        self.t = torch.empty(n, dtype=torch.int32, **f)
        self.loss, self.lse, self.g = torch.empty(n, **f), torch.empty(n, **f), torch.empty(n, **f)
        self.all = [self.loss, self.lse, self.dx, self.dw, self.p, self.m, self.v]
        b = {q: e.wrap(v) for q, v in vars(self).items() if isinstance(v, torch.Tensor)}
        copy = {"copy": b["w"]} if dtype == torch.bfloat16 else {}
        self.b = b
        self.plan = eb.AdamW(e, [eb.AdamWTensor(p=b["p"], g=b["dw"], m=b["m"], v=b["v"], weight_decay=0.01, **copy)])

    def fill(self, seed):
        g = gen(seed)
        self.x.copy_(randn(g, self.n, self.d))
        self.p.copy_(0.3 * randn(g, self.k, self.d))
        self.w.copy_(self.p)
        self.t.copy_(torch.randint(0, self.k, (self.n,), generator=g, device="cuda"))
        self.g.copy_(randn(g, self.n))
        self.m.zero_(), self.v.zero_()

    def run(self, seed):
        self.fill(seed)
        b, a = self.b, (self.n, self.d)
        self.e.linear_cross_entropy(b["x"], *a, b["w"], self.k, b["t"], b["loss"], b["lse"])
        self.e.linear_cross_entropy_backward(b["x"], *a, b["w"], self.k, b["t"], b["lse"], b["g"],
                                             b["dx"], b["dw"])
        self.plan.step(lr=1e-2, step=1)
        return [v.clone() for v in self.all]


def finish(steps, engines):
    for s in steps:
        s.plan.free()
        for v in s.b.values():
            v.free()
    for e in engines:
        e.close()


@pytest.mark.parametrize("dtype,n,k,d", TYPES)
def test_in_order_on_a_side_stream(dtype, n, k, d):
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        e = eb.Engine(0, stream=side.cuda_stream)
        s = Step(e, dtype, n, k, d)
        want = []
        for seed in range(4):  # one at a time
            want.append(s.run(seed))
            side.synchronize()
        got = [s.run(seed) for seed in range(4)]
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
        if dtype == torch.float32:
            s.fill(3)
            z = s.x.double() @ s.w.double().T
            t = s.t.long()[:, None]
            loss = torch.logsumexp(z, 1) - z.gather(1, t)[:, 0]
            assert float((got[3][0].double() - loss).abs().max()) < 1e-4
        e.sync()
        finish([s], [e])
    side.synchronize()


def test_two_engines_at_once_on_two_streams():
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    engines, steps = [], []
    for st, (dtype, n, k, d) in zip(streams, [(torch.float32, 700, 1100, 264), (torch.bfloat16, 900, 3000, 136)]):
        with torch.cuda.stream(st):
            engines.append(eb.Engine(0, stream=st.cuda_stream))
            steps.append(Step(engines[-1], dtype, n, k, d))
    want = []
    for st, s in zip(streams, steps):
        with torch.cuda.stream(st):
            want.append([s.run(seed) for seed in range(6)])
        st.synchronize()
    got = [[], []]
    for seed in range(6):
        for i, (st, s) in enumerate(zip(streams, steps)):
            with torch.cuda.stream(st):
                got[i].append(s.run(seed))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert all(torch.equal(u, v) for u, v in zip(p, q))
    finish(steps, engines)
