"""The training operators of a cluster head, as they are measured.

A head on top of embedding rows is trained against cluster labels: the rows
are layer-normalised, scored against one prototype per cluster under a softmax
cross entropy, and the prototypes and the norm's weights take an AdamW step.
Each case is one pass through one of these operators. `run` computes it in
plain torch operations (32 bits, rounded once at the end), or, with `own`, by
the engine's calls.
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = 0xFFFFFFFF   # target of a row that carries no label
EPS = 1e-5            # layer norm
BLOCK = 256           # elements that share a scale of the 8-bit states
LR, BETA1, BETA2, ADAM_EPS, DECAY, STEP = 1e-4, 0.9, 0.95, 1e-8, 0.01, 10


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One request's rows at serving: launch latency.
        {"name": "norm fwd 32x768 f32", "op": "norm", "backward": False, "rows": 32, "d": 768,
         "dtype": "f32"},
        # A whole bound data set normalised once.
        {"name": "norm fwd 200000x768 bf16", "op": "norm", "backward": False, "rows": 200000,
         "d": 768, "dtype": "bf16"},
        # A training batch of rows whose width fits no vector load.
        {"name": "norm bwd 16411x387 f32", "op": "norm", "backward": True, "rows": 16411, "d": 387,
         "dtype": "f32"},
        # The largest training batch.
        {"name": "norm bwd 131072x1024 bf16", "op": "norm", "backward": True, "rows": 131072,
         "d": 1024, "dtype": "bf16"},
        # A few rows scored against a large set of prototypes at serving.
        {"name": "ce fwd 8x65536x1024 bf16", "op": "ce", "backward": False, "n": 8, "k": 65536,
         "d": 1024, "dtype": "bf16"},
        # The smallest clustering: a mini-batch against a few dozen prototypes.
        {"name": "ce step 1000x32x64 f32", "op": "ce", "backward": True, "n": 1000, "k": 32,
         "d": 64, "dtype": "f32"},
        # The ordinary training batch.
        {"name": "ce step 16384x1024x768 bf16", "op": "ce", "backward": True, "n": 16384,
         "k": 1024, "d": 768, "dtype": "bf16"},
        # Full precision, every size odd.
        {"name": "ce step 3001x5003x385 f32", "op": "ce", "backward": True, "n": 3001, "k": 5003,
         "d": 385, "dtype": "f32"},
        # The largest set of prototypes, forward and gradients.
        {"name": "ce step 16384x65536x1024 bf16", "op": "ce", "backward": True, "n": 16384,
         "k": 65536, "d": 1024, "dtype": "bf16"},
        # The small head's three tensors: launch latency.
        {"name": "adamw 3 tensors f32", "op": "adamw", "tensors": 3, "total": 26112,
         "states": "f32"},
        # A head under an encoder: many tensors, matrices and vectors.
        {"name": "adamw 160 tensors f32", "op": "adamw", "tensors": 160, "total": 120000000,
         "states": "f32"},
        # The same kind of model, larger, with its states in 8 bits and 16-bit copies of its weights.
        {"name": "adamw 160 tensors fp8", "op": "adamw", "tensors": 160, "total": 400000000,
         "states": "fp8"},
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    return min(v | 1, hi) if rng.random() < 0.4 else v


def draw(rng):
    op = rng.choice(["norm", "ce", "ce", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        d = _log_int(rng, 2, 4096)
        rows = _log_int(rng, 1, max(2, min(200000, 131072 * 1024 * 2 // (d * SIZE[dtype]))))
        return {"op": op, "backward": rng.random() < 0.5, "rows": rows, "d": d, "dtype": dtype}
    if op == "ce":
        most = 16384 * 65536 * 1024 // (8 if dtype == "f32" else 1)
        while True:
            n, k, d = _log_int(rng, 1, 16384), _log_int(rng, 2, 65536), _log_int(rng, 4, 1024)
            if n * k * d <= most:
                return {"op": op, "backward": rng.random() < 0.7, "n": n, "k": k, "d": d,
                        "dtype": dtype}
    tensors = _log_int(rng, 1, 200)
    return {"op": op, "tensors": tensors, "total": max(tensors, _log_int(rng, 1000, 120000000)),
            "states": rng.choice(["f32", "fp8", "bf16 weights"])}


def _sizes(case):
    """The tensors' lengths: spread over the logarithm, odd ones among them, `total` in all."""
    rng = random.Random(case["tensors"] * 1000003 + case["total"])
    part = [math.exp(rng.uniform(0.0, 9.0)) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * p / sum(part))) for p in part]


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"norm": _prepare_norm, "ce": _prepare_ce, "adamw": _prepare_adamw}[case["op"]](case, g)
    s["case"] = case
    if own:
        _hold(s)
    return s


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_norm(case, g):
    rows, d, t = case["rows"], case["d"], DTYPES[case["dtype"]]
    # Rows of an encoder: each with its own spread and offset.
    x = _normal(g, rows, d) * (0.2 + 2.0 * torch.rand(rows, 1, generator=g, device="cuda"))
    x = (x + 0.5 * _normal(g, rows, 1)).to(t)
    s = {"x": x, "weight": 1.0 + 0.1 * _normal(g, d), "bias": 0.1 * _normal(g, d),
         "y": torch.empty_like(x), "mean": torch.empty(rows, device="cuda"),
         "rstd": torch.empty(rows, device="cuda")}
    if case["backward"]:
        s["dy"] = _normal(g, rows, d).to(t)
        f = x.float()
        s["mean"] = f.mean(1)
        s["rstd"] = (f - s["mean"][:, None]).square().mean(1).add(EPS).rsqrt()
        s["dx"] = torch.empty_like(x)
        s["dweight"] = torch.empty(d, device="cuda")
        s["dbias"] = torch.empty(d, device="cuda")
    return s


def _prepare_ce(case, g):
    n, k, d, t = case["n"], case["k"], case["d"], DTYPES[case["dtype"]]
    # Unit prototypes; rows that lean towards their own prototype by differing amounts.
    w = _normal(g, k, d)
    w = w / w.norm(dim=1, keepdim=True)
    target = torch.randint(0, k, (n,), generator=g, device="cuda")
    lean = 8.0 * torch.rand(n, 1, generator=g, device="cuda")
    x = (_normal(g, n, d) + lean * w[target]).to(t)
    none = torch.rand(n, generator=g, device="cuda") < 0.05
    kept = int(n - none.sum())
    target = torch.where(none, torch.full_like(target, IGNORE), target)
    # The mean over the labelled rows; 16-bit floats of the small range train on a scaled loss.
    row = 1.0 if case["dtype"] == "f16" else 1.0 / max(kept, 1)
    s = {"x": x, "w": w.to(t), "target": target.to(torch.uint32), "scale": 1.5,
         "loss": torch.empty(n, device="cuda"), "lse": torch.empty(n, device="cuda")}
    if case["backward"]:
        s["dloss"] = torch.full((1,), row, device="cuda")
        s["dx"] = torch.empty_like(x)
        s["dw"] = torch.empty_like(s["w"])
    return s


def _prepare_adamw(case, g):
    sizes = _sizes(case)
    at, end = [], 0
    for n in sizes:  # every tensor starts on blocks of its own, and so do its scales; the gaps hold zeros
        at.append(end)
        end += -(-n // (4 * BLOCK)) * (4 * BLOCK)
    live = torch.zeros(end, device="cuda")
    for a, n in zip(at, sizes):
        live[a:a + n] = 1.0
    states, s = case["states"], {"sizes": sizes, "at": at}
    s["p"] = 0.05 * _normal(g, end) * live
    s["g"] = 1e-3 * _normal(g, end) * live
    m = 5e-4 * _normal(g, end) * live
    v = 1e-6 * _normal(g, end).square() * live
    if states == "fp8":
        s["g"] = s["g"].to(torch.bfloat16)
        s["copy"] = s["p"].to(torch.bfloat16)
        s["m"], s["m_scale"] = _to_fp8(m)
        s["v"], s["v_scale"] = _to_fp8(v.sqrt())
    else:
        s["m"], s["v"] = m, v
        if states == "bf16 weights":
            s["p"], s["g"] = s["p"].to(torch.bfloat16), s["g"].to(torch.bfloat16)
    return s


def _engine():
    """One engine for the process, on torch's current stream."""
    import emeans_b200 as eb

    if not _engines:
        _engines.append(eb.Engine(0, stream=torch.cuda.current_stream().cuda_stream))
    return _engines[0]


_engines = []


def _hold(s):
    """The engine's buffers over the state's tensors, and the optimizer's plan."""
    import emeans_b200 as eb

    e = _engine()
    s["engine"] = e
    if s["case"]["op"] != "adamw":
        s["buf"] = {k: e.wrap(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
        return

    def part(name, a, n):
        return e.wrap(s[name][a:a + n]) if name in s else None

    def scales(name, a, n):
        a, n = a // BLOCK, -(-n // BLOCK)
        return e.wrap(s[name][a:a + n]) if name in s else None

    s["plan"] = eb.AdamW(e, [eb.AdamWTensor(
        p=part("p", a, n), g=part("g", a, n), m=part("m", a, n), v=part("v", a, n),
        m_scale=scales("m_scale", a, n), v_scale=scales("v_scale", a, n), copy=part("copy", a, n),
        weight_decay=DECAY) for a, n in zip(s["at"], s["sizes"])])


# ---------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)[s["case"]["op"]](s)


def _own_norm(s):
    e, b, rows, d = s["engine"], s["buf"], s["case"]["rows"], s["case"]["d"]
    if s["case"]["backward"]:
        e.layer_norm_backward(b["dy"], b["x"], rows, d, b["weight"], b["mean"], b["rstd"],
                              b["dx"], b["dweight"], b["dbias"])
        return {"dx": s["dx"], "dweight": s["dweight"], "dbias": s["dbias"]}
    e.layer_norm(b["x"], rows, d, b["weight"], b["bias"], b["y"], eps=EPS, mean=b["mean"],
                 rstd=b["rstd"])
    return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}


def _plain_norm(s):
    x = s["x"].float()
    if s["case"]["backward"]:
        dy = s["dy"].float()
        u = (x - s["mean"][:, None]) * s["rstd"][:, None]
        h = dy * s["weight"]
        dx = (h - h.mean(1, keepdim=True) - u * (h * u).mean(1, keepdim=True)) * s["rstd"][:, None]
        return {"dx": dx.to(s["x"].dtype), "dweight": (dy * u).sum(0), "dbias": dy.sum(0)}
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = (c.square().mean(1) + EPS).rsqrt()
    y = c * rstd[:, None] * s["weight"] + s["bias"]
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _own_ce(s):
    e, b, c = s["engine"], s["buf"], s["case"]
    e.linear_cross_entropy(b["x"], c["n"], c["d"], b["w"], c["k"], b["target"], b["loss"],
                           b["lse"], scale=s["scale"])
    out = {"loss": s["loss"], "lse": s["lse"]}
    if c["backward"]:
        e.linear_cross_entropy_backward(b["x"], c["n"], c["d"], b["w"], c["k"], b["target"],
                                        b["lse"], b["dloss"], b["dx"], b["dw"], scale=s["scale"])
        out.update(dx=s["dx"], dw=s["dw"])
    return out


def _plain_ce(s):
    x, w, t = s["x"].float(), s["w"].float(), s["target"].to(torch.int64)
    live = t != IGNORE
    t = torch.where(live, t, torch.zeros_like(t))[:, None]
    z = (x @ w.T).mul_(s["scale"])
    top = z.amax(1, keepdim=True)
    lse = (z - top).exp_().sum(1).log() + top[:, 0]
    loss = torch.where(live, lse - z.gather(1, t)[:, 0], torch.zeros_like(lse))
    out = {"loss": loss, "lse": lse}
    if s["case"]["backward"]:
        p = z.sub_(lse[:, None]).exp_()
        p.scatter_add_(1, t, torch.full_like(t, -1, dtype=torch.float32))
        p.mul_(torch.where(live, s["dloss"] * s["scale"], torch.zeros_like(lse))[:, None])
        out["dx"] = (p @ w).to(s["x"].dtype)
        out["dw"] = (p.T @ x).to(s["w"].dtype)
    return out


def _adamw_outputs(s):
    return {k: s[k] for k in ("p", "m", "v", "m_scale", "v_scale", "copy") if k in s}


def _own_adamw(s):
    s["plan"].step(LR, STEP, beta1=BETA1, beta2=BETA2, eps=ADAM_EPS)
    return _adamw_outputs(s)


def _to_fp8(v):
    """Blocks of 256 values as 8-bit floats (e4m3) and one 32-bit scale each."""
    b = v.reshape(-1, BLOCK)
    scale = b.abs().amax(1) * (1.0 / 448.0)
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    q = (b * inv[:, None]).clamp_(-448.0, 448.0)
    return q.to(torch.float8_e4m3fn).reshape(-1), scale


def _root_to_fp8(r):
    """_to_fp8 for the second moment's root: what is above zero stays above zero."""
    q, scale = _to_fp8(r)
    least = torch.full_like(r, 2.0 ** -9)
    return torch.where(r > 0, torch.maximum(q.float(), least), q.float()).to(q.dtype), scale


def _from_fp8(q, scale):
    return (q.float().reshape(-1, BLOCK) * scale[:, None]).reshape(-1)


def _plain_adamw(s):
    eight = "m_scale" in s
    p, g = s["p"].float(), s["g"].float()
    m = _from_fp8(s["m"], s["m_scale"]) if eight else s["m"]
    v = _from_fp8(s["v"], s["v_scale"]).square() if eight else s["v"]
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    root = v.sqrt()
    size, fix = LR / (1.0 - BETA1 ** STEP), 1.0 / math.sqrt(1.0 - BETA2 ** STEP)
    p = p * (1.0 - LR * DECAY) - m / (root * fix + ADAM_EPS) * size
    s["p"].copy_(p)
    if eight:
        q, scale = _to_fp8(m)
        s["m"].copy_(q), s["m_scale"].copy_(scale)
        q, scale = _root_to_fp8(root)
        s["v"].copy_(q), s["v_scale"].copy_(scale)
        s["copy"].copy_(p)
    else:
        s["m"].copy_(m), s["v"].copy_(v)
    return _adamw_outputs(s)


_run_plain = {"norm": _plain_norm, "ce": _plain_ce, "adamw": _plain_adamw}
_run_own = {"norm": _own_norm, "ce": _own_ce, "adamw": _own_adamw}


# ---------------------------------------------------------------- the work of a pass

def work(case):
    if case["op"] == "norm":
        n, d, e = case["rows"], case["d"], SIZE[case["dtype"]]
        if case["backward"]:  # dy, x and the statistics in; dx and two weight gradients out
            return {"bytes": 3 * n * d * e + 8 * n + 12 * d, "flops": 13 * n * d}
        return {"bytes": 2 * n * d * e + 8 * n + 8 * d, "flops": 8 * n * d}
    if case["op"] == "ce":
        n, k, d, e = case["n"], case["k"], case["d"], SIZE[case["dtype"]]
        if case["backward"]:  # the scores and the two gradients' products
            return {"bytes": 2 * (n + k) * d * e + 12 * n, "flops": 6 * n * k * d}
        return {"bytes": (n + k) * d * e + 12 * n, "flops": 2 * n * k * d}
    n = sum(_sizes(case))
    each = {"f32": 28, "fp8": 8 + 2 + 4 + 2 + 16 / BLOCK, "bf16 weights": 4 + 2 + 16}[case["states"]]
    return {"bytes": each * n, "flops": 16 * n}


# ---------------------------------------------------------------- the values in 64 bits

def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "norm":
        return _exact_norm(case, _prepare_norm(case, g))
    if case["op"] == "ce":
        return _exact_ce(case, _prepare_ce(case, g))
    return _exact_adamw(case, _prepare_adamw(case, g))


def _exact_norm(case, s):
    x, w = s["x"].double(), s["weight"].double()
    if not case["backward"]:
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = 1.0 / torch.sqrt(var + EPS)
        y = torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], w)
        return {"y": y, "mean": mean, "rstd": rstd}
    dy, r = s["dy"].double(), s["rstd"].double()[:, None]
    u = (x - s["mean"].double()[:, None]) * r
    a, d = dy * w, case["d"]
    dx = (r / d) * (d * a - a.sum(1, keepdim=True) - u * (a * u).sum(1, keepdim=True))
    return {"dx": dx, "dweight": torch.einsum("nd,nd->d", dy, u), "dbias": dy.sum(0)}


def _exact_ce(case, s):
    n, k = case["n"], case["k"]
    x, w = s["x"].double(), s["w"].double()
    target = s["target"].to(torch.int64)
    loss, lse = x.new_zeros(n), x.new_zeros(n)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    step = max(1, (1 << 28) // k)
    for a in range(0, n, step):
        b = min(n, a + step)
        z = s["scale"] * (x[a:b] @ w.T)
        lse[a:b] = torch.logsumexp(z, 1)
        rows = torch.nonzero(target[a:b] != IGNORE)[:, 0]
        cols = target[a:b][rows]
        loss[a + rows] = lse[a + rows] - z[rows, cols]
        if case["backward"]:
            p = torch.zeros_like(z)
            p[rows] = torch.softmax(z[rows], 1)
            p[rows, cols] -= 1.0
            p *= s["dloss"].double() * s["scale"]
            dx[a:b] = p @ w
            dw += p.T @ x[a:b]
    out = {"loss": loss, "lse": lse}
    if case["backward"]:
        out.update(dx=dx, dw=dw)
    return out


def _exact_adamw(case, s):
    def scaled(v):
        scale = v.reshape(-1, BLOCK).abs().amax(1) / 448.0
        return (v.reshape(-1, BLOCK) / scale.clamp_min(1e-300)[:, None]).reshape(-1), scale

    eight, p, g = "m_scale" in s, s["p"].double(), s["g"].double()
    m, v = s["m"].double(), s["v"].double()
    if eight:
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    p = p - LR * DECAY * p
    p = p - LR * (m / (1.0 - BETA1 ** STEP)) / ((v / (1.0 - BETA2 ** STEP)).sqrt() + ADAM_EPS)
    if not eight:
        return {"p": p, "m": m, "v": v}
    out = {"p": p, "copy": p}
    out["m"], out["m_scale"] = scaled(m)
    out["v"], out["v_scale"] = scaled(v.sqrt())
    return out
