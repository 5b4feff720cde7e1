"""Operators of the training step that are measured one by one: layer normalisation (forward,
backward, with the residual add), the Newton-Schulz orthogonalisation of matrices, and the
Muon update that uses it.

``listed()`` are fixed cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes a
case's inputs on the GPU, ``run`` is one pass as a user's program calls it (``own``) or the same
mathematics in plain torch operations, ``exact`` the definition in 64 bits, ``work`` the bytes
and operations a pass cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

LN_EPS = 1e-5
NS_EPS = 1e-7
NS_STEPS = 5
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
# learning rate and weight decay of the 100M configuration; usual momentum
LR, WEIGHT_DECAY, MOMENTUM = 3e-4, 0.1, 0.95
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def _ln(name, mode, rows, n, dtype):
    return {"name": name, "op": "layernorm", "mode": mode, "rows": rows, "n": n, "dtype": dtype}


def _ns(name, batch, m, n, dtype, rank=0):
    return {"name": name, "op": "orthogonalize", "batch": batch, "m": m, "n": n, "dtype": dtype, "rank": rank}


def _muon(name, layers, d, d_kv, d_ff, rank=0):
    return {"name": name, "op": "muon", "layers": layers, "d": d, "d_kv": d_kv, "d_ff": d_ff, "rank": rank}


def listed():
    return [
        # one token of a width-4096 model while generating: latency
        _ln("ln_fwd_1x4096_bf16", "fwd", 1, 4096, "bf16"),
        # an evaluation pass of the 100M model over 4 packs of 2048 tokens
        _ln("ln_fwd_8192x768_fp32", "fwd", 8192, 768, "fp32"),
        # the 100M model's training step: fp32 residual stream plus the bf16 projection, then the norm
        _ln("ln_add_8192x768", "add", 8192, 768, "fp32"),
        # a long batch of a width-4096 model with bf16 activations, forward and backward
        _ln("ln_train_16384x4096_bf16", "train", 16384, 4096, "bf16"),
        # a ragged batch at an odd width: no row but the first is 16-byte aligned
        _ln("ln_train_4001x1409_fp32", "train", 4001, 1409, "fp32"),
        # one K or V projection of the 100M model alone: latency
        _ns("ns_1x256x768", 1, 256, 768, "fp32"),
        # every Q and O projection of the 100M model
        _ns("ns_24x768x768", 24, 768, 768, "fp32"),
        # the gate projections of the 100M model (more rows than columns), bf16 momenta, a strong low-rank part
        _ns("ns_12x2048x768_bf16", 12, 2048, 768, "bf16", 16),
        # odd sizes and few tokens behind the gradient: five matrices of rank 24 plus noise
        _ns("ns_5x333x1407_rank24", 5, 333, 1407, "fp32", 24),
        # all hidden matrices of the 49M model (8 layers, short documents)
        _muon("muon_49m", 8, 512, 256, 1408),
        # all hidden matrices of the 100M model
        _muon("muon_100m", 12, 768, 256, 2048, 64),
        # eight layers of the 1.1B model
        _muon("muon_1b_8layers", 8, 2048, 256, 5632),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(("layernorm", "orthogonalize", "muon"))
    if op == "layernorm":
        mode = rng.choice(("fwd", "train", "add"))
        n = _log(rng, 32, 8192)
        if rng.random() < 0.5:
            n = -(-n // 32) * 32
        rows = _log(rng, 1, min(32768, 16384 * 4096 // n))
        return {"op": op, "mode": mode, "rows": rows, "n": n,
                "dtype": "fp32" if mode == "add" else rng.choice(("fp32", "bf16"))}
    if op == "orthogonalize":
        m, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.5:
            m, n = -(-m // 16) * 16, -(-n // 16) * 16
        small, large = min(m, n), max(m, n)
        one = 4 * small * small * large + 2 * small**3
        batch = _log(rng, 1, max(1, min(48, 10**12 // one)))
        return {"op": op, "batch": batch, "m": m, "n": n, "dtype": rng.choice(("fp32", "bf16")),
                "rank": rng.choice((0, 0, max(1, small // 16)))}
    d = 64 * rng.randint(4, 24)
    return {"op": op, "layers": rng.randint(1, 8), "d": d, "d_kv": max(64, d // rng.choice((1, 2, 4)) // 64 * 64),
            "d_ff": 8 * rng.randint(d // 4, d // 2), "rank": rng.choice((0, 32))}


def _muon_shapes(c):
    d, kv, ff = c["d"], c["d_kv"], c["d_ff"]
    return {"q": (d, d), "k": (kv, d), "v": (kv, d), "o": (d, d), "gate": (ff, d), "up": (ff, d), "down": (d, ff)}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _matrices(gen, batch, m, n, rank):
    """Gradients of linear layers: noise, plus ``rank`` common directions ten times as strong."""
    dev = gen.device
    g = torch.randn(batch, m, n, generator=gen, device=dev)
    if rank:
        u = torch.randn(batch, m, rank, generator=gen, device=dev)
        v = torch.randn(batch, rank, n, generator=gen, device=dev)
        g = g + torch.bmm(u, v) * (10.0 / rank**0.5)
    return g * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = gen.device
    op = case["op"]
    if op == "layernorm":
        rows, n, dt = case["rows"], case["n"], _DTYPES[case["dtype"]]

        def rand(*shape):
            return torch.randn(*shape, generator=gen, device=dev)

        # a residual stream: a common offset and a few channels far larger than the rest
        x = rand(rows, n) + 0.25
        x[:, :: max(1, n // 5)] *= 8.0
        s = {"op": op, "mode": case["mode"], "x": x.to(dt), "w": 1.0 + 0.1 * rand(n), "b": 0.1 * rand(n)}
        if case["mode"] == "add":
            s["delta"] = rand(rows, n).to(torch.bfloat16)
            s["dsum"] = rand(rows, n)
            s["dy"] = rand(rows, n).to(torch.bfloat16)
        elif case["mode"] == "train":
            s["dy"] = rand(rows, n).to(dt)
        if case["mode"] != "fwd":
            for k in ("x", "w", "b", "delta"):
                if k in s:
                    s[k].requires_grad_(True)
        return s
    if op == "orthogonalize":
        g = _matrices(gen, case["batch"], case["m"], case["n"], case["rank"])
        return {"op": op, "g": g.to(_DTYPES[case["dtype"]])}
    layers = case["layers"]
    shapes = _muon_shapes(case)
    p = [0.02 * torch.randn(layers, m, n, generator=gen, device=dev) for m, n in shapes.values()]
    g = [_matrices(gen, layers, m, n, case["rank"]) for m, n in shapes.values()]
    mom = [0.3 * _matrices(gen, layers, m, n, case["rank"]) for m, n in shapes.values()]
    return {"op": op, "p": p, "g": g, "m": mom}


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    return {"layernorm": _run_layernorm, "orthogonalize": _run_orthogonalize, "muon": _run_muon}[state["op"]](state)


def _run_layernorm(s):
    if own:
        from packbalance_b200.ops.layernorm import add_layernorm, layernorm

        if s["mode"] == "fwd":
            return layernorm(s["x"], s["w"], s["b"], LN_EPS)
        if s["mode"] == "train":
            y = layernorm(s["x"], s["w"], s["b"], LN_EPS)
            return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"]))
        total, y = add_layernorm(s["x"], s["delta"], s["w"], s["b"], LN_EPS)
        grads = torch.autograd.grad((total, y), (s["x"], s["delta"], s["w"], s["b"]), (s["dsum"], s["dy"]))
        return (total.detach(), y.detach(), *grads)
    with torch.no_grad():
        x, w, b = s["x"].float(), s["w"], s["b"]
        if s["mode"] == "add":
            x = x + s["delta"].float()
        centred = x - x.mean(-1, keepdim=True)
        rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + LN_EPS)
        xhat = centred * rstd
        y = (xhat * w + b).to(torch.bfloat16 if s["mode"] == "add" else s["x"].dtype)
        if s["mode"] == "fwd":
            return y
        dy = s["dy"].float()
        dw, db = (dy * xhat).sum(0), dy.sum(0)
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        if s["mode"] == "train":
            return y, dx.to(s["x"].dtype), dw, db
        dx = dx + s["dsum"]
        return x, y, dx, dx.to(torch.bfloat16), dw, db


def _plain_newton_schulz(u):
    """Five products a X + (b A + c A A) X with A = X X^T, from X = u / (|u| + eps), in 32 bits."""
    a, b, c = NS_COEFFICIENTS
    x = u.float()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(NS_STEPS):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


def _run_orthogonalize(s):
    if own:
        from packbalance_b200.ops.muon import orthogonalize

        return orthogonalize(s["g"])
    return _plain_newton_schulz(s["g"]).to(torch.bfloat16).contiguous()


def _run_muon(s):
    if own:
        from packbalance_b200.ops.muon import muon_update_

        muon_update_(s["p"], s["g"], s["m"], lr=LR, momentum=MOMENTUM, weight_decay=WEIGHT_DECAY)
        return {"p": s["p"], "m": s["m"]}
    for p, g, m in zip(s["p"], s["g"], s["m"]):
        m.mul_(MOMENTUM).add_(g, alpha=1.0 - MOMENTUM)
        o = _plain_newton_schulz(g * (1.0 - MOMENTUM) + m * MOMENTUM)
        p.mul_(1.0 - LR * WEIGHT_DECAY).sub_(o, alpha=LR * 0.2 * max(p.shape[-2:]) ** 0.5)
    return {"p": s["p"], "m": s["m"]}


# ---------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if s["op"] == "layernorm":
            return _exact_layernorm(s)
        if s["op"] == "orthogonalize":
            return _polar(s["g"].double())
        out = {"p": [], "m": []}
        for p, g, m in zip(s["p"], s["g"], s["m"]):
            p, g, m = p.double(), g.double(), m.double()
            m = m + (1.0 - MOMENTUM) * (g - m)
            step = _polar(g + MOMENTUM * (m - g))
            out["p"].append(p - LR * (WEIGHT_DECAY * p + 0.2 * math.sqrt(max(p.shape[1], p.shape[2])) * step))
            out["m"].append(m)
        return out


def _exact_layernorm(s):
    t = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    x = t["x"] + t["delta"] if s["mode"] == "add" else t["x"]
    n = x.shape[1]
    mean = x.sum(1, keepdim=True) / n
    std = torch.sqrt(((x - mean) ** 2).sum(1, keepdim=True) / n + LN_EPS)
    z = (x - mean) / std
    y = z * t["w"] + t["b"]
    if s["mode"] == "fwd":
        return y
    dz = t["dy"] * t["w"]
    dx = (dz - dz.sum(1, keepdim=True) / n - z * ((dz * z).sum(1, keepdim=True) / n)) / std
    dw, db = (t["dy"] * z).sum(0), t["dy"].sum(0)
    if s["mode"] == "train":
        return y, dx, dw, db
    dx = dx + t["dsum"]
    return x, y, dx, dx, dw, db


def _polar(u):
    """The same five steps on the smaller side's Gram matrix, one matrix at a time, in 64 bits."""
    a, b, c = NS_COEFFICIENTS
    out = torch.empty_like(u)
    for i, x in enumerate(u):
        x = x / (torch.linalg.matrix_norm(x) + NS_EPS)
        for _ in range(NS_STEPS):
            if x.shape[0] <= x.shape[1]:
                gram = x @ x.T
                x = a * x + b * (gram @ x) + c * (gram @ (gram @ x))
            else:
                gram = x.T @ x
                x = a * x + b * (x @ gram) + c * ((x @ gram) @ gram)
        out[i] = x
    return out


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def _ns_flops(batch, m, n):
    # per step: the Gram matrix and its square have one half each that symmetry gives, then one full product
    small, large = min(m, n), max(m, n)
    return batch * NS_STEPS * (small * (small + 1) * large + small * (small + 1) * small + 2 * small * small * large)


def work(case):
    if case["op"] == "layernorm":
        rows, n = case["rows"], case["n"]
        e = 4 if case["dtype"] == "fp32" else 2
        if case["mode"] == "fwd":
            return {"bytes": rows * n * 2 * e + 8 * n, "flops": 8 * rows * n}
        if case["mode"] == "train":  # x and dy in, y and dx out, w, b, dw, db
            return {"bytes": rows * n * 4 * e + 16 * n, "flops": 22 * rows * n}
        # x, delta, dsum, dy in; sum, y, dx in both types out
        return {"bytes": rows * n * (4 + 2 + 4 + 2 + 4 + 2 + 4 + 2) + 16 * n, "flops": 24 * rows * n}
    if case["op"] == "orthogonalize":
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["batch"] * case["m"] * case["n"] * (e + 2),
                "flops": _ns_flops(case["batch"], case["m"], case["n"])}
    shapes = _muon_shapes(case).values()
    total = sum(case["layers"] * m * n for m, n in shapes)
    return {"bytes": total * 4 * 5, "flops": sum(_ns_flops(case["layers"], m, n) for m, n in shapes) + 10 * total}
