"""Gradient norms and clipping: the cases they are measured on, in plain form and through the framework.

Three operators. `norm`: the norm over all tensors of a list of gradients (and each tensor's own, where asked).
`clip`: that list scaled so that its norm is at most max_norm. `elements`: each batch element's gradient, spread over
the tensors of a solver's backward, scaled by its own norm.
"""
import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # the policy's update at every PPO minibatch: actor and critic MLP for horizon 2, one small call
        {"name": "norm_policy_t2", "op": "norm", "list": "mlp", "horizon": 2, "dtype": "f32", "p": 2.0, "per_tensor": False},
        # half-precision gradients of a mid-sized network, largest magnitude (a loss scaler's overflow test)
        {"name": "norm_max_f16", "op": "norm", "list": "many", "tensors": 45, "values": 11_000_003, "dtype": "f16", "p": math.inf, "per_tensor": False},
        # gradients packed end to end into one bucket, logged per tensor
        {"name": "norm_bucket_bf16", "op": "norm", "list": "bucket", "tensors": 400, "values": 300_000_017, "dtype": "bf16", "p": 2.0, "per_tensor": True},
        # the same update's clipping: small, latency counts
        {"name": "clip_policy_t2", "op": "clip", "list": "mlp", "horizon": 2, "dtype": "f32", "p": 2.0, "ratio": 0.2},
        # a mid-sized network whose norm is below the bound: nothing changes, in place
        {"name": "clip_below_f32", "op": "clip", "list": "many", "tensors": 31, "values": 8_000_011, "dtype": "f32", "p": 2.0, "ratio": 3.0},
        # a bucket of bf16 gradients, tensors at odd offsets
        {"name": "clip_bucket_bf16", "op": "clip", "list": "bucket", "tensors": 200, "values": 100_000_007, "dtype": "bf16", "p": 2.0, "ratio": 0.35},
        # the solver's own gradients (x0, C, c) of the training-scale rollout, B=16384, T=20, clipped together
        {"name": "clip_rollout_t20", "op": "clip", "list": "solver", "batch": 16384, "horizon": 20, "dtype": "f32", "p": 2.0, "ratio": 0.1},
        # one control tick's batch, B=16, T=5, each element by itself
        {"name": "elements_b16_t5", "op": "elements", "cost": "dense", "n": 14, "batch": 16, "horizon": 5, "dtype": "f32", "time_major": True, "bad": 0},
        # the policy's sigmoid output at training scale, a few diverged solves zeroed
        {"name": "elements_sigmoid_t20", "op": "elements", "cost": "sigmoid", "n": 14, "batch": 16384, "horizon": 20, "dtype": "f32", "time_major": False, "bad": 7},
        # the 13-state rotor model, batch-major, B=4096, T=20: rows of 17x17 blocks, no 16-byte multiples
        {"name": "elements_rotor13_t20", "op": "elements", "cost": "dense", "n": 17, "batch": 4096, "horizon": 20, "dtype": "f32", "time_major": False, "bad": 0},
        # dense costs in the operator's own layout at training scale
        {"name": "elements_rollout_t20", "op": "elements", "cost": "dense", "n": 14, "batch": 16384, "horizon": 20, "dtype": "f32", "time_major": True, "bad": 0},
        # the long-horizon stress workload, B=65536, T=50: 2.8 GB of gradients
        {"name": "elements_stress_t50", "op": "elements", "cost": "dense", "n": 14, "batch": 65536, "horizon": 50, "dtype": "f32", "time_major": True, "bad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "clip", "elements", "elements"])
    if op == "elements":
        # at most the listed stress workload's values
        horizon = _log(rng, 1, 60)
        cost, n = rng.choice([("dense", 14), ("dense", 17), ("sigmoid", 14)])
        width = horizon * (n * n + n) if cost == "dense" else 28 * horizon
        batch = _log(rng, 1, max(2, min(70_000, 400_000_000 // width)))
        return {"op": op, "cost": cost, "n": n, "batch": batch, "horizon": horizon, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
                "time_major": cost == "dense" and rng.random() < 0.6, "bad": rng.choice([0, 0, min(batch, 3)])}
    kind = rng.choice(["mlp", "many", "bucket", "solver"])
    case = {"op": op, "list": kind, "dtype": rng.choice(["f32", "bf16", "f16"]), "p": rng.choice([2.0, 2.0, 2.0, math.inf])}
    if kind == "mlp":
        case["horizon"] = rng.randint(1, 50)
    elif kind == "solver":
        case["batch"], case["horizon"], case["dtype"] = _log(rng, 8, 20_000), rng.randint(1, 20), "f32"
    else:
        case["tensors"] = _log(rng, 1, 40) if kind == "many" else _log(rng, 2, 1500)
        case["values"] = _log(rng, 100 * case["tensors"], 200_000_000)
    if op == "norm":
        case["per_tensor"] = rng.random() < 0.5
    else:
        case["ratio"] = rng.choice([0.05, 0.5, 0.9, 3.0])
    return case


def _sizes(case):
    """The shapes of a case's tensors."""
    if case["op"] == "elements":
        b, t, n = case["batch"], case["horizon"], case["n"]
        lead = (t, b) if case["time_major"] else (b, t)
        return [(b, n - 4), (b, 28 * t)] if case["cost"] == "sigmoid" else [(b, n - 4), lead + (n, n), lead + (n,)]
    if case["list"] == "mlp":
        shapes = []
        for last in (28 * case["horizon"], 1):
            for i, o in ((64, 512), (512, 512), (512, last)):
                shapes += [(o, i), (o,)]
        return shapes
    if case["list"] == "solver":
        b, t = case["batch"], case["horizon"]
        return [(b, 10), (t, b, 14, 14), (t, b, 14)]
    # sizes spread over their logarithm, mostly odd, that add up to `values`
    rng = random.Random(case["tensors"] * 7919 + case["values"])
    weights = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    room = case["values"] - case["tensors"]
    sizes = [1 + int(room * w / sum(weights)) for w in weights]
    sizes[-1] += case["values"] - sum(sizes)
    return [(s,) for s in sizes]


def _count(case):
    return sum(math.prod(s) for s in _sizes(case))


@functools.cache
def _native():
    at = os.path.join(os.getcwd(), "ca-ac-mpc_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ilqr_native
    return ilqr_native


def prepare(case, seed):
    shapes, dtype = _sizes(case), DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["op"] == "elements":
        # the size of an element's gradient varies by orders of magnitude from solve to solve
        b = case["batch"]
        scale = torch.exp(1.5 * torch.randn(b, generator=gen, device="cuda")) * (4.0 / math.sqrt(_count(case) / b))
        grads, dims = [], []
        for s in shapes:
            d = 1 if case["time_major"] and len(s) > 2 else 0
            g = torch.randn(s, generator=gen, device="cuda")
            view = [1] * len(s)
            view[d] = b
            g.mul_(scale.view(view))
            grads.append(g.to(dtype))
            dims.append(d)
        if case["bad"]:
            rows = torch.randperm(b, generator=gen, device="cuda")[: case["bad"]]
            grads[0][rows, 0] = math.inf
            grads[-1].select(dims[-1], int(rows[0])).fill_(math.nan)
        state.update(grads=grads, dims=dims, max_norm=4.0, out=[torch.empty_like(g) for g in grads])
        return state
    sizes = [math.prod(s) for s in shapes]
    # magnitudes differ from tensor to tensor, as those of layers do
    scales = (torch.rand(len(sizes), generator=gen, device="cuda") * 4.0 - 2.0).exp().tolist()
    flat = torch.randn(sum(sizes), generator=gen, device="cuda") * 0.01
    for v, s in zip(flat.split(sizes), scales):
        v.mul_(s)
    flat = flat.to(dtype)
    packed = case["list"] == "bucket"
    grads = [v.view(s) if packed else v.clone().view(s) for v, s in zip(flat.split(sizes), shapes)]
    state["grads"] = grads
    if case["op"] == "clip":
        # the bound as a part of the norm that such gradients have
        size = max(s for s in scales) * 0.05 if case["p"] == math.inf else 0.01 * math.sqrt(sum(s * s * n for s, n in zip(scales, sizes)))
        state["max_norm"] = case["ratio"] * size
        if case["ratio"] > 1.0:
            state["out"] = grads
        else:
            out = torch.empty_like(flat) if packed else None
            state["out"] = [v.view(s) for v, s in zip(out.split(sizes), shapes)] if packed else [torch.empty_like(g) for g in grads]
            state["out_flat"] = out
        if packed and case["ratio"] > 1.0:
            state["out_flat"] = flat
    return state


def _plain_norm(grads, p):
    if p == math.inf:
        each = torch.stack([g.float().abs().max().double() for g in grads])
        return each.max(), each
    each = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads])
    return each.sum().sqrt(), each.sqrt()


def _run_norm(state, case):
    grads, p, per = state["grads"], case["p"], case["per_tensor"]
    if own:
        got = _native().grad_norm(grads, norm_type=p, per_tensor=per)
        return {"norm": got[0], "norms": got[1]} if per else {"norm": got}
    total, each = _plain_norm(grads, p)
    return {"norm": total.float(), "norms": each.float()} if per else {"norm": total.float()}


def _run_clip(state, case):
    grads, out = state["grads"], state["out"]
    if own:
        _, norm = _native().clip_grad_norm(grads, state["max_norm"], norm_type=case["p"], out=out)
    else:
        total, _ = _plain_norm(grads, case["p"])
        norm, scale = total.float(), (state["max_norm"] / (total + EPS)).clamp(max=1.0).float()
        [o.copy_(g.float() * scale) for g, o in zip(grads, out)]
    flat = state.get("out_flat")
    return {"norm": norm, "grads": out if flat is None else flat}


def _run_elements(state, case):
    grads, dims, out = state["grads"], state["dims"], state["out"]
    if own:
        _, norms = _native().clip_grad_elements(grads, state["max_norm"], batch_dims=dims, zero_nonfinite=case["bad"] > 0, out=out)
        return {"norms": norms, "grads": out}
    squares = sum(g.float().square().sum([i for i in range(g.dim()) if i != d], dtype=torch.float64) for g, d in zip(grads, dims))
    norms = squares.sqrt()
    scale = (state["max_norm"] / (norms + EPS)).clamp(max=1.0).float()
    lost = ~norms.isfinite() if case["bad"] else None
    [_scaled(g, d, o, scale, lost) for g, d, o in zip(grads, dims, out)]
    return {"norms": norms.float(), "grads": out}


def _scaled(g, d, o, scale, lost):
    view = [1] * g.dim()
    view[d] = -1
    o.copy_(g.float() * scale.view(view))
    if lost is not None:
        o.masked_fill_(lost.view(view), 0.0)


def run(state):
    case = state["case"]
    return {"norm": _run_norm, "clip": _run_clip, "elements": _run_elements}[case["op"]](state, case)


def work(case):
    n, size = _count(case), BYTES[case["dtype"]]
    if case["op"] == "norm":
        return {"bytes": n * size + 4 * (1 + (len(_sizes(case)) if case["per_tensor"] else 0)), "flops": 2 * n}
    if case["op"] == "clip":
        # below the bound and in place every value stays as it is
        return {"bytes": n * size * (1 if case["ratio"] > 1.0 else 2) + 4, "flops": (2 if case["ratio"] > 1.0 else 3) * n}
    return {"bytes": 2 * n * size + 4 * case["batch"], "flops": 3 * n}


def exact(case, seed):
    state = prepare(case, seed)
    wide = [g.double() for g in state["grads"]]
    if case["op"] == "elements":
        b = case["batch"]
        rows = [w.movedim(d, 0).reshape(b, -1) for w, d in zip(wide, state["dims"])]
        norms = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(r, dim=1) for r in rows]), dim=0)
        scale = torch.where(norms + EPS > state["max_norm"], state["max_norm"] / (norms + EPS), torch.ones_like(norms))
        scale = torch.where(norms.isnan(), norms, scale)
        done = []
        for w, d in zip(wide, state["dims"]):
            view = [b if i == d else 1 for i in range(w.dim())]
            y = w * scale.view(view)
            done.append(torch.where(norms.isfinite().view(view), y, torch.zeros_like(y)) if case["bad"] else y)
        return {"norms": norms, "grads": done}
    p = case["p"]
    each = torch.stack([torch.linalg.vector_norm(w.reshape(-1), ord=p) for w in wide])
    norm = torch.linalg.vector_norm(each, ord=p)
    if case["op"] == "norm":
        return {"norm": norm, "norms": each} if case["per_tensor"] else {"norm": norm}
    scale = min(1.0, state["max_norm"] / (float(norm) + EPS))
    done = [w * scale for w in wide]
    return {"norm": norm, "grads": torch.cat([w.reshape(-1) for w in done]) if state.get("out_flat") is not None else done}
