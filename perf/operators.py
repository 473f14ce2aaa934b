"""The training operators on the GPU, case by case: layer norm (forward; forward and backward) and the clipping of gradients
to a global norm.

`own` says which side `run` takes: False computes the operators in their plain form, elementary torch operations in 32 bits
that are rounded once at the end; True makes the calls a trainer makes of rebel_amd.training.
"""
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def _norm(name, op, rows, cols, dtype, params, act=None, pad=0):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "params": params, "act": act, "pad": pad}


def _clip(name, layout, tensors, numel, dtype, p, reached):
    return {"name": name, "op": "clip", "layout": layout, "tensors": tensors, "numel": numel, "dtype": dtype, "p": p,
            "reached": reached}


def listed():
    return [
        # one query through one block of the value net (n_hidden = 256): latency
        _norm("forward one row", "forward", 1, 256, "f32", "f32", "gelu"),
        # every leaf of 4 096 lanes of the 1 die x 6 faces game in one batch
        _norm("forward leaf batch", "forward", 270336, 256, "f32", "f32", "gelu"),
        # a wide net in half precision: evaluation of a long batch
        _norm("forward wide bf16", "forward", 8192, 4096, "bf16", "bf16"),
        # odd width, rows that lie in a wider buffer (a slice of concatenated features)
        _norm("forward slice odd f16", "forward", 5001, 1537, "f16", "f32", "gelu", 30),
        # the trainer's batch of 512 examples through one block of the value net
        _norm("train batch 512", "train", 512, 256, "f32", "f32", "gelu"),
        # half-precision activations over 32-bit master weights
        _norm("train bf16 over f32", "train", 16384, 2048, "bf16", "f32"),
        # odd rows and width
        _norm("train odd f16", "train", 4099, 1023, "f16", "f16", "gelu"),
        # few long rows: the axis is longer than one workgroup's registers hold
        _norm("train long rows", "train", 24, 65537, "f32", "f32"),
        # the largest: a big batch of wide rows
        _norm("train largest", "train", 32768, 8192, "bf16", "bf16"),
        # the value net's own ten gradients
        _clip("clip value net", "net2", 10, 0, "f32", "2", True),
        # many ragged tensors of two types whose norm stays under the bound, as most steps' does
        _clip("clip ragged unreached", "ragged", 360, 60_000_000, "mixed", "2", False),
        # a large model's gradients, more than any cache holds
        _clip("clip large", "ragged", 200, 400_000_000, "f32", "2", True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["forward", "train", "train", "clip"])
    if kind == "clip":
        tensors = _log_uniform(rng, 1, 600)
        return {"op": "clip", "layout": "ragged", "tensors": tensors, "numel": max(tensors, _log_uniform(rng, 1000, 200_000_000)),
                "dtype": rng.choice(["f32", "bf16", "f16", "mixed"]), "p": rng.choice(["2", "2", "2", "1", "inf"]),
                "reached": rng.random() < 0.7}
    cols = _log_uniform(rng, 8, 70000)
    rows = _log_uniform(rng, 1, max(2, min(400_000, 130_000_000 // cols)))
    dtype = rng.choice(["f32", "f16", "bf16"])
    return {"op": kind, "rows": rows, "cols": cols, "dtype": dtype, "params": rng.choice(["f32", dtype]),
            "act": rng.choice([None, "gelu"]), "pad": rng.choice([0, 0, 0, rng.randrange(1, 70)])}


def _sizes(case):
    """(numel, dtype) of each gradient: a few matrices hold nearly everything, the vectors between them little."""
    if case["layout"] == "net2":  # body.0, body.1, body.4, body.5, output of the 1 die x 6 faces net
        return [(n, "f32") for n in (256 * 27, 256, 256, 256, 256 * 256, 256, 256, 256, 6 * 256, 6)]
    r = random.Random(case["tensors"] * 1_000_003 + case["numel"])
    share = [r.random() ** 4 + 1e-4 for _ in range(case["tensors"])]
    total = sum(share)
    numel = [max(1, int(case["numel"] * s / total)) for s in share]
    return [(n, case["dtype"] if case["dtype"] != "mixed" else r.choice(["bf16", "bf16", "f32"])) for n in numel]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "clip":
        sizes = _sizes(case)
        held = {}  # the gradients of a type lie in one buffer, each at a 512-byte boundary
        params = []
        place = {d: 0 for _, d in sizes}
        at = []
        for n, d in sizes:
            at.append(place[d])
            place[d] += -(-n * SIZE[d] // 512) * 512 // SIZE[d]
        for d in sorted(place):
            held[d] = torch.zeros(place[d], dtype=DTYPES[d], device="cuda")
        for (n, d), o in zip(sizes, at):
            p = torch.nn.Parameter(torch.empty(n, dtype=DTYPES[d], device="cuda"))
            p.grad = held[d][o:o + n]
            p.grad.copy_(normal(n) * (0.02 + 0.1 * float(torch.rand((), generator=g, device="cuda"))))
            params.append(p)
        bound = (0.01 if case["p"] == "inf" else 0.5) if case["reached"] else 1e9
        return {"op": "clip", "params": params, "held": [held[d] for d in sorted(held)], "p": float(case["p"]), "bound": bound,
                "tighten": 0.9999 if case["reached"] else 1.0}
    rows, cols, t = case["rows"], case["cols"], DTYPES[case["dtype"]]
    wide = torch.empty(rows, cols + case["pad"], dtype=t, device="cuda")
    x = wide[:, :cols]
    x.copy_(normal(rows, cols))
    x.mul_(torch.rand(rows, 1, generator=g, device="cuda") * 2 + 0.1).add_(normal(rows, 1))  # each row has its own scale and mean
    x[96::97] = 0  # rows that are padding
    state = {"op": case["op"], "x": x.detach(), "w": (1 + 0.2 * normal(cols)).to(DTYPES[case["params"]]),
             "b": (0.2 * normal(cols)).to(DTYPES[case["params"]]), "act": case["act"]}
    if case["op"] == "train":
        state["dy"] = (normal(rows, cols) * 0.05).to(t)
        for k in ("x", "w", "b"):
            state[k].requires_grad_(True)
    return state


def _plain_norm(state):
    x, w, b = state["x"].float(), state["w"].float(), state["b"].float()
    d = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
    h = d * r
    z = h * w + b
    cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) if state["act"] else None
    y = (z * cdf if state["act"] else z).to(state["x"].dtype)
    if state["op"] == "forward":
        return y
    g = state["dy"].float()
    if state["act"]:
        g = g * (cdf + z * torch.exp(-0.5 * z.square()) * (2 * torch.pi) ** -0.5)
    gw = g * w
    dx = r * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(state["x"].dtype), "dw": (g * h).sum(0).to(state["w"].dtype),
            "db": g.sum(0).to(state["b"].dtype)}


def _plain_clip(state, bound):
    grads = [p.grad for p in state["params"]]
    if state["p"] == float("inf"):
        norm = torch.stack([g.float().abs().amax() for g in grads]).amax()
    elif state["p"] == 1.0:
        norm = torch.stack([g.float().abs().sum() for g in grads]).sum()
    else:
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    c = torch.clamp(bound / (norm + 1e-6), max=1.0)
    [g.copy_(g.float() * c) for g in grads]
    return norm


def run(state):
    if state["op"] == "clip":
        # the bound is tightened a little from step to step, so that a pass that clips never finds the gradients clipped
        state["bound"] *= state["tighten"]
        if own:
            from rebel_amd import training

            norm = training.clip_grad_norm_(state["params"], state["bound"], state["p"])
        else:
            with torch.no_grad():
                norm = _plain_clip(state, state["bound"])
        return {"norm": norm, "grads": state["held"]}
    if not own:
        with torch.no_grad():
            return _plain_norm(state)
    from rebel_amd import training

    x, w, b = state["x"], state["w"], state["b"]
    y = training.layer_norm(x, w, b, eps=EPS, activation=state["act"])
    if state["op"] == "forward":
        return y
    dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def work(case):
    if case["op"] == "clip":
        sizes = _sizes(case)
        n = sum(k for k, _ in sizes)
        held = sum(k * SIZE[d] for k, d in sizes)
        return {"bytes": held * (2 if case["reached"] else 1) + 4, "flops": n * (3 if case["reached"] else 2)}
    n = case["rows"] * case["cols"]
    size, param = SIZE[case["dtype"]], SIZE[case["params"]] * case["cols"]
    act = bool(case["act"])
    if case["op"] == "forward":  # x and the two parameters in, y out
        return {"bytes": 2 * n * size + 2 * param, "flops": n * (8 + 20 * act)}
    # x, dy and the parameters in; y, dx and the parameters' gradients out
    return {"bytes": 4 * n * size + 4 * param, "flops": n * (24 + 40 * act)}


def exact(case, seed):
    """The operators' definitions in 64 bits; the gradients are those that differentiation of the definition gives."""
    state = prepare(case, seed)
    if case["op"] == "clip":
        bound = state["bound"] * state["tighten"]
        values = [h.double() for h in state["held"]]  # what lies between the gradients is zero
        norm = torch.stack([torch.linalg.vector_norm(v, state["p"]) for v in values])
        norm = torch.linalg.vector_norm(norm, state["p"])
        factor = min(1.0, bound / (float(norm) + 1e-6))
        return {"norm": norm, "grads": [v * factor for v in values]}
    x, w, b = (state[k].detach().double().requires_grad_(case["op"] == "train") for k in ("x", "w", "b"))
    moment = (x * x).mean(-1, keepdim=True) - x.mean(-1, keepdim=True) ** 2
    z = (x - x.mean(-1, keepdim=True)) / torch.sqrt(moment + EPS) * w + b
    y = 0.5 * z * torch.erfc(-z / 2 ** 0.5) if case["act"] else z
    if case["op"] == "forward":
        return y
    dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
