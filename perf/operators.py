"""The 4-bit projections and the residual norm between them: what they compute, on which inputs.

``run`` computes each operator from elementary torch operations in 32 bits, or, where ``own`` is
true, by the framework's public calls.  Three operators:

* ``linear``: y = x (q * s)^T + b with 4-bit q and one bf16 scale s per output channel and group of
  input features,
* ``gateup``: h = silu(x Wg^T) * (x Wu^T), both weights as above (the first half of a gated MLP),
* ``norm``: r' = a r + b act(gate) rms(y; w_post), x' = rms(r'; w_pre), the step between two blocks.
"""

import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _sbq():
    return importlib.import_module("spikingbrain-cpu_b200")


# ---- cases -----------------------------------------------------------------------------------------

def _linear(name, m, k, n, group, x, y, bias=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "group": group, "x": x, "y": y, "bias": bias}


def _gateup(name, m, k, n, group, x, y):
    return {"name": name, "op": "gateup", "m": m, "k": k, "n": n, "group": group, "x": x, "y": y}


def _norm(name, m, d, y, r, x, post, gate, act, scale):
    return {"name": name, "op": "norm", "m": m, "d": d, "y": y, "r": r, "x": x, "post": post, "gate": gate, "act": act,
            "scale": scale}


def listed():
    return [
        # one token through the key projection of the checkpoint (8 heads of 128): the smallest call, latency only
        _linear("linear 1x2560x1024", 1, 2560, 1024, 128, "f16", "f16"),
        # one token through the benchmark's square projection
        _linear("linear 1x4096x4096", 1, 4096, 4096, 128, "f16", "f32"),
        # one token through the tied head over the whole vocabulary
        _linear("linear 1x2560x151936", 1, 2560, 151936, 128, "bf16", "f32"),
        # eight sequences decoded together through the MLP's down projection, fp32 activations
        _linear("linear 8x12288x4096 f32", 8, 12288, 4096, 64, "f32", "f32"),
        # a small ragged batch, sizes that are multiples of nothing, small groups, a bias
        _linear("linear 45x2500x4099 odd", 45, 2500, 4099, 32, "bf16", "bf16", True),
        # the reference's 512-token prompt chunk through the checkpoint's MLP, fp32 activations and output
        _linear("linear 512x2560x9728 f32", 512, 2560, 9728, 128, "f32", "f32"),
        # a long prompt through the benchmark's MLP projection
        _linear("linear 4096x4096x12288", 4096, 4096, 12288, 128, "f16", "f16"),
        # the MLP's first half, one token
        _gateup("gateup 1x4096x12288", 1, 4096, 12288, 128, "f16", "f16"),
        # the MLP's first half, a long prompt
        _gateup("gateup 2048x4096x12288", 2048, 4096, 12288, 64, "bf16", "f16"),
        # the step between two blocks, one token
        _norm("norm 1x4096", 1, 4096, "f32", "f32", "f16", True, "none", "none", True),
        # the same for a long prompt, pre-norm only (no post norm, plain residual)
        _norm("norm 8192x4096", 8192, 4096, "f32", "f32", "f16", False, "none", "none", False),
        # a gate per element, both norms, 16-bit residual, an odd width
        _norm("norm 3001x2559 gated", 3001, 2559, "bf16", "bf16", "bf16", True, "full", "sigmoid", True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "gateup", "norm", "norm"))
    if op == "norm":
        d = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            d = max(64, d // 64 * 64)
        m = _log(rng, 1, max(1, 8192 * 4096 // d))
        return {"op": "norm", "m": m, "d": d, "y": rng.choice(("f32", "f16", "bf16")), "r": rng.choice(("f32", "f32", "bf16")),
                "x": rng.choice(("f16", "bf16", "f32")), "post": rng.random() < 0.6,
                "gate": rng.choice(("none", "vector", "token", "full")), "act": rng.choice(("none", "sigmoid", "silu", "tanh")),
                "scale": rng.random() < 0.5}
    k, n = _log(rng, 64, 12288), _log(rng, 16, 24576)
    if rng.random() < 0.7:
        k, n = max(64, k // 64 * 64), max(16, n // 16 * 16)
    most = 4096 * 4096 * 12288 // (2 if op == "gateup" else 1)
    m = _log(rng, 1, max(1, min(4096, most // (k * n))))
    c = {"op": op, "m": m, "k": k, "n": n, "group": rng.choice((32, 64, 128, 128)), "x": rng.choice(("f32", "f16", "bf16")),
         "y": rng.choice(("f32", "f16", "bf16"))}
    if op == "linear":
        c["bias"] = rng.random() < 0.3
    return c


# ---- inputs ----------------------------------------------------------------------------------------

def _weight(gen, n, k, group):
    """A weight N(0, 0.02) quantised by group: q int8 [n, k] in [-7, 7], scale bf16 [n, ceil(k / group)]."""
    groups = -(-k // group)
    w = torch.zeros(n, groups * group, device="cuda")
    w[:, :k] = torch.randn(n, k, generator=gen, device="cuda") * 0.02
    w = w.view(n, groups, group)
    scale = (w.abs().amax(dim=2).clamp_min(1e-8) / 7.0).to(torch.bfloat16)
    q = (w / scale.float()[:, :, None]).round().clamp(-7, 7).to(torch.int8)
    return q.view(n, groups * group)[:, :k].contiguous(), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "norm":
        m, d = case["m"], case["d"]
        # a block's output, the running residual (a few times larger), learned weights around one
        state["branch"] = rand(m, d).to(DTYPES[case["y"]])
        state["residual"] = (rand(m, d) * 4.0).to(DTYPES[case["r"]])
        state["pre_weight"] = 1.0 + 0.1 * rand(d)
        state["post_weight"] = 1.0 + 0.1 * rand(d) if case["post"] else None
        shape = {"none": None, "vector": (d,), "token": (m, 1), "full": (m, d)}[case["gate"]]
        state["gate_value"] = None if shape is None else rand(*shape).to(DTYPES[case["y"]])
        state["scales"] = (0.75, 1.25) if case["scale"] else (1.0, 1.0)  # of the residual, of the block's output
        return state
    m, k, n, group = case["m"], case["k"], case["n"], case["group"]
    state["x_in"] = rand(m, k).to(DTYPES[case["x"]])
    state["weights"] = [_weight(gen, n, k, group) for _ in range(2 if case["op"] == "gateup" else 1)]
    state["bias_value"] = rand(n) * 0.1 if case.get("bias") else None
    if own:
        # the modules a program holds after loading its weights
        sbq = _sbq()
        linears = [sbq.Int4Linear.from_quantized(q, s, state["bias_value"], group=group) for q, s in state["weights"]]
        if case["op"] == "gateup":
            # the module takes all three projections; only its first half is run here
            down = sbq.Int4Linear.from_quantized(torch.zeros(16, n, dtype=torch.int8, device="cuda"),
                                                 torch.ones(16, -(-n // group), dtype=torch.bfloat16, device="cuda"), None,
                                                 group=group)
            state["module"] = sbq.FusedGatedMLP(*linears, down, h_dtype=DTYPES[case["y"]])
        else:
            linears[0].out_dtype = DTYPES[case["y"]]
            state["module"] = linears[0]
    return state


# ---- one pass --------------------------------------------------------------------------------------

def _product(x, q, scale, group):
    """x (q * s)^T in fp32: the group scales spread over their columns, then one matrix product."""
    w = q.float() * scale.float().repeat_interleave(group, dim=1)[:, :q.shape[1]]
    return x.float() @ w.t()


def _rms(v, weight):
    return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * weight


def run(state):
    op = state["op"]
    if own:
        if op == "linear":
            return state["module"](state["x_in"])
        if op == "gateup":
            return state["module"].gateup(state["x_in"])
        a, b = state["scales"]
        r, x = _sbq().residual_norm(state["branch"], state["residual"], pre_weight=state["pre_weight"],
                                    post_weight=state["post_weight"], gate=state["gate_value"], gate_act=state["act"],
                                    residual_scale=a, branch_scale=b, eps=EPS, out_dtype=DTYPES[state["x"]])
        return {"residual": r, "x": x}
    if op == "norm":
        h = state["branch"].float()
        if state["post_weight"] is not None:
            h = _rms(h, state["post_weight"])
        if state["gate_value"] is not None:
            g = state["gate_value"].float()
            if state["act"] == "sigmoid":
                g = 1.0 / (1.0 + torch.exp(-g))
            elif state["act"] == "silu":
                g = g / (1.0 + torch.exp(-g))
            elif state["act"] == "tanh":
                g = torch.tanh(g)
            h = g * h
        a, b = state["scales"]
        r = a * state["residual"].float() + b * h
        x = _rms(r, state["pre_weight"])
        return {"residual": r.to(DTYPES[state["r"]]), "x": x.to(DTYPES[state["x"]])}
    y = _product(state["x_in"], *state["weights"][0], state["group"])
    if op == "gateup":
        up = _product(state["x_in"], *state["weights"][1], state["group"])
        y = y / (1.0 + torch.exp(-y)) * up
    elif state["bias_value"] is not None:
        y = y + state["bias_value"]
    return y.to(DTYPES[state["y"]])


def work(case):
    if case["op"] == "norm":
        m, d = case["m"], case["d"]
        gate = {"none": 0, "vector": d, "token": m, "full": m * d}[case["gate"]] * SIZE[case["y"]]
        weights = 4 * d * (2 if case["post"] else 1)
        return {"bytes": m * d * (SIZE[case["y"]] + 2 * SIZE[case["r"]] + SIZE[case["x"]]) + gate + weights,
                "flops": 14 * m * d}
    m, k, n, group = case["m"], case["k"], case["n"], case["group"]
    mats = 2 if case["op"] == "gateup" else 1
    weight = n * k // 2 + 2 * n * -(-k // group)
    return {"bytes": mats * weight + m * k * SIZE[case["x"]] + m * n * SIZE[case["y"]] + (4 * n if case.get("bias") else 0),
            "flops": 2 * m * n * k * mats}


# ---- the definition in 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        y, r = state["branch"].double(), state["residual"].double()
        d = y.shape[1]
        if state["post_weight"] is not None:
            y = y / (y.square().sum(1, keepdim=True) / d + EPS).sqrt() * state["post_weight"].double()
        if state["gate_value"] is not None:
            g = state["gate_value"].double()
            g = {"none": lambda v: v, "sigmoid": lambda v: v.sigmoid(), "silu": lambda v: v * v.sigmoid(),
                 "tanh": lambda v: v.tanh()}[case["act"]](g)
            y = y * g
        a, b = state["scales"]
        r = r * a + y * b
        x = r / (r.square().sum(1, keepdim=True) / d + EPS).sqrt() * state["pre_weight"].double()
        return {"residual": r, "x": x}
    x, group = state["x_in"].double(), case["group"]
    out = []
    for q, scale in state["weights"]:
        y = torch.zeros(x.shape[0], q.shape[0], dtype=torch.float64, device="cuda")
        for g in range(scale.shape[1]):  # group by group: integer weights first, then the group's scale
            cols = slice(g * group, min((g + 1) * group, q.shape[1]))
            y += (x[:, cols] @ q[:, cols].double().t()) * scale[:, g].double()
        out.append(y)
    if case["op"] == "gateup":
        return out[0] * out[0].sigmoid() * out[1]
    return out[0] if state["bias_value"] is None else out[0] + state["bias_value"].double()
