"""What the operators for 8-bit weights and routed experts cost: cases, their plain form and their definition in 64 bits.

Three operators: `route` (router scores to experts and weights), `linear` (a linear layer whose weight is e4m3 with one float32 scale per block
of 128 x 128 and whose input is quantised per token and block of 128 columns), `experts` (the routed experts' gated feed-forward in that form).
A case is a dict of plain values; `prepare` makes its inputs on the GPU, `run` is one pass, in the framework's kernels where `own` is true."""
import math

import numpy as np
import torch

own = False

BLOCK = 128
TOP = 448.0          # the largest e4m3 value


# ------------------------------------------------------------------ cases
def _route(name, n, experts, top, score, groups=1, top_groups=1, group_best=2, bias=True, renormalise=True, scale=1.0):
    return {"name": name, "kind": "route", "n": n, "experts": experts, "top": top, "score": score, "groups": groups, "top_groups": top_groups,
            "group_best": group_best, "bias": bias, "renormalise": renormalise, "scale": scale}


def _linear(name, n, m, k, epilogue, x, out):
    return {"name": name, "kind": "linear", "n": n, "m": m, "k": k, "epilogue": epilogue, "x": x, "out": out}


def _experts(name, n, experts, top, width, inner):
    return {"name": name, "kind": "experts", "n": n, "experts": experts, "top": top, "width": width, "inner": inner}


def listed():
    return [
        # the router of a step of one decoded token, and of a long step of prompts, both with groups and a balance bias
        _route("route_1", 1, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5),
        _route("route_16384", 16384, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5),
        # a router without groups: softmax over an odd number of experts, a ragged step
        _route("route_softmax_777", 777, 90, 6, "softmax", 1, 1, 1, False, False, 1.0),
        # an output projection of one decoded token (width 2,048), added to nothing: the smallest product
        _linear("linear_1", 1, 2048, 2048, "store", "bfloat16", "float32"),
        # gate and up projection of a decode step of eight requests (feed-forward of 8,192)
        _linear("linear_gated_8", 8, 16384, 2048, "gated", "bfloat16", "bfloat16"),
        # a down projection of 64 requests at the sizes of an 8B decoder
        _linear("linear_64", 64, 4096, 14336, "store", "bfloat16", "float32"),
        # a ragged prompt portion through sizes that nothing divides, 32-bit activations
        _linear("linear_odd_333", 333, 2500, 2056, "store", "float32", "float32"),
        # a prompt step of 4,096 tokens through the gate and up projection of an 8B decoder: the largest product
        _linear("linear_gated_4096", 4096, 28672, 4096, "gated", "bfloat16", "bfloat16"),
        # one decoded token, 32 requests and a prompt through small routed experts
        _experts("experts_1", 1, 64, 6, 2048, 1408),
        _experts("experts_32", 32, 64, 6, 2048, 1408),
        _experts("experts_2000", 2000, 64, 6, 2048, 1408),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    kind = rng.choice(["route", "linear", "linear", "experts"])
    if kind == "route":
        score = rng.choice(["sigmoid", "softmax"])
        n = _spread(rng, 1, 16384)
        if rng.random() < 0.5:
            groups = rng.choice([2, 4, 8, 16])
            size = rng.randint(4, 256 // groups)
            top_groups = rng.randint(1, groups)
            top = rng.randint(1, min(8, top_groups * size))
            return _route("", n, groups * size, top, score, groups, top_groups, rng.choice([1, 2]), rng.random() < 0.7, rng.random() < 0.7,
                          rng.choice([1.0, 2.5]))
        experts = rng.randint(8, 256)
        return _route("", n, experts, rng.randint(1, min(8, experts)), score, 1, 1, 1, rng.random() < 0.5, rng.random() < 0.5, 1.0)
    if kind == "linear":
        gated = rng.random() < 0.4
        while True:
            n, k = _spread(rng, 1, 4096), _spread(rng, 128, 14336)
            m = _spread(rng, 128, 14336) * 2
            if rng.random() < 0.5:
                k, m = (k + 127) // 128 * 128, (m + 255) // 256 * 256
            if m * k <= 28672 * 4096 and k <= 14336:
                break
        return _linear("", n, m, k, "gated" if gated else "store", rng.choice(["bfloat16", "bfloat16", "float32"]),
                       "bfloat16" if gated else rng.choice(["bfloat16", "float32"]))
    experts = _spread(rng, 4, 64)
    return _experts("", _spread(rng, 1, 2000), experts, rng.randint(1, min(6, experts)), _spread(rng, 256, 2048), _spread(rng, 128, 1408))


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)


def _activations(gen, n, k, dtype):
    """Normed activations: every token near unit size, a few columns much larger than the rest, as decoders have them."""
    x = torch.randn(n, k, generator=gen, device="cuda")
    x *= torch.exp(0.3 * torch.randn(n, 1, generator=gen, device="cuda"))
    columns = torch.rand(k, generator=gen, device="cuda") < 0.004
    return torch.where(columns, 12.0 * x, x).to(dtype)


def _weight(gen, count, m, k):
    """`count` matrices [m, k] in e4m3 and their scales [count, ceil(m / 128), ceil(k / 128)], as a checkpoint stores them."""
    bm, bk = -(-m // BLOCK), -(-k // BLOCK)
    q = torch.empty(count, m, k, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(count, bm, bk, device="cuda")
    for c in range(count):
        w = torch.randn(m, k, generator=gen, device="cuda", dtype=torch.float32) * (0.7 / math.sqrt(k))
        padded = torch.zeros(bm * BLOCK, bk * BLOCK, device="cuda")
        padded[:m, :k] = w
        blocks = padded.view(bm, BLOCK, bk, BLOCK)
        s = blocks.abs().amax(dim=(1, 3)) / TOP
        q[c] = (blocks / s[:, None, :, None]).reshape(bm * BLOCK, bk * BLOCK)[:m, :k].to(torch.float8_e4m3fn)
        scales[c] = s
    return q, scales


def prepare(case, seed):
    gen = _generator(seed)
    state = dict(case)
    if case["kind"] == "route":
        n, E = case["n"], case["experts"]
        state["logits"] = torch.randn(n, E, generator=gen, device="cuda") * 1.5
        state["bias_values"] = torch.randn(E, generator=gen, device="cuda") * 0.05 if case["bias"] else None
        state["choice"] = torch.empty(n, case["top"], dtype=torch.int32, device="cuda")
        state["weights"] = torch.empty(case["top"], n, device="cuda")
        return state
    if case["kind"] == "linear":
        n, m, k = case["n"], case["m"], case["k"]
        gated = case["epilogue"] == "gated"
        state["x_values"] = _activations(gen, n, k, getattr(torch, case["x"]))
        state["q"], state["scales"] = _weight(gen, 2, m // 2, k) if gated else _weight(gen, 1, m, k)
        state["result"] = torch.empty(n, m // 2 if gated else m, dtype=getattr(torch, case["out"]), device="cuda")
        if own:
            from stride_b200.kernels.linear import Fp8Weight, Linear
            from stride_b200.parts.context import Workspace
            weight = Fp8Weight.stack([Fp8Weight(q, s) for q, s in zip(state.pop("q"), state.pop("scales"))])
            state["layer"] = Linear(weight, torch.bfloat16)
            state["workspace"] = Workspace(torch.device("cuda"), n)
        return state
    n, E, top, W, F = (case[key] for key in ("n", "experts", "top", "width", "inner"))
    state["x_values"] = _activations(gen, n, W, torch.bfloat16)
    # experts as a router would choose them, some more often than others
    popularity = 0.5 * torch.randn(E, generator=gen, device="cuda")
    scores = torch.sigmoid(torch.randn(n, E, generator=gen, device="cuda") + popularity)
    best, at = torch.topk(scores, top, dim=1)
    state["choice"] = at.to(torch.int32).contiguous()
    state["weights"] = (best / best.sum(dim=1, keepdim=True)).t().contiguous()
    gate, up, down = _weight(gen, E, F, W), _weight(gen, E, F, W), _weight(gen, E, W, F)
    state["result"] = torch.empty(n, W, dtype=torch.bfloat16, device="cuda")
    if own:
        from stride_b200.kernels.linear import Fp8Experts, Fp8Weight
        pairs = [Fp8Weight(q[e], s[e]) for e in range(E) for q, s in (gate, up)]
        state["layer"] = Fp8Experts(pairs, [Fp8Weight(down[0][e], down[1][e]) for e in range(E)])
        state["scratch"] = state["layer"].scratch(n, top)
    else:
        state["gate"], state["up"], state["down"] = gate, up, down
    return state


# ------------------------------------------------------------------ the plain form
def _quantised(x):
    """x [n, k] as the values that its e4m3 form stands for, in 32 bits."""
    n, k = x.shape
    bk = -(-k // BLOCK)
    padded = torch.zeros(n, bk * BLOCK, device=x.device)
    padded[:, :k] = x.float()
    blocks = padded.view(n, bk, BLOCK)
    mantissa, exponent = torch.frexp(blocks.abs().amax(dim=2, keepdim=True))        # amax = mantissa 2^exponent, mantissa in [1/2, 1)
    e = torch.where(mantissa == 0, torch.full_like(exponent, -100), exponent - 9 + (mantissa > 0.875).to(exponent.dtype)).clamp(min=-100)
    s = torch.ldexp(torch.ones_like(mantissa), e)
    return ((blocks / s).to(torch.float8_e4m3fn).float() * s).view(n, bk * BLOCK)[:, :k]


def _widened(q, scales):
    m, k = q.shape
    return q.float() * scales.repeat_interleave(BLOCK, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]


def _plain_route(state):
    z = state["logits"].double()
    n, E = z.shape
    if state["score"] == "softmax":
        s = torch.exp(z - z.amax(dim=1, keepdim=True))
        s = s / s.sum(dim=1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    c = s if state["bias_values"] is None else s + state["bias_values"].double()
    if state["groups"] > 1:
        members = c.view(n, state["groups"], -1)
        best = torch.sort(members, dim=2, descending=True).values[:, :, :state["group_best"]].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :state["top_groups"]]
        allowed = torch.zeros(n, state["groups"], dtype=torch.bool, device=z.device).scatter_(1, kept, True)
        c = torch.where(allowed.repeat_interleave(E // state["groups"], 1), c, torch.full_like(c, -math.inf))
    choice = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :state["top"]]
    w = torch.gather(s, 1, choice)
    if state["renormalise"]:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return choice.to(torch.int32), (w * state["scale"]).t().float()


def _plain_linear(state):
    x = _quantised(state["x_values"])
    products = [x @ _widened(q, s).t() for q, s in zip(state["q"], state["scales"])]
    if state["epilogue"] == "gated":
        g, u = products
        return (g / (1.0 + torch.exp(-g)) * u).to(state["result"].dtype)
    return products[0].to(state["result"].dtype)


def _plain_experts(state):
    x, choice, weights = _quantised(state["x_values"]), state["choice"], state["weights"]
    out = torch.zeros(x.shape[0], state["width"], device=x.device)
    results = torch.zeros(state["top"], x.shape[0], state["width"], device=x.device)
    for e in range(state["experts"]):
        token, k = torch.nonzero(choice == e, as_tuple=True)
        rows = x[token]
        g = rows @ _widened(state["gate"][0][e], state["gate"][1][e]).t()
        u = rows @ _widened(state["up"][0][e], state["up"][1][e]).t()
        z = _quantised(g / (1.0 + torch.exp(-g)) * u)
        results[k, token] = weights[k, token][:, None] * (z @ _widened(state["down"][0][e], state["down"][1][e]).t())
    for k in range(state["top"]):
        out += results[k]
    return out.to(state["result"].dtype)


def run(state):
    if not own:
        return {"route": _plain_route, "linear": _plain_linear, "experts": _plain_experts}[state["kind"]](state)
    from stride_b200.kernels import ops
    if state["kind"] == "route":
        ops.route_experts(state["logits"], state["choice"], state["weights"], score=state["score"], bias=state["bias_values"], groups=state["groups"],
                          top_groups=state["top_groups"], group_best=state["group_best"], renormalise=state["renormalise"], scale=state["scale"])
        return state["choice"], state["weights"]
    if state["kind"] == "linear":
        if state["epilogue"] == "gated":
            state["layer"].forward_swiglu(state["x_values"], state["result"], None, workspace=state["workspace"])
        else:
            state["layer"].forward(state["x_values"], state["result"], workspace=state["workspace"])
        return state["result"]
    state["layer"].forward(state["x_values"], state["choice"], state["weights"], state["result"], state["scratch"])
    return state["result"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"bfloat16": 2, "float32": 4}
    n = case["n"]
    if case["kind"] == "route":
        E = case["experts"]
        return {"bytes": n * (4 * E + 8 * case["top"]) + (4 * E if case["bias"] else 0), "flops": 4 * n * E}
    if case["kind"] == "linear":
        m, k = case["m"], case["k"]
        wide = m // 2 if case["epilogue"] == "gated" else m
        blocks = (2 if wide < m else 1) * -(-wide // BLOCK) * -(-k // BLOCK)
        return {"bytes": n * k * size[case["x"]] + m * k + 4 * blocks + n * wide * size[case["out"]], "flops": 2 * n * m * k}
    E, top, W, F = case["experts"], case["top"], case["width"], case["inner"]
    used = E * (1.0 - (1.0 - top / E) ** n)          # experts that at least one of n tokens chose, if all are chosen alike
    return {"bytes": int(used * 3 * W * F * (1 + 4 / BLOCK ** 2)) + n * W * 4 + n * top * 8, "flops": 6 * n * top * W * F}


# ------------------------------------------------------------------ the definition in 64 bits, on its own
def _grid(x):
    """x [n, k] float64 rounded to the e4m3 grid of its blocks."""
    n, k = x.shape
    out = torch.empty_like(x)
    for b in range(0, k, BLOCK):
        part = x[:, b:b + BLOCK]
        amax = part.abs().max(dim=1).values.cpu().numpy()
        e = np.full(n, -100.0)
        some = amax > 0
        e[some] = np.maximum(np.ceil(np.log2(amax[some] / TOP)), -100.0)
        # (the logarithm may land beside a whole number: the smallest power of two that is large enough decides)
        e = np.where(np.exp2(e - 1) * TOP >= amax, np.maximum(e - 1, -100.0), e)
        e = np.where(np.exp2(e) * TOP < amax, e + 1, e)
        s = torch.from_numpy(np.exp2(e)).to(x.device)[:, None]
        v = part / s
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=1e-30))), min=-6.0) - 3.0)
        out[:, b:b + BLOCK] = torch.round(v / step) * step * s
    return out


def _full(q, scales):
    m, k = q.shape
    w = q.to(torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= float(scales[i, j])
    return w


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["kind"] == "route":
        z = state["logits"].cpu().numpy().astype(np.float64)
        n, E = z.shape
        if case["score"] == "softmax":
            s = np.exp(z - z.max(1)[:, None])
            s /= s.sum(1)[:, None]
        else:
            s = 1.0 / (1.0 + np.exp(-z))
        c = s + (state["bias_values"].cpu().numpy().astype(np.float64) if case["bias"] else 0.0)
        if case["groups"] > 1:
            parts = np.split(c, case["groups"], axis=1)
            score = np.stack([np.sort(p, axis=1)[:, ::-1][:, :case["group_best"]].sum(1) for p in parts], axis=1)
            order = np.argsort(-score, axis=1, kind="stable")[:, case["top_groups"]:]
            for row in range(n):
                for g in order[row]:
                    size = E // case["groups"]
                    c[row, g * size:(g + 1) * size] = -np.inf
        choice = np.argsort(-c, axis=1, kind="stable")[:, :case["top"]]
        w = np.take_along_axis(s, choice, axis=1)
        if case["renormalise"]:
            w = w / (w.sum(1)[:, None] + 1e-20)
        return choice.astype(np.int32), np.ascontiguousarray((w * case["scale"]).T)
    if case["kind"] == "linear":
        x = _grid(state["x_values"].double())
        products = [x @ _full(q, s).t() for q, s in zip(state["q"], state["scales"])]
        if case["epilogue"] == "gated":
            g, u = products
            return g / (1.0 + torch.exp(-g)) * u
        return products[0]
    x = _grid(state["x_values"].double())
    out = torch.zeros(case["n"], case["width"], dtype=torch.float64, device="cuda")
    choice = state["choice"].cpu().numpy()
    for e in range(case["experts"]):
        rows, ks = np.nonzero(choice == e)
        if len(rows) == 0:
            continue
        gate, up, down = (_full(state[key][0][e], state[key][1][e]) for key in ("gate", "up", "down"))
        at = torch.from_numpy(rows).cuda()
        g, u = x[at] @ gate.t(), x[at] @ up.t()
        z = _grid(g / (1.0 + torch.exp(-g)) * u)
        w = state["weights"][torch.from_numpy(ks).cuda(), at].double()
        out.index_add_(0, at, w[:, None] * (z @ down.t()))
    return out
