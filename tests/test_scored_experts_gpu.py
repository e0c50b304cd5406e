"""The feed-forward of scored experts as a checkpoint in 8 bits has it: its shared expert in 8 bits too, and whole models of it under both step drivers."""
from __future__ import annotations

import contextlib
import dataclasses

import pytest
import torch

import plain_fp8 as plain
import plain_llama
from conftest import TEST_GAIN_STD, TEST_STD, random_tokens
from test_fp8 import CONFIG as LLAMA
from test_fp8_model_gpu import QuantisedInput, _engine, _logits

pytestmark = pytest.mark.gpu

BF, F64 = torch.bfloat16, torch.float64
DEV = "cuda"


def _values(w):
    return plain.weight_values(w.q[:, :w.shape[1]].float(), w.scales)


def _shared(x, gate, up, down):
    """(out, bound) of the shared expert: its gated product is rounded to bfloat16 and quantised again for the down product."""
    z, ez = plain.gated(plain.quantised_values(x), gate, up)
    stored = z.to(BF).to(F64)
    zv = plain.quantised_values(stored)
    # (what is stored may be the neighbouring bfloat16 value, a whole step off)
    slack = plain.requantised_slack(stored, ez + 2.0 ** -7 * z.abs())
    return zv @ down.T, plain.product_bound(zv, down) + slack @ down.abs().T


@pytest.mark.parametrize("W,F,shared", [(256, 136, 128), (256, 200, 136), (384, 128, 72)])
@pytest.mark.parametrize("n", [1, 20, 100, 250])
def test_shared_expert_in_8_bits(W, F, shared, n):
    from stride_b200.kernels.linear import Fp8Weight
    from stride_b200.parts import BuildEnv, PartSpec, ResidualStream, Workspace, part_class
    from stride_b200.parts.context import step_context
    E, top = 12, 3
    g = torch.Generator().manual_seed(W + n)
    rnd = lambda *shape, std=1.0: std * torch.randn(*shape, generator=g)
    names = {r: tuple(f"e{e}.{r}" for e in range(E)) for r in ("gate", "up", "down")}
    t = {"router": rnd(E, W, std=W ** -0.5).to(BF)}
    for prefix, inner in [(f"e{e}", F) for e in range(E)] + [("s", shared)]:
        for r, shape in (("gate", (inner, W)), ("up", (inner, W)), ("down", (W, inner))):
            t[f"{prefix}.{r}"] = Fp8Weight.quantize(rnd(*shape, std=shape[1] ** -0.5).to(DEV))
    tensors = {"router": "router", **names, **{f"shared_{r}": f"s.{r}" for r in ("gate", "up", "down")}}
    spec = PartSpec("scored_experts", {"hidden_size": W, "intermediate_size": F, "experts": E, "top": top, "shared": shared}, tensors)
    part = part_class("feed_forward", "scored_experts")(spec, BuildEnv(torch.device(DEV), BF, 256, 512))
    assert all(p.fp8 for name, p in part.tensor_plan().items() if name != "router")
    part.bind({k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in t.items()})
    ws, x, base = Workspace(DEV, 256), rnd(n, W).to(BF), rnd(n, W)

    def run(rows):
        ctx = step_context([(1, len(rows), 0)], ws, BF, [1] * len(rows))
        stream = ResidualStream(base[rows].to(DEV))
        part.forward(ctx, x[rows].to(DEV), stream)
        stream.fold()
        return stream.h.cpu()

    got = run(list(range(n)))
    z = x.double() @ t["router"].double().T
    choice, weights = plain.route(z, top, "sigmoid")
    clear = torch.ones(n, dtype=torch.bool)
    for sign in (-1.0, 1.0):          # (tokens whose choice the router's 32-bit sums may make otherwise)
        clear &= (plain.route(z + sign * 1e-5 * torch.randn(n, E, generator=g, dtype=F64), top, "sigmoid")[0] == choice).all(dim=1)
    assert clear.float().mean() >= 0.9
    want, bound = plain.experts(x.to(DEV, F64), choice.to(DEV), weights.to(DEV), *([_values(t[f"e{e}.{r}"]) for e in range(E)] for r in ("gate", "up", "down")))
    bound = bound + 2.0 ** -18 * top * want.abs().amax(dim=1, keepdim=True)          # a weight is off by 2^-18 of itself at most
    more, more_bound = _shared(x.to(DEV, F64), *(_values(t[f"s.{r}"]) for r in ("gate", "up", "down")))
    total = (base.to(DEV, F64) + want + more).cpu()
    ok = (got.double() - total).abs() <= (bound + more_bound).cpu() + 2.0 ** -21 * (total.abs() + base.double().abs() + more.cpu().abs())
    assert ok[clear].all()
    for i in sorted({0, n // 2, n - 1}):
        assert torch.equal(run([i])[0], got[i]), f"row {i} alone differs from the row in company"


# ------------------------------------------------------------------ whole models
E, TOP, F, SHARED = 16, 3, 136, 128
CONFIG = {**LLAMA, "architectures": ["ScoredExpertsForTest"], "intermediate_size": 256}


@contextlib.contextmanager
def architecture():
    """A Llama whose feed-forwards are scored experts, registered as an architecture of its own."""
    from stride_b200.config import Architecture, LlamaConfig, register_architecture, registry
    from stride_b200.config.llama_spec import llama_model_spec
    from stride_b200.parts import PartSpec
    from stride_b200.parts.spec import LayerSpec

    def spec(cfg):
        base = llama_model_spec(cfg)
        layers = []
        for i, layer in enumerate(base.layers):
            p = f"model.layers.{i}.mlp."
            names = {r: tuple(f"{p}experts.{e}.{r}_proj.weight" for e in range(E)) for r in ("gate", "up", "down")}
            names.update({f"shared_{r}": f"{p}shared_experts.{r}_proj.weight" for r in ("gate", "up", "down")})
            ff = PartSpec("scored_experts", {"hidden_size": cfg.hidden_size, "intermediate_size": F, "experts": E, "top": TOP, "groups": 4, "top_groups": 2,
                                             "scale": 2.5, "shared": SHARED},
                          {"router": p + "gate.weight", "bias": p + "gate.e_score_correction_bias", **names})
            layers.append(LayerSpec(layer.block, {**layer.parts, "feed_forward": ff}))
        return dataclasses.replace(base, layers=tuple(layers))

    register_architecture(Architecture("ScoredExpertsForTest", LlamaConfig.from_dict, spec))
    try:
        yield
    finally:
        del registry._ARCHITECTURES["ScoredExpertsForTest"]


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from stride_b200.weights.random_init import write_random_model
    with architecture():
        yield write_random_model(tmp_path_factory.mktemp("scored") / "m", CONFIG, 11, std=TEST_STD, gain_std=TEST_GAIN_STD)


def test_model_does_not_depend_on_the_portions_or_the_driver(folder):
    """The same bits whole and in portions, from the native program and part by part."""
    tokens = random_tokens(CONFIG["vocab_size"], 200, 2)
    native, python = _engine(folder), _engine(folder, native_step=False)
    assert native._program is not None and python._program is None
    want = _logits(native, tokens, [200])
    assert torch.isfinite(want).all()
    for engine, portions in ((native, [1] * 20 + [16, 17, 33, 64, 50]), (native, [130, 70]), (python, [200]), (python, [40, 1, 1, 100, 58])):
        assert torch.equal(_logits(engine, tokens, portions), want), portions


def test_generation_with_experts_does_not_depend_on_company(folder):
    """Greedy tokens of requests side by side (decode steps from recorded graphs) and alone."""
    from stride_b200 import LLM
    llm = LLM(str(folder), dtype="bfloat16", max_rows=64, max_slots=6, kv_pages=64, page_size=16)
    prompts = [random_tokens(CONFIG["vocab_size"], n, 10 + n) for n in (5, 33, 70, 1)]
    together = [o.tokens for o in llm.generate(prompts, max_new_tokens=12)]
    assert llm.engine.graph_replays > 0
    for prompt, tokens in zip(prompts, together):
        assert llm.generate([prompt], max_new_tokens=12)[0].tokens == tokens


class Experts:
    """The feed-forward in the place of a down projection: `x @ experts.to(dtype).T` of the plain implementation, whose gated product is x itself."""
    T = property(lambda self: self)

    def __init__(self, loaded, prefix, quantised):
        self.router, self.bias, self.quantised = loaded[prefix + "gate.weight"].to(F64), loaded[prefix + "gate.e_score_correction_bias"], quantised
        take = lambda name: _values(loaded[f"{prefix}{name}_proj.weight"])
        self.matrices = [[take(f"experts.{e}.{r}") for e in range(E)] for r in ("gate", "up", "down")]
        self.shared = [take(f"shared_experts.{r}") for r in ("gate", "up", "down")]

    def to(self, dtype):
        return self

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        x, self = args
        x, dtype = x.to(F64), x.dtype
        choice, weights = plain.route(x @ self.router.T, TOP, "sigmoid", self.bias, 4, 2, 2, True, 2.5)
        if self.quantised:
            out = plain.experts(x, choice, weights, *self.matrices)[0] + _shared(x, *self.shared)[0]
        else:
            out = plain.silu(x @ self.shared[0].T) * (x @ self.shared[1].T) @ self.shared[2].T
            for e, (gate, up, down) in enumerate(zip(*self.matrices)):
                rows, ks = torch.nonzero(choice == e, as_tuple=True)
                out.index_add_(0, rows, weights[ks, rows][:, None] * ((plain.silu(x[rows] @ gate.T) * (x[rows] @ up.T)) @ down.T))
        return out.to(dtype)


def test_model_against_the_plain_implementation(folder, monkeypatch):
    """By the median over tokens: rounding may give a token another expert, and then its logits are others."""
    from stride_b200.kernels.linear import Fp8Weight
    from stride_b200.weights.loader import load_weights
    from stride_b200.weights.random_init import model_plan
    monkeypatch.setattr(plain_llama, "swiglu", lambda x, gate, up: x)
    loaded = load_weights(folder, model_plan(CONFIG), "cpu", CONFIG)
    cfg, tokens = plain_llama.PlainConfig.from_dict(CONFIG), random_tokens(CONFIG["vocab_size"], 150, 1)

    def forward(quantised, act_dtype):
        w = {n: (QuantisedInput(_values(t)) if quantised else _values(t).float()) if isinstance(t, Fp8Weight) else t.float() for n, t in loaded.items()}
        for i in range(cfg.num_hidden_layers):
            p = f"model.layers.{i}.mlp."
            w.update({p + "gate_proj.weight": None, p + "up_proj.weight": None, p + "down_proj.weight": Experts(loaded, p, quantised)})
        return plain_llama.forward(cfg, w, tokens, act_dtype=act_dtype)

    exact, want = forward(False, None), forward(True, BF)
    got = _logits(_engine(folder), tokens, [150]).cpu()
    off, noise = (got - want).abs().mean(dim=1), (want - exact).abs().mean(dim=1)
    assert off.median() <= 0.5 * noise.median()
