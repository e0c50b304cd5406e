"""8-bit weights inside the engine: a Llama whose projections are stored in 8 bits, and the feed-forward of scored experts, against the plain
implementations with the inputs of those products quantised at the same places."""
from __future__ import annotations

import pytest
import torch

import plain_fp8 as plain
import plain_llama
from conftest import TEST_GAIN_STD, TEST_STD, logit_tolerance, random_tokens
from test_fp8 import CONFIG

pytestmark = pytest.mark.gpu

BF, F64 = torch.bfloat16, torch.float64
DEV = "cuda"


class QuantisedInput:
    """A weight that quantises what it is multiplied with: `x @ weight.to(dtype).T` of the plain implementation."""

    def __init__(self, values):
        self.values = values

    def to(self, dtype):
        return self

    T = property(lambda self: self)

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        x, w = args
        return (plain.quantised_values(x.to(F64)) @ w.values.T).to(x.dtype)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    """(folder, plain configuration, plain weights as they stand, the same with quantised inputs)."""
    from stride_b200.kernels.linear import Fp8Weight
    from stride_b200.weights.loader import load_weights
    from stride_b200.weights.random_init import model_plan, write_random_model
    folder = write_random_model(tmp_path_factory.mktemp("fp8") / "m", CONFIG, 7, std=TEST_STD, gain_std=TEST_GAIN_STD)
    loaded = load_weights(folder, model_plan(CONFIG), "cpu")
    whole = {n: w.to(torch.float32) for n, w in loaded.items()}
    rounded = {n: QuantisedInput(plain.weight_values(w.q[:, :w.shape[1]].float(), w.scales)) if isinstance(w, Fp8Weight) else whole[n] for n, w in loaded.items()}
    return folder, plain_llama.PlainConfig.from_dict(CONFIG), whole, rounded


def _engine(folder, dtype="bfloat16", **kw):
    from stride_b200 import Engine, EngineOptions
    return Engine(folder, EngineOptions(dtype=dtype, max_rows=256, max_full_rows=256, max_slots=6, kv_pages=64, page_size=16, **kw))


def _logits(engine, tokens, portions):
    from stride_b200 import StepEntry
    slot, at, out = engine.cache.acquire_slot(), 0, []
    for n in portions:
        assert engine.cache.ensure(slot, at + n)
        out.append(engine.step([StepEntry(slot, at, tokens[at:at + n], list(range(n)))]).clone())
        at += n
    engine.cache.release_slot(slot)
    return torch.cat(out)


def test_logits_against_the_plain_implementation(model):
    folder, cfg, whole, rounded = model
    tokens = random_tokens(CONFIG["vocab_size"], 150, 1)
    exact = plain_llama.forward(cfg, whole, tokens)
    got = _logits(_engine(folder, "float32"), tokens, [150]).cpu()
    assert (got - exact).abs().max() <= logit_tolerance("float32", exact)
    want = plain_llama.forward(cfg, rounded, tokens, act_dtype=BF)
    noise = (want - exact).abs()
    got = _logits(_engine(folder), tokens, [150]).cpu()
    assert (got - want).abs().max() <= logit_tolerance("bfloat16", want, float(noise.max()))
    assert (got - want).abs().mean() <= 0.5 * float(noise.mean())


def test_logits_do_not_depend_on_the_portions_or_the_driver(model):
    folder = model[0]
    tokens = random_tokens(CONFIG["vocab_size"], 200, 2)
    native, python = _engine(folder), _engine(folder, native_step=False)
    assert native._program is not None and python._program is None
    want = _logits(native, tokens, [200])
    for engine, portions in ((native, [1] * 20 + [16, 17, 33, 64, 50]), (native, [130, 70]), (python, [200]), (python, [40, 1, 1, 100, 58])):
        assert torch.equal(_logits(engine, tokens, portions), want), portions


def test_generation_does_not_depend_on_company(model):
    """Greedy tokens of requests side by side (decode steps from recorded graphs) and alone."""
    from stride_b200 import LLM
    llm = LLM(str(model[0]), dtype="bfloat16", max_rows=64, max_slots=6, kv_pages=64, page_size=16)
    prompts = [random_tokens(CONFIG["vocab_size"], n, 10 + n) for n in (5, 33, 70, 1)]
    together = [o.tokens for o in llm.generate(prompts, max_new_tokens=12)]
    for prompt, tokens in zip(prompts, together):
        assert llm.generate([prompt], max_new_tokens=12)[0].tokens == tokens


@pytest.mark.parametrize("rows", [96, 200])
def test_projections_whose_matrices_cannot_be_stacked_are_refused(tmp_path, rows):
    """Heads whose queries are no whole number of 128 rows: the bfloat16 engine says so, the float32 engine runs them."""
    from stride_b200.weights.random_init import write_random_model
    config = {**CONFIG, "num_attention_heads": rows // 8, "num_key_value_heads": rows // 8, "head_dim": 8, "num_hidden_layers": 1}
    folder = write_random_model(tmp_path / "m", config, 1)
    with pytest.raises(ValueError, match="cannot be stacked"):
        _engine(folder)
    assert torch.isfinite(_logits(_engine(folder, "float32"), [1, 2, 3], [3])).all()


EXPERTS = [(64, 8, 2, 32, 0, {}), (256, 16, 4, 200, 136, {"groups": 4, "top_groups": 2, "scale": 2.5}), (200, 12, 3, 264, 0, {"score": "softmax", "renormalise": False}),
           (128, 64, 6, 128, 64, {"groups": 8, "top_groups": 3, "group_best": 1})]


@pytest.mark.parametrize("W,E,top,F,shared,params", EXPERTS)
@pytest.mark.parametrize("n", [1, 37, 250])
@pytest.mark.parametrize("biased", [False, True])
def test_scored_experts(W, E, top, F, shared, params, n, biased):
    """The part alone, adding to a stream; a token alone in the same bits."""
    from stride_b200.kernels.linear import Fp8Weight
    from stride_b200.parts import BuildEnv, PartSpec, ResidualStream, Workspace, part_class
    from stride_b200.parts.context import step_context
    g = torch.Generator().manual_seed(W + E + n)
    rnd = lambda *shape, std=1.0: std * torch.randn(*shape, generator=g)
    names = {r: tuple(f"e{e}.{r}" for e in range(E)) for r in ("gate", "up", "down")}
    t = {"router": rnd(E, W, std=W ** -0.5).to(BF), **({"bias": rnd(E, std=0.1)} if biased else {})}
    for e in range(E):
        for r, shape in (("gate", (F, W)), ("up", (F, W)), ("down", (W, F))):
            t[f"e{e}.{r}"] = Fp8Weight.quantize(rnd(*shape, std=shape[1] ** -0.5).to(DEV))
    tensors = {"router": "router", **({"bias": "bias"} if biased else {}), **names}
    if shared:
        tensors.update({f"shared_{r}": f"s.{r}" for r in ("gate", "up", "down")})
        for r, shape in (("gate", (shared, W)), ("up", (shared, W)), ("down", (W, shared))):
            t[f"s.{r}"] = rnd(*shape, std=shape[1] ** -0.5).to(BF)
    spec = PartSpec("scored_experts", {"hidden_size": W, "intermediate_size": F, "experts": E, "top": top, "shared": shared, **params}, tensors)
    part = part_class("feed_forward", "scored_experts")(spec, BuildEnv(torch.device(DEV), BF, 256, 512))
    assert set(part.tensor_plan()) == set(t)
    part.bind({k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in t.items()})
    ws = Workspace(DEV, 256)
    x, base = rnd(n, W).to(BF), rnd(n, W)

    def run(rows):
        ctx = step_context([(1, len(rows), 0)], ws, BF, [1] * len(rows))
        stream = ResidualStream(base[rows].to(DEV))
        part.forward(ctx, x[rows].to(DEV), stream)
        stream.fold()
        return stream.h.cpu()

    got = run(list(range(n)))
    z = x.double() @ t["router"].double().T
    kw = {k: v for k, v in params.items() if k != "score"}
    choice, weights = plain.route(z, top, params.get("score", "sigmoid"), t.get("bias"), **kw)
    # (the router's 32-bit sums may choose otherwise where scores are closer than they tell apart: those tokens are left out, few of them)
    clear = torch.ones(n, dtype=torch.bool)
    for sign in (-1.0, 1.0):
        nudged = z + sign * 1e-5 * torch.randn(n, E, generator=g, dtype=F64)
        clear &= (plain.route(nudged, top, params.get("score", "sigmoid"), t.get("bias"), **kw)[0] == choice).all(dim=1)
    assert clear.float().mean() >= 0.9
    values = [[plain.weight_values(w.q[:, :w.shape[1]].float(), w.scales) for w in (t[f"e{e}.{r}"] for e in range(E))] for r in ("gate", "up", "down")]
    want, bound = plain.experts(x.to(DEV, F64), choice.to(DEV), weights.to(DEV), *values)
    want, bound = want.cpu(), bound.cpu()
    # the router's products are 32-bit sums: a score, and with it a weight, is off by 2^-18 of itself at most (256 terms, unit logits)
    bound = bound + 2.0 ** -18 * top * want.abs().amax(dim=1, keepdim=True)
    if shared:
        xs = x.double()
        a, b, c = (t[f"s.{r}"].double() for r in ("gate", "up", "down"))
        inner = plain.silu(xs @ a.T) * (xs @ b.T)
        want = want + inner.to(BF).double() @ c.T
        bound = bound + 2.0 ** -7 * (inner.abs() @ c.abs().T)                   # its gated product rounded to bfloat16, sums of bfloat16 products
    total = base.double() + want
    ok = (got.double() - total).abs() <= bound + 2.0 ** -22 * (total.abs() + base.double().abs())
    assert ok[clear].all()
    for i in sorted({0, n // 2, n - 1}):
        assert torch.equal(run([i])[0], got[i]), f"row {i} alone differs from the row in company"
