"""8-bit weights on the CPU: what they stand for, how matrices are stacked, checkpoints that hold them, and what is refused."""
from __future__ import annotations

import json

import pytest
import torch

import plain_fp8 as plain

CONFIG = {
    "architectures": ["LlamaForCausalLM"], "hidden_size": 256, "intermediate_size": 200, "num_hidden_layers": 2, "num_attention_heads": 4,
    "num_key_value_heads": 2, "head_dim": 64, "vocab_size": 300, "rope_theta": 10000.0, "tie_word_embeddings": True, "rms_norm_eps": 1e-5,
    "max_position_embeddings": 512, "quantization_config": {"quant_method": "fp8", "weight_block_size": [128, 128], "activation_scheme": "dynamic"},
}


def _weight(M, K, seed=0):
    from stride_b200.kernels.linear import Fp8Weight
    return Fp8Weight.quantize(torch.randn(M, K, generator=torch.Generator().manual_seed(seed)))


@pytest.mark.parametrize("M,K", [(1, 1), (128, 128), (130, 257), (300, 15), (64, 640)])
def test_what_a_weight_stands_for(M, K):
    w = torch.randn(M, K, generator=torch.Generator().manual_seed(M))
    from stride_b200.kernels.linear import Fp8Weight
    got = Fp8Weight.quantize(w)
    values = plain.weight_values(got.q[:, :K].float(), got.scales)
    assert (values - w.double()).abs().max() <= 2.0 ** -4 * w.abs().max()           # half a step of the largest element
    assert (got.to(torch.float32).double() - values).abs().max() <= 2.0 ** -24 * values.abs().max()
    assert got.stride % 16 == 0 and got.stride >= K and got.q.data_ptr() % 16 == 0
    if got.stride > K:
        assert (got.q.view(torch.uint8)[:, K:] == 0).all()


def test_a_block_of_zeros_and_columns_of_a_wider_matrix():
    from stride_b200.kernels.linear import Fp8Weight
    w = torch.zeros(200, 300)
    w[130:, :100] = 3.0
    got = Fp8Weight.quantize(w)
    assert torch.equal(got.to(torch.float32), w)
    inner = Fp8Weight(got.q[:, :300], got.scales)
    assert torch.equal(inner.to(torch.float32), w)
    narrow = Fp8Weight(got.q[:64, :128], got.scales[:1, :1])
    assert torch.equal(narrow.to(torch.float32), w[:64, :128])


def test_stacked_weights():
    from stride_b200.kernels.linear import Fp8Weight
    a, b, c = _weight(256, 100, 1), _weight(128, 100, 2), _weight(70, 100, 3)
    stacked = Fp8Weight.stack([a, b, c])
    assert stacked.in_blocks and stacked.halves == 1
    assert torch.equal(stacked.to(torch.float32), torch.cat([w.to(torch.float32) for w in (a, b, c)]))
    pair = Fp8Weight.stack([c, _weight(70, 100, 4)])
    assert pair.halves == 2 and not pair.in_blocks
    assert torch.equal(pair.to(torch.float32)[:70], c.to(torch.float32))
    assert torch.equal(pair.to(torch.float32)[70:], _weight(70, 100, 4).to(torch.float32))
    with pytest.raises(ValueError, match="cannot be stacked"):
        Fp8Weight.stack([c, a])
    with pytest.raises(ValueError, match="same number of columns"):
        Fp8Weight.stack([a, _weight(128, 101)])
    with pytest.raises(ValueError, match="plain matrices"):
        Fp8Weight.stack([pair, c])


def test_weights_that_are_refused():
    from stride_b200.kernels.linear import Fp8Experts, Fp8Weight
    w = _weight(130, 129)
    with pytest.raises(TypeError):
        Fp8Weight(torch.zeros(4, 4), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="scales"):
        Fp8Weight(w.q[:, :129], w.scales[:1])
    with pytest.raises(ValueError, match="scales"):
        Fp8Weight(w.q[:, :129], w.scales.double())
    with pytest.raises(ValueError, match="gate and an up matrix"):
        Fp8Experts([w, w], [w])
    with pytest.raises(ValueError, match="gate and an up matrix"):
        Fp8Experts([_weight(8, 16)], [_weight(16, 8)])


def test_calls_without_a_device_are_refused():
    from stride_b200.kernels import ops
    from stride_b200.kernels.linear import Linear
    from stride_b200.parts.context import Workspace
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.route_experts(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(1, 2))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.quantize_fp8(torch.zeros(2, 16), torch.zeros(2, 16).to(torch.float8_e4m3fn), torch.zeros(1, 2))
    layer = Linear(_weight(128, 64), torch.bfloat16)
    with pytest.raises(ValueError, match="workspace"):
        layer.forward(torch.zeros(2, 64), torch.zeros(2, 128))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer.forward(torch.zeros(2, 64), torch.zeros(2, 128), workspace=Workspace(torch.device("cpu"), 2))


def test_a_stacked_weight_that_has_only_the_gated_product_is_no_plain_layer_of_a_program():
    from types import SimpleNamespace
    from stride_b200.kernels.linear import Fp8Weight, Linear
    from stride_b200.parts.context import Workspace
    added = []
    program = SimpleNamespace(workspace=Workspace(torch.device("cpu"), 2), h=torch.zeros(2, 128), take_fresh=lambda: None, need_folded=lambda what: None,
                              add=lambda *a, **k: added.append(a))
    layer = Linear(Fp8Weight.stack([_weight(64, 32), _weight(64, 32)]), torch.bfloat16)
    x, flat = torch.zeros(2, 32), torch.zeros(256)
    with pytest.raises(ValueError, match="only has the gated product"):
        layer.emit_partials(program, x, flat)
    with pytest.raises(ValueError, match="only has the gated product"):
        layer.emit(program, x, flat.view(2, 128))
    with pytest.raises(ValueError, match="only has the gated product"):
        layer.emit_add(program, x)
    assert not added


def test_the_float32_engine_takes_what_the_weight_stands_for():
    from stride_b200.kernels.linear import Linear
    w = _weight(130, 200)
    layer = Linear(w, torch.float32)
    assert layer.fp8 is None and torch.equal(layer.weight, w.to(torch.float32))


def test_checkpoint_with_8_bit_matrices(tmp_path):
    from stride_b200.kernels.linear import Fp8Weight
    from stride_b200.weights.loader import load_weights
    from stride_b200.weights.random_init import model_plan, random_tensors, write_random_model
    folder = write_random_model(tmp_path / "m", CONFIG, 3)
    plan = model_plan(CONFIG)
    loaded = load_weights(folder, plan, "cpu")
    assert set(loaded) == {n for n in plan if n != "lm_head.weight"}
    given = random_tensors(CONFIG, 3)
    for name, want in plan.items():
        if name not in loaded:
            continue
        assert isinstance(loaded[name], Fp8Weight) == want.fp8
        if want.fp8:
            assert torch.equal(loaded[name].q[:, :want.shape[1]].view(torch.uint8), given[name].view(torch.uint8))
            assert torch.equal(loaded[name].scales, given[name + "_scale_inv"])
        else:
            assert torch.equal(loaded[name], given[name])
    header = json.loads((folder / "model.safetensors").read_bytes()[8:8 + int.from_bytes((folder / "model.safetensors").read_bytes()[:8], "little")])
    assert header["model.layers.0.mlp.up_proj.weight"]["dtype"] == "F8_E4M3"


@pytest.mark.parametrize("break_it,match", [
    (lambda t: t.pop("model.layers.0.mlp.up_proj.weight_scale_inv"), "missing tensors"),
    (lambda t: t.update({"model.layers.0.mlp.up_proj.weight_scale_inv": torch.ones(1, 2)}), "wrong shapes"),
    (lambda t: t.update({"model.norm.weight_scale_inv": torch.ones(1, 1)}), "unexpected tensors"),
    (lambda t: t.update({"model.embed_tokens.weight": t["model.embed_tokens.weight"].to(torch.float8_e4m3fn),
                         "model.embed_tokens.weight_scale_inv": torch.ones(3, 2)}), "does not take")])
def test_checkpoints_that_do_not_fit(tmp_path, break_it, match):
    from stride_b200.weights.loader import WeightsError, load_weights
    from stride_b200.weights.random_init import model_plan, random_tensors
    from stride_b200.weights.safetensors_io import write_safetensors
    tensors = random_tensors(CONFIG, 3)
    break_it(tensors)
    write_safetensors(tmp_path / "model.safetensors", tensors)
    with pytest.raises(WeightsError, match=match):
        load_weights(tmp_path, model_plan(CONFIG), "cpu")


@pytest.mark.parametrize("change", [{"quant_method": "awq"}, {"weight_block_size": [64, 128]}, {"weight_block_size": None}, {"activation_scheme": "static"},
                                    {"fmt": "e5m2"}])
def test_quantisations_that_are_refused(change):
    from stride_b200.config.llama import ConfigError, LlamaConfig
    LlamaConfig.from_dict(CONFIG)
    with pytest.raises(ConfigError, match="quantization_config"):
        LlamaConfig.from_dict({**CONFIG, "quantization_config": {**CONFIG["quantization_config"], **change}})


def _experts_spec(**params):
    from stride_b200.parts import PartSpec
    names = {r: tuple(f"e{e}.{r}" for e in range(8)) for r in ("gate", "up", "down")}
    return PartSpec("scored_experts", {"hidden_size": 64, "intermediate_size": 32, "experts": 8, "top": 2, **params}, {"router": "router", **names})


@pytest.mark.parametrize("params", [{"top": 9}, {"top": 0}, {"groups": 3}, {"groups": 4, "top_groups": 5}, {"groups": 4, "top_groups": 1, "top": 3},
                                    {"group_best": 3}, {"score": "relu"}])
def test_scored_experts_that_are_refused(params):
    from stride_b200.parts import BuildEnv, part_class
    env = BuildEnv(torch.device("cpu"), torch.bfloat16, 8, 64)
    part_class("feed_forward", "scored_experts")(_experts_spec(groups=4, top_groups=2), env)
    with pytest.raises(ValueError, match="scored experts"):
        part_class("feed_forward", "scored_experts")(_experts_spec(**params), env)


def test_scored_experts_take_8_bit_matrices_in_the_bfloat16_engine():
    from stride_b200.parts import BuildEnv, part_class
    make = part_class("feed_forward", "scored_experts")
    with pytest.raises(ValueError, match="bfloat16 engine"):
        make(_experts_spec(), BuildEnv(torch.device("cpu"), torch.float32, 8, 64))
    part = make(_experts_spec(), BuildEnv(torch.device("cpu"), torch.bfloat16, 8, 64))
    tensors = {n: torch.zeros(p.shape, dtype=torch.bfloat16) for n, p in part.tensor_plan().items()}
    with pytest.raises(TypeError, match="8 bits"):
        part.bind(tensors)


OTHER = {"quant_method": "fp8", "weight_block_size": [64, 128], "activation_scheme": "dynamic"}


@pytest.mark.parametrize("given", [OTHER, {"quant_method": "awq", "bits": 4}, {"kv_cache_scheme": {"num_bits": 8}}, "none"])
def test_a_quantisation_of_another_kind_counts_only_where_matrices_are_in_8_bits(tmp_path, given):
    """Plain matrices load whatever the key says, and random ones are written plain; 8-bit ones beside it are refused by name."""
    from stride_b200.config import ConfigError, resolve_architecture
    from stride_b200.weights.loader import load_weights
    from stride_b200.weights.random_init import model_plan, random_tensors, write_random_model
    from stride_b200.weights.safetensors_io import write_safetensors
    config = {**CONFIG, "quantization_config": given}
    assert resolve_architecture(config).parse_config(config).hidden_size == CONFIG["hidden_size"]
    folder = write_random_model(tmp_path / "m", config, 3)
    plan = model_plan(config)
    loaded = load_weights(folder, plan, "cpu", config)
    assert all(isinstance(t, torch.Tensor) and t.dtype == torch.bfloat16 for t in loaded.values())
    write_safetensors(folder / "model.safetensors", random_tensors(CONFIG, 3))
    with pytest.raises(ConfigError, match="is stored in 8 bits; .*quantization_config needs"):
        load_weights(folder, plan, "cpu", config)
    assert load_weights(folder, plan, "cpu", CONFIG)


def test_random_weights_of_other_designs_go_by_the_form_too():
    from stride_b200.weights.random_init import random_tensors
    from keralorn_cases import KERALORN_P
    plain_names = set(random_tensors(KERALORN_P, 1))
    assert set(random_tensors({**KERALORN_P, "quantization_config": OTHER}, 1)) == plain_names
    assert set(random_tensors({**KERALORN_P, "quantization_config": CONFIG["quantization_config"]}, 1)) >= plain_names


def test_weights_on_several_devices_are_refused():
    """(The kernels get addresses: one of another device's memory, or of the host's, must not reach them.)"""
    from stride_b200.kernels.linear import Fp8Experts, Fp8Weight
    w = _weight(128, 64)
    with pytest.raises(ValueError, match="has its scales there too"):
        Fp8Weight(w.q, w.scales.to("meta"))
    elsewhere = Fp8Weight(torch.empty(64, 128, dtype=torch.float8_e4m3fn, device="meta"), torch.empty(1, 1, device="meta"))
    with pytest.raises(ValueError, match="all on one device"):
        Fp8Experts([w, w], [elsewhere])


def test_calls_with_tensors_beside_the_current_device_are_refused(monkeypatch):
    """Tensors of two devices, or of one that is not the current: refused before anything is launched (devices made up on the host)."""
    from types import SimpleNamespace
    from stride_b200.kernels import ops

    class On(torch.Tensor):
        """A host tensor that says it lies on a CUDA device."""
        at = 0
        is_cuda = True
        device = property(lambda self: torch.device("cuda", self.at))

        def get_device(self):
            return self.at

    def on(at, *shape, dtype=torch.float32):
        t = torch.zeros(*shape).to(dtype).as_subclass(On)
        t.at = at
        return t

    monkeypatch.setattr(ops, "_fn", lambda *a: (None, lambda *args: pytest.fail("launched")))
    monkeypatch.setattr(ops, "_device", lambda: 0)
    for where in ([1] * 6, [0, 1, 0, 0, 0, 0], [0, 0, 1, 0, 0, 0], [0, 0, 0, 1, 0, 0], [0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 0, 1]):
        a, b, c, d, e, f = where
        weight = SimpleNamespace(q=on(c, 128, 16, dtype=torch.float8_e4m3fn), scales=on(c, 1, 1), shape=(128, 16), stride=16, halves=1, in_blocks=True)
        q, scales = on(a, 2, 16, dtype=torch.float8_e4m3fn), on(b, 1, 2)
        if 1 in where[:3]:
            with pytest.raises(ValueError, match="quantize_fp8: tensors on .*the current device is cuda:0"):
                ops.quantize_fp8(on(c, 2, 16), q, scales)
        if 1 in where[:4]:
            with pytest.raises(ValueError, match="gemm_fp8: tensors on"):
                ops.gemm_fp8(q, scales, weight, on(d, 2, 128))
            with pytest.raises(ValueError, match="linear_fp8: tensors on"):
                ops.Fp8Linear(weight, q, scales)(on(d, 2, 16), on(a, 2, 128))
            with pytest.raises(ValueError, match="linear_fp8: tensors on"):
                ops.Fp8Linear(weight, q, scales)(on(a, 2, 16), on(d, 2, 128))
            with pytest.raises(ValueError, match="route_experts: tensors on"):
                ops.route_experts(on(a, 2, 4), on(b, 2, 1, dtype=torch.int32), on(c, 1, 2), bias=on(d, 4))
        layer = SimpleNamespace(at=a, down=on(a, 16, 16), width=16, address=0)
        with pytest.raises(ValueError, match="experts_fp8: tensors on"):
            ops.experts_fp8(on(b, 2, 16), on(c, 2, 1, dtype=torch.int32), on(d, 1, 2), layer, on(e, 2, 16), on(f, 64, dtype=torch.uint8))


def test_experts_of_stacked_matrices():
    """A stacked matrix whose second half's scales begin beside a multiple of 128 rows has more blocks of scales than an expert's is read with."""
    from stride_b200.kernels.linear import Fp8Experts, Fp8Weight
    stacked, down = Fp8Weight.stack([_weight(100, 64, 1), _weight(100, 64, 2)]), _weight(64, 200)
    assert stacked.shape == (200, 64) and stacked.scales.shape[0] == 2
    narrow = Fp8Weight.stack([_weight(40, 64, 1), _weight(40, 64, 2)])          # (two blocks of scales where 80 rows have one)
    with pytest.raises(ValueError, match="plain ones"):
        Fp8Experts([narrow, narrow], [_weight(64, 80)])
    with pytest.raises(ValueError, match="plain ones"):
        Fp8Experts([stacked, stacked], [down])
    whole = Fp8Weight.stack([_weight(128, 64, 1), _weight(128, 64, 2)])
    layer = Fp8Experts([whole, whole], [_weight(64, 256)])
    assert layer.gate_up_scales.shape[0] == 4 and layer.inner == 256


def test_random_weights_of_a_model_with_scored_experts():
    """A part that runs in the bfloat16 engine alone has a plan, and random weights, like any other."""
    from stride_b200.weights.random_init import model_plan, random_tensors
    from test_scored_experts_gpu import CONFIG as SCORED, architecture
    with architecture():
        plan, tensors = model_plan(SCORED), random_tensors(SCORED, 3)
    name = "model.layers.1.mlp.experts.15.down_proj.weight"
    assert plan[name].fp8 and tensors[name].dtype == torch.float8_e4m3fn and tensors[name + "_scale_inv"].shape == (2, 2)
    assert not plan["model.layers.1.mlp.gate.weight"].fp8
