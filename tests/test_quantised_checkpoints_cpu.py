"""What loading makes of checkpoints whose weights are codes: parts that stay in floating point, other schemes than the one that is multiplied in
8 bits (CPU)."""
import copy

import pytest
import torch

from gllm_b200.models import registry
from gllm_b200.models.weight_utils import CheckpointReader
from tests.test_quantised_serving_cpu import W8A8, _cfg, _state


def _load(cfg, sd):
    model = registry.build_model(cfg, "cpu")
    model.load_weights(CheckpointReader.from_state_dict(sd))
    return model


def _scheme(part, **over):
    c = copy.deepcopy(W8A8)
    c["config_groups"]["group_0"][part].update(over)
    return c


def test_a_head_in_8_bits_comes_with_its_scales():
    """The head is multiplied in the compute dtype, so its codes are taken times their scales."""
    sd = _state(_cfg(), True)
    w = sd["lm_head.weight"]
    s = w.abs().amax(1, keepdim=True) / 127
    sd["lm_head.weight"], sd["lm_head.weight_scale"] = torch.round(w / s).to(torch.int8), s
    model = _load(_cfg(quantization_config={**W8A8, "ignore": []}), sd)
    assert torch.equal(model.lm_head_w[: w.shape[0]], sd["lm_head.weight"].float() * s)
    assert float((model.lm_head_w[: w.shape[0]] - w).abs().max()) <= 0.51 * float(s.max())


@pytest.mark.parametrize("config,per_tensor", [(_scheme("weights", strategy="tensor"), True), (_scheme("input_activations", dynamic=False), False)])
def test_other_schemes_load_the_values_that_their_codes_stand_for(config, per_tensor):
    cfg = _cfg(quantization_config=config)
    sd = _state(cfg, True)
    name = "model.layers.1.mlp.down_proj.weight"
    if per_tensor:
        for k in [k for k in sd if k.endswith("weight_scale")]:
            sd[k] = sd[k].amax().reshape(1)
    model = _load(cfg, sd)
    assert model.spec.quant is None
    assert torch.equal(model.layers[1].mlp.down_w, sd[name].float() * sd[name + "_scale"].float())


def test_one_scale_for_a_tensor_is_one_for_each_channel():
    """Asked for 8-bit linears, codes with a scale per tensor are multiplied as they are."""
    cfg = _cfg(weights_int8=True)
    sd = _state(cfg, True)
    name = "model.layers.0.self_attn.o_proj.weight"
    sd[name + "_scale"] = torch.tensor(0.01)
    at = _load(cfg, sd).layers[0].attn
    assert torch.equal(at.o_w, sd[name]) and (at.o_ws == 0.01).all()


def test_fp8_codes_with_a_scale_per_channel():
    sd = _state(_cfg(), False)
    name = "model.layers.0.mlp.down_proj.weight"
    w = sd[name]
    s = w.abs().amax(1, keepdim=True) / 448
    sd[name], sd[name + "_scale"] = (w / s).to(torch.float8_e4m3fn), s
    model = _load(_cfg(), sd)
    assert torch.equal(model.layers[0].mlp.down_w, sd[name].float() * s)


@pytest.mark.parametrize("held", [True, False])
@pytest.mark.parametrize("change", [
    lambda sd, n: sd.pop(n + "_scale"),                                                                    # codes alone
    lambda sd, n: sd.update({n + "_scale": torch.ones(sd[n].shape[0], 4)}),                                # groups of columns
    lambda sd, n: sd.update({n + "_scale": torch.ones(3)}),
    lambda sd, n: sd.update({n + "_zero_point": torch.full((sd[n].shape[0], 1), 3, dtype=torch.int8)}),    # not symmetric
])
def test_codes_that_are_not_understood_are_refused(change, held):
    cfg = _cfg(quantization_config=W8A8 if held else _scheme("input_activations", dynamic=False))
    sd = _state(cfg, True)
    change(sd, "model.layers.1.mlp.down_proj.weight")
    with pytest.raises(ValueError):
        _load(cfg, sd)


def test_zero_points_of_zero_are_none():
    cfg = _cfg(quantization_config=W8A8)
    sd = _state(cfg, True)
    name = "model.layers.1.mlp.down_proj.weight"
    sd[name + "_zero_point"] = torch.zeros(sd[name].shape[0], 1, dtype=torch.int8)
    assert torch.equal(_load(cfg, sd).layers[1].mlp.down_w, sd[name])


@pytest.mark.parametrize("name", ["self_attn.o_proj", "mlp.down_proj"])
def test_linears_left_out_of_the_quantisation(name):
    """A checkpoint in 8 bits that keeps some linears in floating point is not quantised behind its back; who asks for it has them quantised."""
    left_out = f"model.layers.0.{name}.weight"
    sd = _state(_cfg(), True)
    sd[left_out] = torch.randn(sd[left_out].shape, generator=torch.Generator().manual_seed(1)) * 0.1
    del sd[left_out + "_scale"]
    config = {**W8A8, "ignore": ["lm_head", left_out.removesuffix(".weight")]}
    with pytest.raises(ValueError, match=name):
        _load(_cfg(quantization_config=config), sd)
    model = _load(_cfg(quantization_config=config, weights_int8=True), sd)
    w, s = {"self_attn.o_proj": (model.layers[0].attn.o_w, model.layers[0].attn.o_ws),
            "mlp.down_proj": (model.layers[0].mlp.down_w, model.layers[0].mlp.down_ws)}[name]
    assert float((w.float() * s[:, None] - sd[left_out]).abs().max()) <= 0.51 * float(s.max())
    assert torch.equal(model.layers[1].mlp.down_w, sd["model.layers.1.mlp.down_proj.weight"])


def test_a_fused_projection_left_out():
    """Models with one tensor for queries, keys and values, or for gate and up."""
    cfg = _cfg("ChatGLMModel", kv_channels=64, multi_query_group_num=2, ffn_hidden_size=192, num_layers=2, add_qkv_bias=False,
               layernorm_epsilon=1e-5, padded_vocab_size=256, quantization_config=W8A8)
    model = registry.build_model(cfg, "cpu")
    sd, pre = {}, "transformer.encoder.layers.{}."
    h = cfg["hidden_size"]
    sd["transformer.embedding.word_embeddings.weight"] = torch.randn(256, h)
    sd["transformer.encoder.final_layernorm.weight"] = torch.ones(h)
    sd["transformer.output_layer.weight"] = torch.randn(256, h)
    for i, layer in enumerate(model.layers):
        p = pre.format(i)
        sd[p + "input_layernorm.weight"] = sd[p + "post_attention_layernorm.weight"] = torch.ones(h)
        for name, w in (("self_attention.query_key_value", layer.attn.qkv_w), ("self_attention.dense", layer.attn.o_w),
                        ("mlp.dense_h_to_4h", layer.mlp.gate_up_w), ("mlp.dense_4h_to_h", layer.mlp.down_w)):
            sd[p + name + ".weight"] = torch.randint(-127, 128, w.shape, dtype=torch.int8)
            sd[p + name + ".weight_scale"] = torch.rand(w.shape[0], 1) * 0.01
    model.load_weights(CheckpointReader.from_state_dict(sd))
    name = pre.format(1) + "mlp.dense_h_to_4h.weight"
    assert torch.equal(model.layers[1].mlp.gate_up_w, sd[name]) and torch.equal(model.layers[1].mlp.gate_up_ws, sd[name + "_scale"][:, 0])
    sd[name] = sd[name].float()
    del sd[name + "_scale"]
    with pytest.raises(ValueError, match="dense_h_to_4h"):
        registry.build_model(cfg, "cpu").load_weights(CheckpointReader.from_state_dict(sd))
