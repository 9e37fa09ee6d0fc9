"""8-bit linears and a 4-bit cache in the engine: loading, page accounting, refusals, whole runs (CPU)."""
import pytest
import torch

from gllm_b200.memory_manager import KVCache
from gllm_b200.model_loader import ModelLoader
from gllm_b200.models import registry
from gllm_b200.models.presets import tiny
from gllm_b200.models.weight_utils import CheckpointReader
from gllm_b200.ops import kv4

W8A8 = {"quant_method": "compressed-tensors", "format": "int-quantized", "ignore": ["lm_head"], "config_groups": {"group_0": {
    "targets": ["Linear"], "weights": {"num_bits": 8, "type": "int", "symmetric": True, "strategy": "channel"},
    "input_activations": {"num_bits": 8, "type": "int", "symmetric": True, "strategy": "token", "dynamic": True}}}}


def _cfg(arch="Qwen3ForCausalLM", **over):
    return registry.HFConfig(tiny(arch, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=192,
                                  **over))


def _state(cfg, held_in_8_bits):
    g = torch.Generator().manual_seed(3)
    h, d, i = cfg["hidden_size"], cfg["head_dim"], cfg["intermediate_size"]
    sd = {"model.embed_tokens.weight": torch.randn(cfg["vocab_size"], h, generator=g), "model.norm.weight": torch.ones(h),
          "lm_head.weight": torch.randn(cfg["vocab_size"], h, generator=g) * 0.1}
    for n in range(cfg["num_hidden_layers"]):
        pre = f"model.layers.{n}."
        sd[pre + "input_layernorm.weight"] = sd[pre + "post_attention_layernorm.weight"] = torch.ones(h)
        sd[pre + "self_attn.q_norm.weight"] = sd[pre + "self_attn.k_norm.weight"] = torch.ones(d)
        for name, rows, cols in (("self_attn.q_proj", 4 * d, h), ("self_attn.k_proj", 2 * d, h), ("self_attn.v_proj", 2 * d, h),
                                 ("self_attn.o_proj", h, 4 * d), ("mlp.gate_proj", i, h), ("mlp.up_proj", i, h), ("mlp.down_proj", h, i)):
            w = torch.randn(rows, cols, generator=g) * 0.1
            if held_in_8_bits:
                s = w.abs().amax(1, keepdim=True) / 100            # not the scale that quantising anew would give
                sd[pre + name + ".weight"] = torch.round(w / s).to(torch.int8)
                sd[pre + name + ".weight_scale"] = s.to(torch.bfloat16)
            else:
                sd[pre + name + ".weight"] = w
    return sd


def test_checkpoint_in_8_bits_is_taken_as_it_is():
    cfg = _cfg(quantization_config=W8A8)
    model = registry.build_model(cfg, "cpu")
    sd = _state(cfg, True)
    model.load_weights(CheckpointReader.from_state_dict(sd))
    pre = "model.layers.1."
    at, mlp = model.layers[1].attn, model.layers[1].mlp
    want = torch.cat([sd[pre + f"self_attn.{x}_proj.weight"] for x in "qkv"])
    scale = torch.cat([sd[pre + f"self_attn.{x}_proj.weight_scale"] for x in "qkv"]).float()[:, 0]
    assert at.qkv_w.dtype == torch.int8 and torch.equal(at.qkv_w, want) and torch.equal(at.qkv_ws, scale)
    assert torch.equal(at.o_w, sd[pre + "self_attn.o_proj.weight"])
    assert torch.equal(mlp.gate_up_w, torch.cat([sd[pre + f"mlp.{x}_proj.weight"] for x in ("gate", "up")])) and not mlp.fused_act
    assert torch.equal(mlp.down_ws, sd[pre + "mlp.down_proj.weight_scale"].float()[:, 0])
    assert model.lm_head_w.dtype == torch.float32


def test_weights_quantised_while_loading():
    cfg = _cfg(weights_int8=True)
    model = registry.build_model(cfg, "cpu")
    sd = _state(cfg, False)
    model.load_weights(CheckpointReader.from_state_dict(sd))
    w = sd["model.layers.0.mlp.down_proj.weight"]
    mlp = model.layers[0].mlp
    back = mlp.down_w.float() * mlp.down_ws[:, None]
    assert ((back - w).abs() <= w.abs().amax(1, keepdim=True) / 127 * 0.501).all() and int(mlp.down_w.abs().max()) == 127


@pytest.mark.parametrize("part", ["weights", "input_activations"])
@pytest.mark.parametrize("over", [{"num_bits": 4}, {"type": "float"}, {"symmetric": False}, {"strategy": "tensor"}, {"dynamic": False}])
def test_other_schemes_are_not_taken_for_it(part, over):
    if part == "weights" and "dynamic" in over:
        pytest.skip("weights have no such entry")
    group = {k: dict(v) if isinstance(v, dict) else v for k, v in W8A8["config_groups"]["group_0"].items()}
    group[part].update(over)
    assert registry._quant(_cfg(quantization_config={**W8A8, "config_groups": {"group_0": group}})) is None


def test_checkpoints_half_in_8_bits_are_refused():
    cfg = _cfg(quantization_config=W8A8)
    sd = _state(cfg, True)
    del sd["model.layers.0.self_attn.k_proj.weight_scale"]
    sd["model.layers.0.self_attn.k_proj.weight"] = sd["model.layers.0.self_attn.k_proj.weight"].float()
    with pytest.raises(ValueError):
        registry.build_model(cfg, "cpu").load_weights(CheckpointReader.from_state_dict(sd))


def test_pages_of_a_4_bit_cache():
    four = KVCache.bytes_per_page(3, 16, 8, 128, 2, four_bit=True)
    assert four == 3 * 2 * 16 * 8 * 72 and KVCache.bytes_per_page(3, 16, 8, 128, 2) == four * 256 // 72
    c = KVCache(2, 5, 32, 8, 64, torch.bfloat16, "cpu", four_bit=True)
    assert c.k_cache[1].dtype == torch.uint8 and kv4.geometry(c.v_cache[0]) == (5, 8, 32, 64)


def _vl_moe():
    text = tiny("Qwen3MoeForCausalLM", hidden_size=128, head_dim=64, num_experts=4, num_experts_per_tok=2, moe_intermediate_size=64)
    text["rope_scaling"] = {"mrope_section": [12, 10, 10], "mrope_interleaved": True}
    vision = dict(depth=1, hidden_size=32, num_heads=2, intermediate_size=64, patch_size=16, spatial_merge_size=2, temporal_patch_size=2,
                  num_position_embeddings=16, deepstack_visual_indexes=[0], in_channels=3, out_hidden_size=128)
    return registry.HFConfig({"architectures": ["Qwen3VLMoeForConditionalGeneration"], "text_config": text, "vision_config": vision,
                              "torch_dtype": "float32", "image_token_id": 5, "video_token_id": 6, "vision_start_token_id": 7,
                              "weights_int8": True})


@pytest.mark.parametrize("make", [
    lambda: registry.build_model(_cfg("Qwen3MoeForCausalLM", num_experts=4, num_experts_per_tok=2, moe_intermediate_size=64, weights_int8=True), "cpu"),
    lambda: registry.build_model(_vl_moe(), "cpu"),
    lambda: registry.build_model(_cfg(weights_int8=True, quantization_config={"quant_method": "fp8", "weight_block_size": [128, 128]}), "cpu"),
    lambda: registry.build_model(registry.HFConfig(tiny("Qwen3ForCausalLM", hidden_size=120, head_dim=64, weights_int8=True)), "cpu"),
    lambda: ModelLoader(tiny(), quantization="int3"),
])
def test_models_without_8_bit_linears_are_refused(make):
    with pytest.raises(ValueError):
        make()


def _llm(cfg, **kw):
    from gllm_b200 import LLM
    kw = {"num_cpu_pages": 64, "maxp": 64, "maxd": 16, "page_size": 16, **kw}
    return LLM(dict(cfg), load_format="dummy", device="cpu", model_max_length=256, log_stats=False, **kw)


@pytest.mark.parametrize("cfg,kw", [
    (tiny(), {"kv_cache_dtype": "int4"}), (_cfg(), {"kv_cache_dtype": "int4", "page_size": 8}), (_cfg(), {"kv_cache_dtype": "int2"}),
])
def test_caches_that_cannot_be_held_in_4_bits_are_refused(cfg, kw):
    with pytest.raises(ValueError):
        _llm(cfg, **kw)


PROMPTS = [[5, 9, 100, 7], list(range(20, 150)), [77] * 33, [3, 1, 4, 1, 5, 9, 2, 6]]


def _tokens(**kw):
    llm = _llm(_cfg(vocab_size=512), kv_cache_dtype="int4", quantization="int8", **kw)
    runner = llm.worker.runner
    assert runner.kv_cache.k_cache[0].dtype == torch.uint8 and runner.model.layers[0].attn.qkv_w.dtype == torch.int8
    outs = llm.generate(tokens=[list(p) for p in PROMPTS], output_lens=[7] * len(PROMPTS), ignore_eos=True, top_k=1, temperature=0.0)
    got = [s.token_ids[len(p):] for s, p in zip(outs, PROMPTS)]
    llm.shutdown()
    return got


def test_engine_with_both():
    """Rows attend to the cache whatever chunk they came in, so chunks, prefix pages and the schedule change nothing."""
    want = _tokens()
    assert all(len(t) == 7 for t in want)
    assert _tokens(maxp=24) == want and _tokens(enable_prefix_caching=False) == want and _tokens(schedule_method="split_pd") == want
