"""Run under torchrun (gloo, 2 ranks): a checkpoint in 8 bits sharded over tensor-parallel ranks, a feed-forward block of it, and the engine on a
4-bit cache. argv: <out file>; one rank alone writes the engine's tokens only."""
import json
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

PROMPTS = [[5, 17, 99, 200, 3, 45, 7], [9] * 40, list(range(20, 120)), [300, 301]]


def _tokens(cfg, tp, port, **kw):
    from gllm_b200 import LLM
    from shard_util import load_global_weights
    llm = LLM(cfg, load_format="dummy", tp_size=tp, maxp=48, maxd=16, num_cpu_pages=128, model_max_length=256, log_stats=False, device="cpu",
              launch_mode="inproc", seed=0, master_port=port, **kw)
    load_global_weights(llm.worker.runner.model, cfg, seed=123)
    runner = llm.worker.runner
    assert runner.kv_cache.k_cache[0].dtype == torch.uint8
    assert (runner.model.layers[0].attn.qkv_w.dtype == torch.int8) == ("quantization" in kw)
    outs = llm.generate(tokens=[list(p) for p in PROMPTS], output_lens=[8] * 4, ignore_eos=True, temperature=0.0, top_k=1)
    return llm, [s.token_ids[len(p):] for s, p in zip(outs, PROMPTS)]


def _shards(world, kv_heads):
    """Each rank's codes and scales are its rows or columns of the checkpoint's; a block of both linears gives the definition's value."""
    from gllm_b200.models import registry, weight_utils as wu
    from gllm_b200.models.presets import tiny
    from gllm_b200.models.weight_utils import CheckpointReader
    from gllm_b200.ops import ref
    from gllm_b200.parallel import state as ps
    from gllm_b200.parallel.tp import make_tp_comm
    from tests.test_quantised_serving_cpu import W8A8
    st = ps.get_state()
    h, d, hq, inter = 128, 64, 4, 192
    cfg = registry.HFConfig(tiny("Qwen3ForCausalLM", hidden_size=h, num_attention_heads=hq, num_key_value_heads=kv_heads, head_dim=d,
                                 intermediate_size=inter, quantization_config=W8A8))
    g = torch.Generator().manual_seed(11)
    sd = {"model.embed_tokens.weight": torch.randn(cfg["vocab_size"], h, generator=g), "model.norm.weight": torch.ones(h),
          "lm_head.weight": torch.randn(cfg["vocab_size"], h, generator=g)}
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        sd[p + "input_layernorm.weight"] = sd[p + "post_attention_layernorm.weight"] = torch.ones(h)
        sd[p + "self_attn.q_norm.weight"] = sd[p + "self_attn.k_norm.weight"] = torch.ones(d)
        for name, n, k in (("self_attn.q_proj", hq * d, h), ("self_attn.k_proj", kv_heads * d, h), ("self_attn.v_proj", kv_heads * d, h),
                           ("self_attn.o_proj", h, hq * d), ("mlp.gate_proj", inter, h), ("mlp.up_proj", inter, h), ("mlp.down_proj", h, inter)):
            sd[p + name + ".weight"] = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
            sd[p + name + ".weight_scale"] = (0.5 + torch.rand(n, 1, generator=g)) * 0.01
    model = registry.build_model(cfg, "cpu")
    model.load_weights(CheckpointReader.from_state_dict(sd))
    r, p = st.tp_rank, "model.layers.1."
    at, mlp = model.layers[1].attn, model.layers[1].mlp
    of = lambda name: (sd[p + name + ".weight"], sd[p + name + ".weight_scale"])  # noqa: E731
    kv0, nkv = wu.kv_head_range(kv_heads, r, world)
    for got, part in ((at.qkv_w, 0), (at.qkv_ws, 1)):
        q, k, v = (of(f"self_attn.{x}_proj")[part] for x in "qkv")
        a, b = r * hq * d // world, (r + 1) * hq * d // world
        assert torch.equal(got, torch.cat([q[a:b], k[kv0 * d:(kv0 + nkv) * d], v[kv0 * d:(kv0 + nkv) * d]]).reshape(got.shape))
    w, s = of("self_attn.o_proj")
    n = hq * d // world
    assert torch.equal(at.o_w, w[:, r * n:(r + 1) * n]) and torch.equal(at.o_ws, s[:, 0])
    w, s = of("mlp.down_proj")
    n = inter // world
    assert torch.equal(mlp.down_w, w[:, r * n:(r + 1) * n]) and torch.equal(mlp.down_ws, s[:, 0])
    # every rank quantises the rows of its own columns; partial sums are added in fp32
    tpc = make_tp_comm(False)
    x = torch.randn(5, h, generator=g)
    got = tpc.row_linear(mlp.act(x, tpc), mlp.down_weight())
    (gw, gs), (uw, us) = of("mlp.gate_proj"), of("mlp.up_proj")
    want = torch.zeros(5, h, dtype=torch.float64)
    for i in range(world):
        rows = slice(i * n, (i + 1) * n)
        act = ref.linear_int8(x, torch.cat([gw[rows], uw[rows]]), torch.cat([gs[rows], us[rows]])[:, 0], silu=True)
        q, step = ref.int8_quant_rows(act)
        want += (q.double() @ w[:, rows].double().t()) * step.double()[:, None] * s.double()[:, 0]
    # three roundings of each part and of their sum: 2^-24 each of magnitudes below `most`
    most = want.abs().max() * 4
    assert float((got.double() - want).abs().max()) <= 8 * 2 ** -24 * float(most), float((got.double() - want).abs().max() / most)


def main():
    out, rank, world = sys.argv[1], int(os.environ.get("RANK", "0")), int(os.environ.get("WORLD_SIZE", "1"))
    port = int(os.environ.get("MASTER_PORT", "29500")) + 1
    from gllm_b200.models.presets import tiny
    cfg = tiny("Qwen3ForCausalLM", num_hidden_layers=3, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
               intermediate_size=192)
    llm, tokens = _tokens(cfg, world, port, kv_cache_dtype="int4")
    if world > 1:
        for kv_heads in (2, 1):                            # one is held by both ranks
            _shards(world, kv_heads)
    llm.shutdown() if world == 1 else llm.close()
    llm, both = _tokens(cfg, world, port + 10, kv_cache_dtype="int4", quantization="int8")
    if rank == 0:
        assert all(len(t) == 8 for t in both)
        with open(out, "w") as f:
            json.dump(tokens, f)
    llm.shutdown()
    if torch.distributed.is_initialized():
        torch.distributed.barrier()
        torch.distributed.destroy_process_group()


if __name__ == "__main__":
    main()
