"""The operators of quantised serving together, as a decoder layer and as the engine run them (GPU)."""
import types

import numpy as np
import pytest
import torch

from gllm_b200.layers import functional as Fn
from gllm_b200.ops import kv4, ref
from tests import kv4_util as U
from tests.test_int8_gpu import product

pytestmark = pytest.mark.gpu
BF16, F64, DEV = torch.bfloat16, torch.float64, "cuda"


@pytest.mark.parametrize("news,decodes", [([1, 1, 1], 3), ([1, 50, 130], 1), ([200], 0)])
def test_a_layer_step_by_step(news, decodes):
    """Projection, rotary write, attention, output projection, gated feed-forward and its second product in one run on one stream; each
    step's result is held to its definition in 64 bits of what the step before gave."""
    torch.manual_seed(sum(news))
    h, hq, hkv, d, inter, page = 512, 8, 2, 64, 640, 16
    t, prior = sum(news), 37
    lens = [n + prior for n in news]
    weight = lambda n, k: (torch.randint(-127, 128, (n, k), device=DEV, dtype=torch.int8), (0.5 + torch.rand(n, device=DEV)) * 0.02 / k ** 0.5)  # noqa: E731
    w_qkv, w_o, w_gu, w_down = weight((hq + 2 * hkv) * d, h), weight(h, hq * d), weight(2 * inter, h), weight(h, inter)
    x = torch.randn(t, h, device=DEV).to(BF16)
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks) + 2
    table = torch.zeros(len(news), max(blocks), dtype=torch.int32)
    order, at = torch.randperm(pages).to(torch.int32), 0
    for s, b in enumerate(blocks):
        table[s, :b] = order[at:at + b]
        at += b
    caches = [torch.zeros(kv4.cache_shape(pages, hkv, d, page), dtype=torch.uint8, device=DEV) for _ in range(2)]
    slot = lambda s, i: table[s].long()[i // page] * page + i % page  # noqa: E731
    rows = []
    for s in range(len(news)):
        i = torch.arange(prior)
        kv = [torch.randn(prior, hkv, d, device=DEV).to(BF16) for _ in range(2)]
        for c, y in zip(caches, kv):
            kv4.write_rows(c, slot(s, i).to(DEV), y)
        rows.append(kv)
    pos = torch.cat([torch.arange(prior, n) for n in lens]).to(torch.int32).to(DEV)
    slots = torch.cat([slot(s, torch.arange(prior, n)) for s, n in enumerate(lens)]).to(torch.int32).to(DEV)
    cs = ref.build_cos_sin_cache(d, 1024, 1e4).to(DEV)
    start = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    inp = types.SimpleNamespace(block_table=table.to(DEV), seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                query_start_loc=torch.from_numpy(start).to(DEV), num_decode_seqs=decodes, num_seqs=len(news), padded_tokens=0,
                                max_q_len=max(news), max_seq_len=max(lens), decode_splits=None,
                                batch=types.SimpleNamespace(seq_lens=np.array(lens, np.int32)))
    qkv = Fn.linear(x, w_qkv)
    before = qkv.clone()
    q, k, v = (y.unflatten(1, (-1, d)) for y in qkv.split([hq * d, hkv * d, hkv * d], 1))
    Fn.rope_kv_write(q, k, v, pos, cs, d, True, None, None, 1e-6, *caches, slots)
    a = Fn.paged_attention(qkv[:, : hq * d], *caches, inp, d ** -0.5, hq, d)
    o = Fn.linear(a, w_o)
    g = Fn.linear_silu_mul(o, w_gu)
    y = Fn.linear(g, w_down)
    want, tol = product(x, *w_qkv)
    assert ((before.to(F64) - want).abs() <= tol).all()
    q0, k0, v0 = (z.unflatten(1, (-1, d)) for z in before.split([hq * d, hkv * d, hkv * d], 1))
    kt, plain = torch.empty_like(k0), [torch.zeros_like(c) for c in caches]
    ref.rope_kv_write(q0, k0, v0, pos, cs, d, True, None, None, 1e-6, *plain, slots)
    assert torch.equal(q, q0)                              # every step of it is one rounded operation
    for got, p in zip(caches, plain):
        assert torch.equal(kv4.read_rows(got, slots), kv4.read_rows(p, slots))
    kt = ref._rope_one(k0.float(), *(c[pos.long()] for c in cs.chunk(2, 1)), d, True).to(BF16)
    for s in range(len(news)):
        mine = slice(start[s], start[s + 1])
        rows[s] = [torch.cat((p, z[mine])) for p, z in zip(rows[s], (kt, v0))]
    want, tol = U.attention(q, rows, lens, news, d ** -0.5, hkv, True)
    assert ((a.view_as(want).to(F64) - want).abs() <= tol).all()
    for got, args, silu in ((o, (a, *w_o), False), (g, (o, *w_gu), True), (y, (g, *w_down), False)):
        want, tol = product(*args, silu=silu)
        assert ((got.to(F64) - want).abs() <= tol).all()


def _gen(device, graphs, prompts, out_len, state=None, **kw):
    from gllm_b200 import LLM
    from gllm_b200.models.presets import tiny
    cfg = tiny("Qwen3ForCausalLM", hidden_size=256, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
               intermediate_size=512, vocab_size=1024, torch_dtype="bfloat16")
    llm = LLM(cfg, load_format="dummy", maxp=128, maxd=64, max_cuda_graph_bs=8, num_gpu_pages=256, num_cpu_pages=256, model_max_length=512,
              log_stats=False, device=device, disable_cuda_graph=not graphs, kv_cache_dtype="int4", quantization="int8", **kw)
    runner = llm.worker.runner
    assert runner.kv_cache.k_cache[0].dtype == torch.uint8 and runner.model.layers[0].attn.o_w.dtype == torch.int8
    if state is not None:
        for (n, p), (_, q) in zip(runner.model.named_parameters(), state):
            p.data.copy_(q.to(p.device))
    outs = llm.generate(tokens=prompts, output_lens=[out_len] * len(prompts), ignore_eos=True)
    toks = [s.token_ids[len(p):] for s, p in zip(outs, prompts)]
    params = [(n, p.detach().cpu().clone()) for n, p in runner.model.named_parameters()]
    graph_steps = runner.stats["graph_steps"]
    llm.shutdown()
    return toks, params, graph_steps


def test_engine_on_the_gpu_and_on_the_cpu():
    prompts = [[5, 9, 100, 7], list(range(20, 190)), [77] * 33, [3, 1, 4, 1, 5, 9, 2, 6]]
    cpu, params, _ = _gen("cpu", False, prompts, 6)
    gpu, _, steps = _gen("cuda", True, prompts, 6, state=params)
    assert steps > 0
    # other roundings on the two sides: the first tokens agree, later ones may part where two logits are next to one another
    assert [x[0] for x in cpu] == [y[0] for y in gpu], (cpu, gpu)
    assert sum(x == y for x, y in zip(cpu, gpu)) >= len(prompts) // 2, (cpu, gpu)


def test_engine_with_graphs_and_without():
    prompts = [[5, 9, 100, 7], list(range(20, 150)), [77] * 33]
    eager, params, _ = _gen("cuda", False, prompts, 8)
    graphs, _, steps = _gen("cuda", True, prompts, 8, state=params)
    assert steps > 0 and eager == graphs


def test_pages_from_the_memory_left():
    """Without a page count the engine takes what 4-bit pages and a step's scratch leave room for."""
    from gllm_b200 import LLM
    from gllm_b200.models.presets import tiny
    cfg = tiny("Qwen3ForCausalLM", hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64, torch_dtype="bfloat16")
    llm = LLM(cfg, load_format="dummy", model_max_length=256, max_cuda_graph_bs=2, log_stats=False, kv_cache_dtype="int4",
              gpu_memory_util=0.02)
    out = llm.generate(tokens=[[1, 2, 3]], output_lens=[4], ignore_eos=True)
    assert len(out[0].token_ids) == 7
    llm.shutdown()
