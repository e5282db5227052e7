"""Serving in eight bits on the CPU path: the engine with an int8 cache and with int8 projections."""
import pytest
import torch

import _int8 as R
from axonml_b200 import llm, server
from axonml_b200.quant import QuantType


def _model(seed=0, **kw):
    torch.manual_seed(seed)
    cfg = llm.LLaMAConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                          num_key_value_heads=2, max_position_embeddings=128)
    return server.QuantizedLlama.from_random(cfg, None, device="cpu", std=0.2, proj_type=QuantType.Q8_0, **kw)


PROMPTS = [[1, 2, 3, 4], [9, 8, 7, 6], [5, 5, 5, 5]]


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.int8])
def test_continuous_batching_matches_sequential_decoding(weights, kv):
    model = _model()
    if weights:
        model.to_int8()
        assert model.int8_weights() and model.weight_bytes() > 0
    together = server.LLMEngine(model, max_batch=4, max_context=48, page_size=16, kv_dtype=kv).generate(PROMPTS, 20)
    alone = [server.LLMEngine(model, max_batch=4, max_context=48, page_size=16, kv_dtype=kv).generate([p], 20)[0] for p in PROMPTS]
    assert together == alone and all(len(x) == 20 for x in together)


def test_every_operator_of_a_run_keeps_its_definition(monkeypatch):
    """A prefill and two decode steps with int8 projections and cache: each call against 64 bits, and their order."""
    m = _model().to_int8()
    rec = R.Recorder(monkeypatch)
    with torch.no_grad():
        cache = server.PagedKVCache(2, 8, 16, m.hkv, m.hd, 2, 4, "cpu", dtype=torch.int8)
        slots = [cache.allocate_seq(), cache.allocate_seq()]
        ids = torch.randint(0, 512, (2, 15), generator=torch.Generator().manual_seed(3))
        for s in slots:
            cache.reserve(s, 17)
        m.prefill(ids, cache, slots)
        for n in (15, 16):
            m.decode(torch.tensor([7, n]), cache, torch.tensor(slots, dtype=torch.int32), torch.tensor([n, n], dtype=torch.int32))
    layer = ["rms_norm_int8", "int8_linear", "kv_write_int8", "quantize_int8", "int8_linear", "rms_norm_int8", "int8_linear", "swiglu_int8",
             "int8_linear"]
    assert rec.names() == layer * 2 + (layer[:3] + ["decode_attention_int8"] + layer[3:]) * 4
    rec.check()


def test_to_int8_leaves_other_parts_and_refuses_gguf(tmp_path):
    m = _model()
    embed = m.embed
    m.to_int8().to_int8()                                # a second call changes nothing
    assert m.embed is embed and m.optimize_layout() is m
    with pytest.raises(ValueError):
        m.to_gguf(tmp_path / "x.gguf")


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(head_dim=40)])
def test_int8_cache_refuses_other_shapes(kw):
    a = dict(num_layers=1, num_pages=2, page_size=16, num_kv_heads=1, head_dim=32, max_seqs=1, max_pages_per_seq=2, device="cpu", dtype=torch.int8)
    server.PagedKVCache(**a)
    with pytest.raises(ValueError):
        server.PagedKVCache(**{**a, **kw})


def test_engine_refuses_other_cache_types():
    with pytest.raises(ValueError):
        server.LLMEngine(_model(), max_batch=1, max_context=16, kv_dtype=torch.float16)
