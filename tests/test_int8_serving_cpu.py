"""The serving engine and model around int8 weights and caches, on the CPU path."""
import types

import pytest
import torch

from axonml_b200 import llm, server
from axonml_b200.quant import QuantType


def _model(**kw):
    cfg = llm.LLaMAConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                          num_key_value_heads=2, max_position_embeddings=128)
    return server.QuantizedLlama.from_random(cfg, None, device="cpu", std=0.2, proj_type=QuantType.Q8_0, **kw)


def test_graphs_of_replaced_weights_are_dropped():
    """An engine keeps its decode graphs only as long as the model has the weights that they were captured with."""
    m = _model()
    eng = server.LLMEngine(m, max_batch=2, max_context=16)
    eng._graphs[2] = "captured"
    assert eng._live_graphs() == {2: "captured"}
    m.to_int8()
    assert eng._live_graphs() == {}
    eng._graphs[2] = "captured again"
    m.to_int8()                                          # nothing is replaced
    assert eng._live_graphs() == {2: "captured again"}


def test_a_plain_holder_of_pages_serves_as_a_cache():
    """prefill and decode take any object with bf16 pages and a block table, as before there were int8 caches."""
    m = _model()
    ids = torch.randint(0, 512, (2, 9), generator=torch.Generator().manual_seed(1))
    slots = torch.tensor([0, 1], dtype=torch.int32)
    got = []
    with torch.no_grad():
        for plain in (False, True):
            c = server.PagedKVCache(2, 8, 4, m.hkv, m.hd, 2, 4, "cpu")
            for s in (c.allocate_seq(), c.allocate_seq()):
                c.reserve(s, 10)
            if plain:
                c = types.SimpleNamespace(k=c.k, v=c.v, block_table=c.block_table, page_size=c.page_size)
            h = m.prefill(ids, c, [0, 1])
            got.append((h, m.decode(torch.tensor([5, 6]), c, slots, torch.tensor([9, 9], dtype=torch.int32))))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("flags", [["--kv-cache", "int8"], ["--weights", "int8"]])
def test_int8_flags_without_a_language_model_are_refused(flags, monkeypatch):
    from axonml_b200.cli.main import main
    from axonml_b200.server import http
    monkeypatch.setattr(http.AxonmlHTTPServer, "serve_forever", lambda self: None)
    with pytest.raises(SystemExit, match="gguf"):
        main(["serve", "--port", "0", *flags])
