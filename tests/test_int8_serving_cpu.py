"""The serving engine and model around int8 weights and caches, on the CPU path."""
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
