"""The serving engine around int8 weights and caches on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu

PROMPTS = [[(13 * i + j) % 19000 for j in range(18)] for i in range(6)]


def _model(proj=None):
    from axonml_b200.llm import LLaMAConfig
    from axonml_b200.quant import QuantType
    from axonml_b200.server import QuantizedLlama
    cfg = LLaMAConfig(vocab_size=20000, hidden_size=1024, intermediate_size=2048, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=4, max_position_embeddings=256)
    return QuantizedLlama.from_random(cfg, None, device="cuda", std=0.05, proj_type=proj or QuantType.Q4_K)


def test_weights_replaced_under_a_live_engine(kernel_status):
    """An engine that has captured its decode graphs answers as a new one does once its model's weights are int8."""
    from axonml_b200.server import LLMEngine
    model = _model()
    engine = LLMEngine(model, max_batch=6, max_context=64)
    engine.generate(PROMPTS, 8)
    assert engine._graphs or not engine.use_graphs
    model.to_int8()
    torch.full((64 << 20,), 7, dtype=torch.uint8, device="cuda")      # over what the old weights left
    got = engine.generate(PROMPTS, 24)
    assert got == LLMEngine(model, max_batch=6, max_context=64).generate(PROMPTS, 24)
