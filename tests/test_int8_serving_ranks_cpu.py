"""int8 projections and cache over two tensor-parallel ranks (gloo): every rank's operator calls against 64 bits."""
import pytest
import torch

import _int8 as R
from tests._mp import run_ranks


class _Calls(R.Recorder):
    """Keeps copies of results: a partial product is summed over the ranks in place afterwards."""

    def _wrap(self, name, fn):
        def call(*args, **kw):
            before = [a.clone() if torch.is_tensor(a) else a for a in args]
            got = fn(*args, **kw)
            if name == "kv_write_int8":
                after = [a.clone() for a in args[2:6]]
            else:
                after = got.clone() if torch.is_tensor(got) else tuple(x.clone() for x in got)
            self.calls.append((name, before, dict(kw), after))
            return got
        return call


def _serve(rank, world, be, path):
    from axonml_b200.parallel import ProcessGroup
    from axonml_b200.server import LLMEngine, QuantizedLlama
    model = QuantizedLlama.from_gguf(path, ProcessGroup(be), device="cpu").to_int8()
    with pytest.MonkeyPatch.context() as mp:
        rec = _Calls(mp)
        tokens = LLMEngine(model, max_batch=4, max_context=48, kv_dtype=torch.int8).generate([[1, 2, 3, 4, 5], [9, 8, 7, 6, 5], [4, 4, 4, 4, 4]], 6)
    rec.check()
    return tokens, sorted(set(rec.names())), len(rec.calls)


def test_two_ranks_serve_in_eight_bits(tmp_path):
    from axonml_b200.llm import LLaMAConfig
    from axonml_b200.quant import QuantType
    from axonml_b200.server import QuantizedLlama
    cfg = LLaMAConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, max_position_embeddings=128)
    path = str(tmp_path / "m.gguf")
    QuantizedLlama.from_random(cfg, None, device="cpu", std=0.2, proj_type=QuantType.Q8_0).to_gguf(path)
    res = run_ranks(_serve, 2, args=(path,))
    (a, names, calls), (b, _, calls1) = res[0][1], res[1][1]
    assert a == b and all(len(x) == 6 for x in a)        # the ranks agree on every token
    assert names == ["decode_attention_int8", "int8_linear", "kv_write_int8", "quantize_int8", "rms_norm_int8", "swiglu_int8"]
    # a layer: two norms, four products, a write, the attention's rows, SwiGLU; five decode steps have the attention too
    assert calls == calls1 == 2 * (9 + 5 * 10)
