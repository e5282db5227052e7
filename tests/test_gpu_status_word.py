"""First calls of an operator from several host threads, each on its own stream."""
import threading

import pytest
import torch

from axonml_b200 import _native as N
from axonml_b200.ops import int8 as I

pytestmark = pytest.mark.gpu


def test_first_calls_from_several_threads(kernel_status):
    W = I.Int8Weight.from_dense(torch.randn(256, 128, device="cuda"))
    q, s = I.quantize_int8(torch.randn(8, 128, device="cuda"))
    want = I.int8_linear(q, s, W.q, W.scale)
    torch.cuda.synchronize()
    saved, words = dict(N._STATUS_PTR), dict(N._STATUS)
    seen, got, errors = [], [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                seen.append(N.status_ptr(torch.cuda.current_device()))
                y = I.int8_linear(q, s, W.q, W.scale)
                torch.cuda.current_stream().synchronize()
                got.append(y)
        except Exception as e:
            errors.append(e)
    try:
        N._STATUS_PTR.clear()
        N._STATUS.clear()
        torch.full((1 << 20,), 1, dtype=torch.int32, device="cuda")       # memory that a new word may come from
        threads = [threading.Thread(target=work) for _ in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not errors and len(set(seen)) == 1 and all(torch.equal(y, want) for y in got)
        N.check_status()
    finally:
        N._STATUS_PTR.clear()
        N._STATUS.clear()
        N._STATUS_PTR.update(saved)
        N._STATUS.update(words)
    torch.cuda.synchronize()
