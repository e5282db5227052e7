"""The kernels' status word is seen by host threads only once it is ready."""
import threading

import torch

from axonml_b200 import _native as N


def test_threads_see_one_word_and_only_when_it_is_ready(monkeypatch):
    monkeypatch.setattr(N, "_STATUS", {})
    made, begun, go, ready = [], threading.Event(), threading.Event(), threading.Event()

    def slow(dev):                                        # the fill of the word, and the wait for it
        t = torch.zeros(4, dtype=torch.int32)
        made.append(t)
        begun.set()
        assert go.wait(60)
        ready.set()
        return t
    monkeypatch.setattr(N, "_new_status_word", slow)
    got, early = [], []

    def use():
        w = N.status_word("cpu")
        early.append(not ready.is_set())
        got.append(w)
    threads = [threading.Thread(target=use) for _ in range(8)]
    for t in threads:
        t.start()
    assert begun.wait(60)
    published = dict(N._STATUS)
    go.set()
    for t in threads:
        t.join()
    assert not published                                  # nothing is seen before it is ready
    assert len(got) == 8 and len(made) == 1 and all(w is made[0] for w in got) and not any(early)
    assert N.status_word("cpu") is made[0]


def test_a_word_for_each_device(monkeypatch):
    monkeypatch.setattr(N, "_STATUS", {})
    w = N.status_word("cpu")
    assert w.tolist() == [0, 0, 0, 0] and N.status_word(torch.device("cpu")) is w and set(N._STATUS) == {("cpu", None)}
