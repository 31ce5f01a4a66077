"""The error word of the ragged path's operators, without a device: first calls of several threads share one, which no
call sees before it is zeroed."""

import threading
import time
import types

import pytest
import torch


@pytest.fixture()
def ops(monkeypatch):
    from okc_b200 import ops
    monkeypatch.setattr(ops, "_WS", {})
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    return ops


def test_first_calls_of_threads_share_a_word(ops, monkeypatch):
    zeroed, made = set(), []
    real = torch.zeros

    def zeros(*a, **k):
        time.sleep(0.02)
        made.append(real(4096, dtype=torch.uint8))
        return made[-1]

    def synchronize():
        time.sleep(0.02)
        zeroed.update(t.data_ptr() for t in made)

    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: types.SimpleNamespace(synchronize=synchronize))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    start, got = threading.Barrier(8), []

    def call(delay):
        start.wait()
        time.sleep(delay)
        word = ops._error_word(0, "linear")
        got.append((word, word in zeroed))

    threads = [threading.Thread(target=call, args=(0.01 * (i % 4),)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and len(got) == 8
    assert all(word == made[0].data_ptr() and ready for word, ready in got)


def test_a_capture_is_refused_and_leaves_nothing(ops, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ops._lib.OkcError, match="capture"):
        ops._error_word(0, "linear")
    assert not ops._WS and not ops._FIRST.locked()
