"""Several error words set in one step, or on several devices: all are named, none is lost."""
import pytest
import torch


def test_every_word_of_every_device_is_named(monkeypatch):
    from mindspeed_b200.ops import gemm as G
    words = {"first": torch.tensor([0x21, 0x703, 0, 0], dtype=torch.int32), "healthy": torch.zeros(4, dtype=torch.int32),
             "second": torch.tensor([0x702, 0, 0, 0], dtype=torch.int32)}
    monkeypatch.setattr(G, "_status", words)
    with pytest.raises(RuntimeError) as e:
        G.check_status()
    text = str(e.value)
    for part in ("time-out, code 0x21 on first", "outside the vocabulary, code 0x703 on first", "routing map", "0x702 on second"):
        assert part in text, text
    assert not any(t.any() for t in words.values())
    G.check_status()


def test_one_device_is_asked(monkeypatch):
    from mindspeed_b200.ops import gemm as G
    words = {d: torch.tensor([0, 0x703, 0, 0], dtype=torch.int32) for d in ("a", "b")}
    monkeypatch.setattr(G, "_status", words)
    with pytest.raises(RuntimeError, match="on a$"):
        G.check_status("a")
    assert not words["a"].any() and words["b"].any()
