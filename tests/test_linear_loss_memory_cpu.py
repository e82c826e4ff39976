"""What the output projection with its loss may hold next to its inputs and outputs: the limit's arithmetic, its refusals and its arguments."""
import random

import pytest
import torch

from mindspeed_b200.ops import linear_cross_entropy as M


def _held(T, H, V, K, limit):
    """Bytes that a training call holds at once: what it keeps for the backward and the scratch of a piece, as the calls allocate them."""
    piece, slab, keep = M._budget(T, H, V, K, limit)
    cols, splits, ldt, words = M._plan(T, H, V, piece, slab, True, keep)
    kept = 4 * (T * H // 2 + words * ldt + 2 * T * K + 3 * T + 2)
    ldz = 0 if words == V else min(cols, (V + 7) // 8 * 8)
    return kept + 2 * max(min(cols, words) * ldt, T * ldz) + 4 * splits * ((T + 31) // 32 * 32) * H + 8, words


def _least(T, H, K):
    """The copy of the hidden states, one part of their gradient, a piece of 256 words."""
    return 2 * T * H + 8 * T * K + 12 * T + 16 + 4 * ((T + 31) // 32 * 32) * H + 512 * ((T + 7) // 8 * 8)


def test_a_call_holds_at_most_its_limit():
    rng = random.Random(0)
    tight = 0
    for _ in range(4000):
        T, H, V, K = int(2 ** rng.uniform(6.1, 17)), 8 * int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(8, 18)), rng.choice([1, 1, 8, 64])
        if 16 * T <= H:
            continue
        limit = int(rng.choice([2 * T * V, 2 * T * V, 2 ** rng.uniform(20, 34)]))
        held, words = _held(T, H, V, K, limit)
        assert held <= max(limit, _least(T, H, K)), (T, H, V, K, limit, held)
        tight += held > 0.5 * limit and words > 0
    assert tight > 100


def test_sizes_of_a_training_step():
    assert M._budget(4096, 4096, 129280, 1, None) == (M.PIECE_BYTES, M.SLAB_BYTES, M.KEEP_BYTES)
    for T, V, some in ((8192, 128256, True), (4096, 129280, True), (4096, 32000, False)):
        held, words = _held(T, 4096, V, 1, 2 * T * V)
        assert held <= 2 * T * V and (8192 <= words < V if some else words == 0)
    T, H = 32768, 4096                                                                    # the module's own bounds hold as well (one part: 4 T H)
    assert _held(T, H, 128256, 1, 2 * T * 128256)[0] <= M.KEEP_BYTES + M.PIECE_BYTES + 4 * T * H + 2 * T * H + 20 * T + 16 < 2 * T * 128256
    piece, slab, keep = M._budget(4096, 4096, 32000, 1, 0)                                # the least
    assert keep == 0 and M._plan(4096, 4096, 32000, piece, slab, True, keep) == (256, 1, 0, 0)
    for T in (1, 64, 100, 256):                                                           # few tokens are not limited
        assert M._budget(T, 4096, 32000, 1, 0) == (M.PIECE_BYTES, M.SLAB_BYTES, M.KEEP_BYTES)


def test_refusals_and_arguments(monkeypatch):
    h, w, lab = torch.randn(5, 8), torch.randn(9, 8), torch.arange(5)
    for bad in (-1, float("nan")):
        with pytest.raises(ValueError, match="memory_limit"):
            M.linear_cross_entropy(h, w, lab, memory_limit=bad)
        with pytest.raises(ValueError, match="memory_limit"):
            M.linear_topk_distillation(h, w, torch.zeros(5, 2), torch.zeros(5, 2, dtype=torch.long), memory_limit=bad)
    assert torch.equal(M.linear_cross_entropy(h, w, lab, memory_limit=0), M.linear_cross_entropy(h, w, lab))


@pytest.mark.parametrize("mb,want", [(0, 2 * 16 * 40 * 4), (3, 3 << 20)])
def test_model_hands_the_limit_on(monkeypatch, mb, want):
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    cfg = TransformerConfig(num_layers=1, hidden_size=32, num_attention_heads=2, use_cpu_initialization=True, linear_cross_entropy_fusion=True,
                            linear_cross_entropy_memory_mb=mb, hidden_dropout=0.0, attention_dropout=0.0)
    seen = []
    for name in ("linear_cross_entropy", "linear_topk_distillation"):
        monkeypatch.setattr(M, name, lambda *a, _own=getattr(M, name), **k: (seen.append(k.get("memory_limit")), _own(*a, **k))[1])
    m = GPTModel(cfg, vocab_size=40, max_sequence_length=16)
    ids = torch.randint(0, 40, (2, 16))
    pos = torch.arange(16).expand(2, -1)
    m(ids, pos, None, labels=ids)
    m(ids, pos, None, labels=ids, distill_targets=(torch.zeros(2, 16, 3), torch.zeros(2, 16, 3, dtype=torch.long)))
    assert seen[0] == want == seen[1]          # fp32 logits of 2 x 16 tokens and 40 words, or what the argument says


def test_argument():
    from mindspeed_b200.training.arguments import parse_args, validate_args
    from test_checkpoint_cpu import ARGS
    assert parse_args(args_list=ARGS + ["--linear-cross-entropy-memory-mb", "700"]).linear_cross_entropy_memory_mb == 700
    with pytest.raises(AssertionError, match="negative"):
        validate_args(parse_args(args_list=ARGS + ["--linear-cross-entropy-memory-mb", "-1"]))
