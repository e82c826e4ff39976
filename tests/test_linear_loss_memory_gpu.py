"""Memory of the output projection with its loss on the GPU: within its limit, never above the path that the model's flag replaces, and the
same numbers whatever the limit."""
import gc
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_linear_cross_entropy_gpu import BF16, FP16, _ce, _ce_target, _compare, _inputs, _kd, _kd_target  # noqa: E402
from test_loss_operators_gpu import one_rank  # noqa: E402, F401

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def _peak(f):
    """(what f returns, bytes above those before it at its highest)."""
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,V,H", [(1003, 20011, 1024), (300, 3000, 136), (70, 9001, 640)])
def test_same_numbers_within_every_limit(T, V, H, dtype):
    h, w, fav, g, gen = _inputs(T, V, H, dtype)
    fav[::7] = -100
    idx = torch.randint(0, V, (T, 20), generator=gen, device="cuda")
    a = torch.randn(T, 20, generator=gen, device="cuda")
    first = None
    for limit in (None, 0, 2 * T * V, T * V, 3 * T * V):
        ce, kd = _ce(h, w, fav, g, memory_limit=limit), _kd(h, w, a, idx, 2.0, g, memory_limit=limit)
        _compare(ce, h, w, _ce_target(fav), 1.0, g)
        _compare(kd, h, w, _kd_target(idx, a, 2.0), 2.0, g)
        first = first or (ce, kd)
        for got, want in zip((ce, kd), first):           # the hidden gradient's sums may be cut elsewhere
            assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("T,V,H", [(2048, 32000, 1024), (1000, 50257, 768), (4096, 32000, 4096)])
def test_a_call_stays_within_its_limit(T, V, H):
    """Beside the loss and the gradients.  The allocator's blocks may be 2 MiB larger than asked for: six of them."""
    from mindspeed_b200.ops.linear_cross_entropy import linear_cross_entropy
    h, w, fav, g, _ = _inputs(T, V, H, BF16)
    h.requires_grad_(True), w.requires_grad_(True)
    call = lambda **k: torch.autograd.grad(linear_cross_entropy(h, w, fav, **k), (h, w), g)
    call()
    ours = 2 * (T * H + V * H) + 8 * T
    for limit in (2 * T * V, T * V):
        assert _peak(lambda: call(memory_limit=limit))[1] <= limit + ours + 12 * MIB
    plain = _peak(lambda: torch.autograd.grad(torch.nn.functional.cross_entropy(h @ w.t(), fav, reduction="none"), (h, w), g.to(BF16)))[1]
    assert _peak(lambda: call(memory_limit=2 * T * V))[1] <= plain


@pytest.mark.parametrize("heads", [0, 2])
@pytest.mark.parametrize("seq", [2048, 1500])
def test_the_flag_does_not_raise_the_peak(one_rank, seq, heads):  # noqa: F811
    """A training step of a model whose logits are most of its memory, with the flag and without, multi-token heads included."""
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    peaks, losses = [], []
    for fused in (False, True):
        cfg = TransformerConfig(num_layers=1, hidden_size=1024, num_attention_heads=8, ffn_hidden_size=1024, hidden_dropout=0.0,
                                attention_dropout=0.0, optimization_level=1, params_dtype=BF16, bf16=True, add_bias_linear=False,
                                normalization="RMSNorm", mtp_num_layers=heads or None, gradient_accumulation_fusion=True,
                                linear_cross_entropy_fusion=fused)
        torch.manual_seed(7)
        m = GPTModel(cfg, vocab_size=32000, max_sequence_length=seq, position_embedding_type="rope").cuda().train()
        for p in m.parameters():
            p.main_grad = torch.zeros_like(p, dtype=torch.float32)
        ids = torch.randint(0, 32000, (1, seq), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
        pos = torch.arange(seq, device="cuda").unsqueeze(0)

        def step():
            loss = m(ids, pos, None, labels=ids).mean()
            loss.backward()
            return loss.detach()
        step()
        loss, peak = _peak(step)
        peaks.append(peak)
        losses.append(float(loss))
        # RMSNorm makes hidden states of norm sqrt(1024): no logit is larger than this
        z = 32 * float(m.output_layer.weight.detach().float().norm(dim=1).max())
        del m
    assert peaks[1] <= peaks[0], [p / MIB for p in peaks]
    # the layers are the same; bf16 logits move each loss by at most twice 2^-8 of the largest, the heads' as much times their factor of 0.1
    assert abs(losses[0] - losses[1]) <= 1.1 * 2 * 2.0 ** -8 * z
