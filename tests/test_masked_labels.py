"""Labels that are no word of the vocabulary (padding other than -100) under --linear-cross-entropy-fusion and --kl-teacher-topk: what a loss
mask takes out may hold anything, as it may without the flags."""
import pytest
import torch


def _model(fused, mtp=None, device="cpu", dtype=torch.float32):
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    cfg = TransformerConfig(num_layers=1, hidden_size=32, num_attention_heads=2, use_cpu_initialization=True, linear_cross_entropy_fusion=fused,
                            hidden_dropout=0.0, attention_dropout=0.0, mtp_num_layers=mtp, params_dtype=dtype, bf16=dtype == torch.bfloat16)
    torch.manual_seed(0)
    return GPTModel(cfg, vocab_size=40, max_sequence_length=16).to(device).train()


def _masked_step(fused, labels, mask, mtp=None, device="cpu", dtype=torch.float32):
    m = _model(fused, mtp, device, dtype)
    ids = torch.arange(32, device=device).reshape(2, 16)
    loss = m(ids, torch.arange(16, device=device).expand(2, -1), None, labels=labels.to(device))
    total = (loss * mask.to(device)).sum()
    total.backward()
    return total.detach().cpu(), {n: p.grad.cpu() for n, p in m.named_parameters() if p.grad is not None}


def _padded():
    labels = torch.arange(32).reshape(2, 16).roll(-1, 1)
    mask = torch.ones(2, 16)
    for at, bad in (((0, 15), -1), ((1, 3), -2), ((1, 14), 40), ((0, 7), 2 ** 40), ((1, 15), -100)):
        labels[at] = bad
        mask[at] = 0
    return labels, mask


def test_masked_labels_may_hold_anything():
    labels, mask = _padded()
    want, grads = _masked_step(False, labels, mask)
    got, fused = _masked_step(True, labels, mask)
    assert torch.isfinite(got) and torch.allclose(got, want, rtol=1e-5) and grads.keys() == fused.keys()
    for n in grads:
        assert torch.allclose(fused[n], grads[n], atol=1e-5), n


def test_masked_labels_of_multi_token_heads():
    """A head's label is the one some tokens on: a masked label is another position's there, so the mask goes with it."""
    labels, mask = _padded()
    mask = mask * mask.roll(-1, 1)
    want, grads = _masked_step(False, labels, mask, mtp=1)
    got, fused = _masked_step(True, labels, mask, mtp=1)
    assert torch.isfinite(got) and torch.allclose(got, want, rtol=1e-5)
    for n in grads:
        assert torch.allclose(fused[n], grads[n], atol=1e-5), n


def test_reported_cross_entropy_of_the_distillation():
    labels, mask = _padded()
    m = _model(True)
    ids = torch.arange(32).reshape(2, 16)
    targets = (torch.zeros(2, 16, 3), torch.arange(96).reshape(2, 16, 3) % 40)
    kl, ce = m(ids, torch.arange(16).expand(2, -1), None, labels=labels, distill_targets=targets)
    plain = _model(False)(ids, torch.arange(16).expand(2, -1), None, labels=labels)
    assert torch.isfinite(kl).all() and torch.allclose((ce * mask).sum(), (plain * mask).sum(), rtol=1e-5)


@pytest.mark.gpu
def test_masked_labels_on_the_gpu():
    from mindspeed_b200.ops.gemm import check_status
    labels, mask = _padded()
    check_status()
    want, grads = _masked_step(False, labels, mask, device="cuda", dtype=torch.bfloat16)
    got, fused = _masked_step(True, labels, mask, device="cuda", dtype=torch.bfloat16)
    check_status()                                           # no word outside the vocabulary is reported
    # bf16 logits, below 4 here, move each of the 27 losses by at most twice 2^-8 of that
    assert torch.isfinite(got) and abs(float(got) - float(want)) <= 27 * 2 * 2.0 ** -8 * 4 + 1e-3
    for n in grads:
        assert torch.isfinite(fused[n]).all()
