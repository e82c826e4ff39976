"""A dense model with and without --linear-cross-entropy-fusion, held to the bound of its own largest logit."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_loss_operators_gpu import one_rank  # noqa: E402, F401

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("seq", [96, 40])
def test_losses_of_a_dense_model(one_rank, tied, seq):  # noqa: F811
    """Without the flag the logits are rounded to bf16, by at most 2^-8 of the largest, which moves a loss by up to twice that; 1e-4 is for the
    exponentials and sums of losses of about ten."""
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    ids = torch.randint(0, 3000, (2, seq), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    pos = torch.arange(seq, device="cuda").expand(2, -1)
    losses, z, state = [], 0.0, None
    for fused in (False, True):
        cfg = TransformerConfig(num_layers=1, hidden_size=256, num_attention_heads=4, ffn_hidden_size=512, hidden_dropout=0.0, attention_dropout=0.0,
                                optimization_level=1, params_dtype=BF16, bf16=True, add_bias_linear=False, normalization="RMSNorm",
                                linear_cross_entropy_fusion=fused)
        m = GPTModel(cfg, vocab_size=3000, max_sequence_length=seq, position_embedding_type="rope",
                     share_embeddings_and_output_weights=tied).cuda().train()
        state = m.state_dict() if state is None else state
        m.load_state_dict(state)
        with torch.no_grad():
            z = max(z, float(m(ids, pos, None).float().abs().max()))
            losses.append(m(ids, pos, None, labels=ids.roll(-1, 1)))
    assert 0 < z and float((losses[0] - losses[1]).abs().max()) <= 2 * 2.0 ** -8 * z + 1e-4
