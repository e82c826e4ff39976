"""Routers whose batches are beyond what the balance loss's kernels take keep the plain form; the operator names its limits."""
import types

import pytest
import torch


@pytest.mark.parametrize("tokens,sequences,dtype,takes", [(4096, 4, torch.float32, True), (1 << 24, 65535, torch.float32, True),
                                                          ((1 << 24) + 1, 1, torch.float32, False), (1 << 20, 65536, torch.float32, False),
                                                          (4096, 4, torch.float64, False)])
@pytest.mark.parametrize("on_gpu", [True, False])
def test_router_asks_for_what_the_kernels_take(tokens, sequences, dtype, takes, on_gpu):
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.parallel.moe.router import TopKRouter
    cfg = TransformerConfig(num_layers=2, hidden_size=32, num_attention_heads=2, num_moe_experts=6, moe_router_topk=2, moe_aux_loss_coeff=0.05,
                            use_cpu_initialization=True, moe_router_load_balancing_type="seq_aux_loss", moe_balance_loss_fusion=True)
    r = TopKRouter(cfg, layer_number=1).train()
    logits = types.SimpleNamespace(is_cuda=on_gpu, dtype=dtype, shape=(tokens, 6))
    assert r._fused_aux(logits, (tokens // sequences, sequences)) == (takes or not on_gpu)


def test_operator_names_its_limits(monkeypatch):
    from mindspeed_b200.ops import balance_loss as M
    monkeypatch.setattr(M.loader, "use_kernels", lambda t: True)
    x, rmap = torch.zeros(65536, 2), torch.zeros(65536, 2, dtype=torch.bool)
    with pytest.raises(ValueError, match="65535"):
        M.router_balance_loss(x, rmap, 1, 0.1, batch_size=65536)
