"""The loss operators together, as a training step uses them: one student's hidden states and output weight under cross entropy, a teacher's
top logits and the balance loss of a router that reads the same hidden states; and a mixture-of-experts model that trains with them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_one_student_under_three_losses():
    """Gradients of the sum against 64 bits.  Bounds: each operator's gradient entries d carry half a step u of bf16 and errors of the scores
    (2 H 2^-23 sum |h w| in a logit), its products round once more (u), and autograd adds the parts in bf16 (u of each partial sum)."""
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    from mindspeed_b200.ops.linear_cross_entropy import linear_cross_entropy, linear_topk_distillation
    T, V, H, E, K, k, tau, coeff = 320, 2000, 256, 16, 12, 2, 2.0, 0.5
    gen = torch.Generator(device="cuda").manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    h = rn(T, H).to(BF16).requires_grad_(True)
    w = (rn(V, H) * 0.1).to(BF16).requires_grad_(True)
    r = (rn(E, H) * 0.1).requires_grad_(True)
    lab = torch.randint(0, V, (T,), generator=gen, device="cuda")
    lab[::5] = -100
    idx, a = torch.randint(0, V, (T, K), generator=gen, device="cuda"), rn(T, K)
    g = 1.0 / T

    x = h.float() @ r.t()
    rmap = torch.zeros(T, E, dtype=torch.bool, device="cuda").scatter_(1, x.detach().topk(k, 1)[1], True)
    bal, counts = router_balance_loss(x, rmap, k, coeff)
    total = linear_cross_entropy(h, w, lab).sum() * g + linear_topk_distillation(h, w, a, idx, tau).sum() * g + bal
    gh, gw, gr = torch.autograd.grad(total, (h, w, r))
    assert torch.equal(counts, rmap.sum(0))

    hd, wd, rd = (t.detach().double() for t in (h, w, r))
    keep = (lab != -100).double()[:, None]
    z = hd @ wd.t()
    p1, p2 = torch.softmax(z, 1), torch.softmax(z / tau, 1)
    q = torch.softmax(a.double() / tau, 1)
    logq = torch.log_softmax(a.double() / tau, 1)
    d1 = (p1 - torch.zeros_like(z).scatter_(1, lab.clamp(min=0)[:, None], 1.0)) * keep * g
    d2 = (p2 - torch.zeros_like(z).scatter_add_(1, idx, q)) * tau * g
    xr = hd @ rd.t()
    pr = torch.softmax(xr, 1)
    f = rmap.sum(0).double()
    C = coeff * E / (T * T * k)
    dx = C * pr * (f - (pr * f).sum(1, keepdim=True))
    ce = ((torch.logsumexp(z, 1) - z.gather(1, lab.clamp(min=0)[:, None])[:, 0]) * keep[:, 0]).sum() * g
    kd = (tau * tau * (q * (logq - torch.log_softmax(z / tau, 1).gather(1, idx))).sum(1)).sum() * g
    want = ce + kd + C * (pr.sum(0) * f).sum()
    dz = (2 * H * 2.0 ** -23 * (hd.abs() @ wd.abs().t())).amax(1, keepdim=True)
    assert abs(float(total.detach()) - float(want)) <= float(((2 + tau) * dz).mean()) + 2.0 ** -17 * float(want.abs())
    u = 2.0 ** -8
    e1, e2 = u * d1.abs() + p1 * torch.expm1(2 * dz) * keep * g, u * d2.abs() + p2 * torch.expm1(2 * dz) * tau * g
    parts = [(d1 @ wd, e1 @ wd.abs() * 1.01), (d2 @ wd, e2 @ wd.abs() * 1.01), (dx @ rd, 2.0 ** -16 * (dx.abs() + C * pr * f) @ rd.abs())]
    tol = sum(e + u * m.abs() * 1.01 for m, e in parts) + u * sum(m.abs() for m, _ in parts) * 2.1 + V * 2.0 ** -23 * ((d1.abs() + d2.abs()) @ wd.abs())
    assert not ((gh.double() - sum(m for m, _ in parts)).abs() > tol).any()
    parts = [(d1.t() @ hd, e1.t() @ hd.abs() * 1.01), (d2.t() @ hd, e2.t() @ hd.abs() * 1.01)]
    tol = sum(e + u * m.abs() * 1.01 for m, e in parts) + u * sum(m.abs() for m, _ in parts) * 1.1 + T * 2.0 ** -23 * ((d1.abs() + d2.abs()).t() @ hd.abs())
    assert not ((gw.double() - sum(m for m, _ in parts)).abs() > tol).any()
    assert not ((gr.double() - dx.t() @ hd).abs() > 2.0 ** -16 * ((dx.abs() + C * pr * f).t() @ hd.abs())).any()


def _model(fused, score, kind):
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    F = torch.nn.functional
    cfg = TransformerConfig(num_layers=2, hidden_size=256, num_attention_heads=4, ffn_hidden_size=512, hidden_dropout=0.0, attention_dropout=0.0,
                            optimization_level=1, params_dtype=BF16, bf16=True, gated_linear_unit=True, activation_func=F.silu,
                            add_bias_linear=False, normalization="RMSNorm", num_moe_experts=8, moe_router_topk=2, moe_ffn_hidden_size=256,
                            moe_grouped_gemm=True, moe_token_dispatcher_type="alltoall", moe_aux_loss_coeff=0.01, moe_router_score_function=score,
                            moe_router_load_balancing_type=kind, linear_cross_entropy_fusion=fused, moe_balance_loss_fusion=fused)
    torch.manual_seed(7)
    return GPTModel(cfg, vocab_size=3000, max_sequence_length=128, position_embedding_type="rope").cuda().train()


@pytest.fixture(scope="module")
def one_rank():
    """A process group of this process alone, gone again (and nothing left in the environment) when the module's tests end."""
    import socket
    import torch.distributed as dist
    from mindspeed_b200.parallel import parallel_state as ps
    from mindspeed_b200.parallel.random import model_parallel_cuda_manual_seed
    mine = not dist.is_initialized()
    if mine:
        with socket.socket() as s:
            s.bind(("127.0.0.1", 0))
            port = s.getsockname()[1]
        dist.init_process_group("nccl", init_method=f"tcp://127.0.0.1:{port}", rank=0, world_size=1)
    parallel = not ps.model_parallel_is_initialized()
    if parallel:
        ps.initialize_model_parallel()
    model_parallel_cuda_manual_seed(1)
    yield
    if parallel:
        ps.destroy_model_parallel()
    if mine:
        dist.destroy_process_group()


@pytest.mark.parametrize("score,kind", [("softmax", "aux_loss"), ("sigmoid", "seq_aux_loss")])
def test_mixture_of_experts_model(one_rank, score, kind):
    """With and without the fused losses.  Without, the logits are rounded to bf16 (2^-8 of up to max |z|), which moves a loss by up to twice
    that and a probability by exp of it; the gradients are compared by their 2-norms, whose two sides each carry bf16 roundings of every
    layer: 2^-8 a layer and product, some ten of them in a row."""
    ids = torch.randint(0, 3000, (2, 128), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    pos = torch.arange(128, device="cuda").expand(2, -1)
    got = []
    first = _model(False, score, kind)
    for fused in (False, True):
        m = _model(fused, score, kind)
        m.load_state_dict(first.state_dict())            # expert weights come from a random stream that goes on
        with torch.no_grad():
            z = m(ids, pos, None).float().abs().max()
        loss = m(ids, pos, None, labels=ids)
        loss.mean().backward()
        got.append((loss.detach(), {n: p.grad.float() for n, p in m.named_parameters() if p.grad is not None}, float(z)))
    (la, ga, z), (lb, gb, _) = got
    assert la.shape == lb.shape == (2, 128) and lb.dtype == torch.float32
    assert float((la - lb).abs().max()) <= 2 * 2.0 ** -8 * z + 1e-4
    assert ga.keys() == gb.keys()
    for n in ga:
        assert torch.isfinite(gb[n]).all()
        assert float((ga[n] - gb[n]).norm()) <= 10 * 2.0 ** -8 * float(ga[n].norm()) + 1e-12, n
    assert any("router" in n for n in ga)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("accumulate", [False, True])
def test_dense_model_and_main_grad(one_rank, tied, accumulate):
    """Output weight of its own or the embedding's, gradients returned or added to fp32 main_grad; bounds as above."""
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    ids = torch.randint(0, 3000, (2, 96), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    labels = ids.roll(-1, 1)
    pos = torch.arange(96, device="cuda").expand(2, -1)
    got, state = [], None
    for fused in (False, True):
        cfg = TransformerConfig(num_layers=1, hidden_size=256, num_attention_heads=4, ffn_hidden_size=512, hidden_dropout=0.0, attention_dropout=0.0,
                                optimization_level=1, params_dtype=BF16, bf16=True, add_bias_linear=False, normalization="RMSNorm",
                                gradient_accumulation_fusion=accumulate, linear_cross_entropy_fusion=fused)
        m = GPTModel(cfg, vocab_size=3000, max_sequence_length=96, position_embedding_type="rope",
                     share_embeddings_and_output_weights=tied).cuda().train()
        state = m.state_dict() if state is None else state
        m.load_state_dict(state)
        if accumulate:
            for p in m.parameters():
                p.main_grad = torch.zeros_like(p, dtype=torch.float32)
        losses = []
        for _ in range(2):                          # two micro-batches
            loss = m(ids, pos, None, labels=labels)
            loss.mean().backward()
            losses.append(loss.detach())
        assert torch.equal(*losses)
        got.append((losses[0], {n: (p.main_grad.clone() if accumulate else 0) + (p.grad.float() if p.grad is not None else 0)
                                for n, p in m.named_parameters()}))
    (la, ga), (lb, gb) = got
    assert float((la - lb).abs().max()) <= 2 * 2.0 ** -8 * 8 + 1e-4
    for n in ga:
        assert torch.isfinite(gb[n]).all() and gb[n].any()
        assert float((ga[n] - gb[n]).norm()) <= 10 * 2.0 ** -8 * float(ga[n].norm()) + 1e-12, n
