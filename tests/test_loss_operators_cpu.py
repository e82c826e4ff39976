"""Loss operators on the CPU: eager forms against the formulas, vocabulary-parallel ranks over gloo, refusals, and the paths that call them
(GPTModel, multi-token heads, quantisation-aware distillation, the router)."""
import os
import sys
import tempfile

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from dist_utils import run_distributed  # noqa: E402
from test_checkpoint_cpu import ARGS  # noqa: E402

from mindspeed_b200.ops.balance_loss import router_balance_loss  # noqa: E402
from mindspeed_b200.ops.linear_cross_entropy import linear_cross_entropy, linear_topk_distillation  # noqa: E402

F = torch.nn.functional


def _inputs(T=23, V=57, H=16, K=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g, requires_grad=True)
    w = torch.randn(V, H, generator=g, requires_grad=True)
    lab = torch.randint(0, V, (T,), generator=g)
    lab[::4] = -100
    idx = torch.randint(0, V, (T, K), generator=g)
    idx[1, 2:] = -1
    idx[2] = -1
    a = torch.randn(T, K, generator=g)
    a[3, 1] = float("-inf")
    return h, w, lab, idx, a, torch.randn(T, generator=g)


def test_cross_entropy_is_torch():
    h, w, lab, _, _, g = _inputs()
    loss = linear_cross_entropy(h, w, lab)
    want = F.cross_entropy((h.double() @ w.double().t()), lab, reduction="none", ignore_index=-100)
    assert loss.dtype == torch.float32 and torch.allclose(loss.double(), want, atol=1e-5) and (loss[::4] == 0).all()
    for x, y in zip(torch.autograd.grad(loss, (h, w), g), torch.autograd.grad(want, (h, w), g.double())):
        assert torch.allclose(x, y, atol=1e-5)
    shaped = linear_cross_entropy(h[:20].view(4, 5, 16), w, lab[:20].view(4, 5).int())
    assert shaped.shape == (4, 5) and torch.equal(shaped.reshape(-1), loss[:20])
    assert torch.equal(linear_cross_entropy(h, w, torch.where(lab == -100, 9, lab), ignore_index=9)[lab == -100], torch.zeros(6))


def test_left_out_rows_hold_anything():
    h, w, lab, _, _, g = _inputs()
    d = h.detach().clone()
    d[lab == -100] = float("nan")
    d.requires_grad_(True)
    clean = torch.autograd.grad(linear_cross_entropy(h, w, lab), (h, w), g)
    dirty = torch.autograd.grad(linear_cross_entropy(d, w, lab), (d, w), g)
    assert all(torch.equal(x, y) for x, y in zip(clean, dirty))


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distillation_is_the_divergence(tau):
    h, w, _, idx, a, g = _inputs()
    loss = linear_topk_distillation(h, w, a, idx, tau)
    z = (h.double() @ w.double().t()) / tau
    lp = F.log_softmax(z, 1)
    want = []
    for t in range(idx.shape[0]):
        ks = [k for k in range(idx.shape[1]) if idx[t, k] >= 0 and a[t, k] != float("-inf")]
        lq = F.log_softmax(a[t, ks].double() / tau, 0)
        want.append(tau * tau * sum((lq[j].exp() * (lq[j] - lp[t, idx[t, k]]) for j, k in enumerate(ks)), torch.zeros((), dtype=torch.float64)))
    want = torch.stack(want)
    assert torch.allclose(loss.double(), want, atol=1e-4) and loss[2] == 0
    for x, y in zip(torch.autograd.grad(loss, (h, w), g), torch.autograd.grad(want, (h, w), g.double())):
        assert torch.allclose(x, y.float(), atol=1e-4)


def test_whole_vocabulary_is_the_full_divergence():
    from mindspeed_b200.qat.qad import kl_from_logits, teacher_top_logits
    h, w, _, _, _, _ = _inputs()
    teacher = torch.randn(h.shape[0], w.shape[0], generator=torch.Generator().manual_seed(4))
    v, i = teacher_top_logits(teacher, w.shape[0])
    full, _ = kl_from_logits(h @ w.t(), teacher, None, 2.0, "sum")
    assert torch.allclose(linear_topk_distillation(h, w, v, i, 2.0).sum(), full, rtol=1e-5)
    with pytest.raises(ValueError, match="vocabulary of 57"):
        teacher_top_logits(teacher, 58)


def test_gradients_follow_differences():
    h, w, lab, idx, a, g = _inputs(T=6, V=11, H=8)
    for f in (lambda h, w: (linear_cross_entropy(h, w, lab).double() * g).sum(),
              lambda h, w: (linear_topk_distillation(h, w, a, idx, 2.0).double() * g).sum()):
        grads = torch.autograd.grad(f(h, w), (h, w))
        gen = torch.Generator().manual_seed(1)
        dh, dw = torch.randn(h.shape, generator=gen), torch.randn(w.shape, generator=gen)
        e = 1e-2
        with torch.no_grad():
            diff = (f(h + e * dh, w + e * dw) - f(h - e * dh, w - e * dw)) / (2 * e)
        slope = sum(float((x * d).sum()) for x, d in zip(grads, (dh, dw)))
        # fp32 losses of size 10 differ by 1e-6 x 10 / e; third derivatives times e^2
        assert float(diff) == pytest.approx(slope, abs=2e-2 * max(1.0, abs(slope)))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_loss_is_the_one_of_the_router(score):
    from mindspeed_b200.parallel.moe.moe_utils import sequence_load_balancing_loss_func, switch_load_balancing_loss_func
    g = torch.Generator().manual_seed(2)
    x = torch.randn(24, 6, generator=g, requires_grad=True)
    rmap = torch.zeros(24, 6, dtype=torch.bool).scatter_(1, x.detach().topk(2, 1)[1], True)
    p = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x) / (torch.sigmoid(x).sum(-1, keepdim=True) + 1e-20)
    for b, want in ((1, switch_load_balancing_loss_func(p, rmap.sum(0).float(), 2, 0.01)),
                    (4, sequence_load_balancing_loss_func(p, rmap, 4, 6, 2, 0.01))):
        loss, counts = router_balance_loss(x, rmap, 2, 0.01, score, b)
        assert torch.allclose(loss, want, rtol=1e-6) and torch.equal(counts, rmap.sum(0)) and not counts.requires_grad
        assert torch.allclose(torch.autograd.grad(loss, x)[0], torch.autograd.grad(want, x, retain_graph=True)[0], atol=1e-9)


def test_logits_that_are_kept():
    from mindspeed_b200.ops import linear_cross_entropy as M
    def kept(T, H, V, train=True, keep=M.KEEP_BYTES):
        return M._plan(T, H, V, M.PIECE_BYTES, M.SLAB_BYTES, train, keep)[2:]
    assert kept(1, 64, 1000) == (64, 1000) and kept(64, 64, 1000, keep=0) == (64, 1000)      # few tokens
    assert kept(100, 1600, 500000, keep=0) == (104, 500000)                                  # an eighth of the weight's bytes
    assert kept(101, 1600, 500000, keep=0) == (0, 0) == kept(101, 1600, 500000, train=False) == kept(1, 64, 1000, train=False)
    assert kept(4096, 4096, 32001) == (4096, 32001)
    assert kept(4090, 512, 32001) == (0, 0) and kept(4090, 1024, 32001) == (4096, 32001)                                                 # making them again costs less
    T, V = 30001, 150000
    ldt, words = kept(T, 4096, V)
    assert ldt == 30008 and words % 256 == 0 and 4 * ldt * words <= M.KEEP_BYTES < 4 * ldt * (words + 256)
    assert kept(2 ** 17, 4096, V) == (0, 0)                                                  # too few words to fill the products


def test_teacher_without_a_number():
    from mindspeed_b200.ops.linear_cross_entropy import linear_topk_distillation
    h, w = torch.randn(3, 8), torch.randn(10, 8)
    a, idx = torch.zeros(3, 2), torch.tensor([[0, 1]] * 3)
    a[1, 0] = float("nan")
    loss = linear_topk_distillation(h, w, a, idx)
    assert torch.isnan(loss).tolist() == [False, True, False]


def test_refusals():
    h, w, lab, idx, a, _ = _inputs()
    for call, err, msg in ((lambda: linear_cross_entropy(h, w[:, :8], lab), ValueError, "do not fit"),
                           (lambda: linear_cross_entropy(h, w[:0], lab), ValueError, "empty weight"),
                           (lambda: linear_cross_entropy(h.bfloat16(), w, lab), TypeError, "weight torch.float32"),
                           (lambda: linear_cross_entropy(h, w, lab.float()), TypeError, "integers"),
                           (lambda: linear_cross_entropy(h, w, lab[:5]), ValueError, "labels"),
                           (lambda: linear_cross_entropy(h, w, torch.full_like(lab, 57)), IndexError, "outside"),
                           (lambda: linear_cross_entropy(h, w, torch.full_like(lab, -1)), IndexError, "outside"),
                           (lambda: linear_cross_entropy(h, w, lab, accumulate_main_grad=True), ValueError, "main_grad"),
                           (lambda: linear_topk_distillation(h, w, a[:, :2], idx), ValueError, "teacher logits"),
                           (lambda: linear_topk_distillation(h, w, a, idx, 0.0), ValueError, "temperature"),
                           (lambda: linear_topk_distillation(h, w, a, idx, float("nan")), ValueError, "temperature"),
                           (lambda: linear_topk_distillation(h, w, a, torch.full_like(idx, 57)), IndexError, "outside"),
                           (lambda: linear_topk_distillation(h, w, torch.zeros(23, 1025), torch.zeros(23, 1025, dtype=torch.long)), ValueError, "1025"),
                           (lambda: linear_topk_distillation(h, w, idx, idx), ValueError, "teacher logits are")):
        with pytest.raises(err, match=msg):
            call()
    x, rmap = torch.zeros(8, 4), torch.zeros(8, 4, dtype=torch.bool)
    for call, err in ((lambda: router_balance_loss(x, rmap[:7], 2, 0.1), ValueError), (lambda: router_balance_loss(x, rmap, 2, 0.1, "relu"), ValueError),
                      (lambda: router_balance_loss(x, rmap, 2, 0.1, batch_size=3), ValueError), (lambda: router_balance_loss(x, rmap.int(), 2, 0.1), TypeError),
                      (lambda: router_balance_loss(x[:0], rmap[:0], 2, 0.1), ValueError)):
        with pytest.raises(err):
            call()


def test_first_call_is_not_captured(monkeypatch):
    from mindspeed_b200.ops import gemm as G
    from mindspeed_b200.ops import linear_cross_entropy as M
    monkeypatch.setattr(G, "_status", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        M._status(torch.device("cpu"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert M._status(torch.device("cpu")).numel() == 4


def test_status_words_name_the_vocabulary(monkeypatch):
    from mindspeed_b200.ops import gemm as G
    words = torch.tensor([0, 0x703, 0, 0], dtype=torch.int32)
    monkeypatch.setattr(G, "_status", {torch.device("cpu"): words})
    with pytest.raises(RuntimeError, match="outside the vocabulary"):
        G.check_status()
    assert not words.any()
    G.check_status()
    words[0] = 0x21
    with pytest.raises(RuntimeError, match="time-out"):
        G.check_status()


def test_no_tokens():
    h, w, lab, idx, a, _ = _inputs()
    for loss in (linear_cross_entropy(h[:0], w, lab[:0]), linear_topk_distillation(h[:0], w, a[:0], idx[:0])):
        assert loss.shape == (0,) and loss.dtype == torch.float32
        gh, gw = torch.autograd.grad(loss.sum(), (h, w))
        assert not gh.any() and not gw.any()
    every = torch.full_like(lab, -100)
    gh, gw = torch.autograd.grad(linear_cross_entropy(h, w, every).sum(), (h, w))
    assert not gh.any() and not gw.any()


def test_main_grad():
    h, w, lab, _, _, g = _inputs()
    p = torch.nn.Parameter(w.detach().clone())
    p.main_grad = torch.ones_like(p)
    seen = []
    p._main_grad_ready_cb = seen.append
    linear_cross_entropy(h, p, lab, accumulate_main_grad=True).backward(g)
    (gw,) = torch.autograd.grad(linear_cross_entropy(h, w, lab), (w,), g)
    assert p.grad is None and seen == [p] and p.grad_added_to_main_grad and torch.allclose(p.main_grad, gw + 1, atol=1e-6)


def _ranks(rank, world):
    import torch.distributed as dist
    dist.init_process_group("gloo", rank=rank, world_size=world)
    grp = dist.group.WORLD
    h, w, lab, idx, a, g = _inputs(V=58)
    per = 58 // world
    ws = w.detach()[rank * per:(rank + 1) * per].requires_grad_(True)
    out = []
    for f in (lambda h, w, grp: linear_cross_entropy(h, w, lab, group=grp), lambda h, w, grp: linear_topk_distillation(h, w, a, idx, 2.0, group=grp)):
        loss, whole = f(h, ws, grp), f(h, w, None)
        gh, gw = torch.autograd.grad(loss, (h, ws), g)
        dist.all_reduce(gh)
        fh, fw = torch.autograd.grad(whole, (h, w), g)
        out.append([float((loss - whole).abs().max()), float((gh - fh).abs().max()), float((gw - fw[rank * per:(rank + 1) * per]).abs().max())])
    dist.destroy_process_group()
    return out


def test_vocabulary_parallel_ranks():
    for r in run_distributed(_ranks, 2):
        assert all(x < 2e-5 for one in r for x in one), r


def _pretrain(rank, world, tp, extra, load=None, save=None, iters=2):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    import pretrain_gpt as pg
    from mindspeed_b200.ops import linear_cross_entropy as M
    from mindspeed_b200.qat import qad
    from mindspeed_b200.training import pretrain
    qad.reset()
    calls = []
    for name in ("linear_cross_entropy", "linear_topk_distillation"):
        own = getattr(M, name)
        setattr(M, name, lambda *a, _own=own, _n=name, **k: (calls.append(_n), _own(*a, **k))[1])
    args = ARGS + ["--tensor-model-parallel-size", str(tp), "--train-iters", str(iters)] + list(extra)
    args += (["--load", load] if load else []) + (["--save", save] if save else [])
    hist = pretrain(pg.train_valid_test_datasets_provider, pg.model_provider, forward_step_func=pg.forward_step, args_list=args)
    return [h["lm loss"] for h in hist], [h.get("kl loss") for h in hist], calls


@pytest.mark.parametrize("tp,extra", [(1, []), (2, ["--sequence-parallel"]), (2, [])])
def test_training_with_the_fused_loss_is_training(tp, extra):
    plain = run_distributed(_pretrain, tp, tp, extra)[0]
    fused = run_distributed(_pretrain, tp, tp, extra + ["--linear-cross-entropy-fusion"])[0]
    assert "linear_cross_entropy" in fused[2] and not plain[2]
    assert fused[0] == pytest.approx(plain[0], rel=1e-5)


def test_multi_token_heads_use_it_too():
    extra = ["--mtp-num-layers", "1"]
    plain = run_distributed(_pretrain, 1, 1, extra)[0]
    fused = run_distributed(_pretrain, 1, 1, extra + ["--linear-cross-entropy-fusion"])[0]
    assert len(fused[2]) >= 4 and len(fused[2]) % 2 == 0 and fused[0] == pytest.approx(plain[0], rel=1e-5)


def test_student_distils_from_the_teachers_top_logits():
    with tempfile.TemporaryDirectory() as d:
        run_distributed(_pretrain, 1, 1, [], None, d)
        q = ["--qad-enable", "--qad-teacher-load", d, "--finetune", "--qat-scheme", "w4a16", "--qat-quant-block-size", "32", "--lr", "2e-3",
             "--kl-temperature", "2.0"]
        full = run_distributed(_pretrain, 1, 1, q, d)[0]
        top = run_distributed(_pretrain, 1, 1, q + ["--kl-teacher-topk", "8"], d)[0]
        assert "linear_topk_distillation" in top[2] and top[1][0] > 1e-6
        assert top[0][0] == pytest.approx(full[0][0], rel=1e-4)                    # the cross entropy beside it
        two = run_distributed(_pretrain, 2, 2, q + ["--kl-teacher-topk", "8"], d)[0]
        assert two[1][0] == pytest.approx(top[1][0], rel=2e-3) and two[0][0] == pytest.approx(top[0][0], rel=1e-4)


def test_output_layer_that_is_watched_is_called():
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.models.gpt_model import GPTModel
    from mindspeed_b200.parallel import parallel_state as ps
    cfg = TransformerConfig(num_layers=1, hidden_size=32, num_attention_heads=2, use_cpu_initialization=True, linear_cross_entropy_fusion=True,
                            hidden_dropout=0.0, attention_dropout=0.0)
    torch.manual_seed(0)
    m = GPTModel(cfg, vocab_size=40, max_sequence_length=16)
    ids = torch.randint(0, 40, (2, 16))
    pos = torch.arange(16).expand(2, -1)
    a = m(ids, pos, None, labels=ids)
    seen = []
    m.output_layer.register_forward_hook(lambda *x: seen.append(1))
    b = m(ids, pos, None, labels=ids)
    assert seen and a.shape == b.shape == (2, 16) and torch.allclose(a, b, atol=1e-5)
    with pytest.raises(RuntimeError, match="not replaced"):
        m(ids, pos, None, labels=ids, distill_targets=(torch.zeros(2, 16, 3), torch.zeros(2, 16, 3, dtype=torch.long)))
    del ps


@pytest.mark.parametrize("score,kind,bias", [("softmax", "aux_loss", False), ("sigmoid", "seq_aux_loss", True)])
def test_router_with_the_fused_balance_loss(score, kind, bias):
    from mindspeed_b200.config import TransformerConfig
    from mindspeed_b200.parallel.moe.router import TopKRouter
    x = torch.randn(8, 3, 32, generator=torch.Generator().manual_seed(1))
    got = []
    for fused in (False, True):
        cfg = TransformerConfig(num_layers=2, hidden_size=32, num_attention_heads=2, num_moe_experts=6, moe_router_topk=2, moe_aux_loss_coeff=0.05,
                                use_cpu_initialization=True, moe_router_score_function=score, moe_router_load_balancing_type=kind,
                                moe_router_enable_expert_bias=bias, moe_balance_loss_fusion=fused)
        torch.manual_seed(3)
        r = TopKRouter(cfg, layer_number=1).train()
        probs, rmap = r(x)
        probs.square().sum().backward()
        got.append((probs.detach(), rmap, r.weight.grad, r.local_tokens_per_expert.clone() if bias else torch.zeros(1)))
    for a, b in zip(*got):
        assert torch.equal(a, b) if a.dtype == torch.bool else torch.allclose(a, b, atol=1e-7)
