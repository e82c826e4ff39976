"""Router balance loss on the sm_100a kernels, against the formulas in 64 bits.

Tolerances.  A score is off by a few units of 2^-22 (approximate exponential and division, a sum of up to 1024 terms): 2^-18 of itself is
safe.  Sums over T tokens in fp32 add T 2^-24 at most.  The gradient's bracket f - sum p f loses up to 2^-18 sum p f by subtraction; bf16
and fp16 gradients are rounded once (half a step)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _reference(x, rmap, topk, coeff, score, B):
    x = x.double()
    T, E = x.shape
    S = T // B
    if score == "softmax":
        p = torch.softmax(x, 1)
        slope = p
    else:
        s = torch.sigmoid(x)
        n = s.sum(1, keepdim=True) + 1e-20
        p, slope = s / n, s * torch.sigmoid(-x) / n
    f = rmap.view(S, B, E).sum(0).double()
    C = coeff * E / (S * S * topk * B)
    loss = C * (p.view(S, B, E).sum(0) * f).sum()
    fr = f.unsqueeze(0).expand(S, B, E).reshape(T, E)
    dot = (p * fr).sum(1, keepdim=True)
    return loss, C * slope * (fr - dot), C * slope * (fr + dot) * 2.0 ** -18


def _case(T, E, k, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + T + E)
    x = (torch.randn(T, E, generator=gen, device="cuda") * 2).to(dtype)
    idx = x.float().topk(k, 1)[1]
    return x, torch.zeros(T, E, dtype=torch.bool, device="cuda").scatter_(1, idx, True)


def _run(x, rmap, k, score, B, g=1.0):
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    x = x.detach().requires_grad_(True)
    loss, counts = router_balance_loss(x, rmap, k, 0.01, score_function=score, batch_size=B)
    (gx,) = torch.autograd.grad(loss * g, (x,))
    return loss.detach(), counts, gx


@pytest.mark.parametrize("T,E,k,B", [(1, 1, 1, 1), (1, 8, 2, 1), (7, 5, 2, 1), (64, 2, 1, 4), (500, 64, 6, 4), (1023, 33, 8, 3), (4096, 256, 8, 1),
                                     (300, 60, 4, 2), (129, 1000, 8, 3), (65, 1023, 3, 1), (20000, 16, 2, 2), (96, 130, 2, 1), (50, 512, 8, 2),
                                     (40, 1024, 2, 4), (70000, 8, 2, 1), (34, 4, 1, 17), (8191, 64, 4, 1), (513, 129, 2, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_values_and_gradient(T, E, k, B, score, dtype):
    T = T // B * B
    x, rmap = _case(T, E, k, dtype)
    loss, counts, gx = _run(x, rmap, k, score, B, 3.0)
    want, grad, tol = _reference(x, rmap, k, 0.01, score, B)
    assert torch.equal(counts, rmap.sum(0)) and counts.dtype == torch.int64
    assert abs(float(loss) - float(want)) <= float(want) * (2.0 ** -18 + T * 2.0 ** -24)
    u = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bad = (gx.double() - 3 * grad).abs() > 3 * tol * (1 + u) + u * 3 * grad.abs() + sub
    assert not bad.any(), float((gx.double() - 3 * grad).abs().max())


def test_layouts_extremes_and_bits():
    x, rmap = _case(300, 64, 6, torch.float32)
    base = _run(x, rmap, 6, "softmax", 3)
    wide = torch.full((300, 72), float("nan"), device="cuda")
    wide[:, :64] = x
    odd = torch.empty(300 * 64 + 1, device="cuda")[1:].view(300, 64).copy_(x)                # 4 bytes off: one expert a load
    for y in (_run(wide[:, :64], rmap, 6, "softmax", 3), _run(x.t().contiguous().t(), rmap.t().contiguous().t(), 6, "softmax", 3),
              _run(x, rmap, 6, "softmax", 3)):
        assert all(torch.equal(a, b) for a, b in zip(y, base))
    got = _run(odd, rmap, 6, "softmax", 3)
    want, grad, tol = _reference(x, rmap, 6, 0.01, "softmax", 3)
    assert torch.equal(got[1], base[1]) and not ((got[2].double() - grad).abs() > tol).any()
    # an expert that is switched off, one that takes all, saturated sigmoids, a map without entries
    y = x.clone()
    y[:, 3] = float("-inf")
    y[:, 5] = 200.0
    y[:, 6] = -200.0
    for score in ("softmax", "sigmoid"):
        loss, counts, gx = _run(y, rmap, 6, score, 1)
        want, grad, tol = _reference(y, rmap, 6, 0.01, score, 1)
        assert torch.isfinite(gx).all() and not ((gx.double() - grad).abs() > tol + 1e-36).any()
        assert abs(float(loss) - float(want)) <= 2.0 ** -17 * float(want)
        loss, counts, gx = _run(x, torch.zeros_like(rmap), 6, score, 1)
        assert float(loss) == 0 and not counts.any() and not gx.any()
    z = x.clone()
    z[7, 2] = float("nan")
    assert torch.isnan(_run(z, rmap, 6, "softmax", 1)[0])


def test_captured_and_on_a_side_stream():
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    x, rmap = _case(512, 64, 6, torch.float32)
    base = _run(x, rmap, 6, "sigmoid", 2)
    xs, ms = x.clone().requires_grad_(True), rmap.clone()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(_run(x, rmap, 6, "sigmoid", 2), base))
        with torch.cuda.graph(graph, stream=side):
            loss, counts = router_balance_loss(xs, ms, 6, 0.01, score_function="sigmoid", batch_size=2)
            (gx,) = torch.autograd.grad(loss, (xs,))
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2):
        x2, m2 = _case(512, 64, 6, torch.float32, seed)
        with torch.no_grad():
            xs.copy_(x2)
        ms.copy_(m2)
        graph.replay()
        assert all(torch.equal(a.detach(), b) for a, b in zip((loss, counts, gx), _run(x2, m2, 6, "sigmoid", 2)))


def test_refusals_on_the_gpu():
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    x, rmap = _case(8, 4, 2, torch.float32)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        router_balance_loss(x.double(), rmap, 2, 0.01)
    with pytest.raises(ValueError, match="at most 1024"):
        router_balance_loss(torch.zeros(2, 1025, device="cuda"), torch.zeros(2, 1025, dtype=torch.bool, device="cuda"), 2, 0.01)
    with pytest.raises(ValueError, match="on cpu"):
        router_balance_loss(x, rmap.cpu(), 2, 0.01)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,batch", [(512, 2, 1), (4096, 6, 4), (3000, 256, 3)])
def test_balanced_loads_have_no_gradient(T, E, batch, score):
    """Every expert takes every token: f is the same for all, and f_e - sum p f is 0 but for what the sigmoid's normaliser adds, a factor
    of 1e-20 / sum s (at most 1e-18 here) of f = S.  The gradient is that times at most C g."""
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    x = torch.randn(T, E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(T)).requires_grad_(True)
    loss, counts = router_balance_loss(x, torch.ones(T, E, dtype=torch.bool, device="cuda"), E, 0.01, score, batch)
    loss.backward()
    S = T // batch
    assert bool((counts == T).all())
    assert float(x.grad.abs().max()) <= 1e-18 * S * 0.01 * E / (S * S * E * batch)


def test_scores_that_do_not_add_up_to_one():
    """Sigmoids so small that the normaliser's 1e-20 counts, against the formula in 64 bits.  A score's relative error is at most 2^-20, and
    the differences of the loads are exact: each of the E + 2 terms of f_e - sum p f is off by 2^-19 of the largest load."""
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    T, E = 64, 12
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = (-46 + torch.randn(T, E, device="cuda", generator=gen)).requires_grad_(True)
    rmap = torch.rand(T, E, device="cuda", generator=gen) < torch.linspace(0.2, 0.9, E, device="cuda")
    loss, _ = router_balance_loss(x, rmap, 2, 0.01, "sigmoid")
    loss.backward()
    s = torch.sigmoid(x.detach().double())
    n = s.sum(1, keepdim=True) + 1e-20
    f = rmap.double().sum(0)
    c = 0.01 * E / (T * T * 2)
    slope = s * (1 - s) / n * c
    want = slope * (f - (s / n * f).sum(1, keepdim=True))
    assert ((x.grad.double() - want).abs() <= slope * f.max() * (E + 2) * 2.0 ** -19).all()
    assert abs(float(loss) - float(c * ((s / n).sum(0) * f).sum())) <= 2.0 ** -18 * float(loss)
