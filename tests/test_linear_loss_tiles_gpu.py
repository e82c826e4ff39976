"""Output projection with its loss where the products run as 256 x 512 tiles, and where kept logits meet the fp32 ``main_grad``.  Tolerances
as in test_linear_cross_entropy_gpu.py."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_linear_cross_entropy_gpu import BF16, FP16, _ce, _ce_target, _compare, _inputs, _kd, _kd_target, _reference, _within  # noqa: E402

pytestmark = pytest.mark.gpu


def _wide(M, N, K, most=1):
    """Whether the kernels' rule (modelled time of the rounds of tiles) takes 256 x 512 tiles for an M x N product that sums over K."""
    pairs, f = torch.cuda.get_device_properties(0).multi_processor_count // 2, np.float32

    def us(splits, width):
        rounds = -(-(-(-M // 256) * -(-N // width) * splits) // pairs)
        blocks = (-(-K // 64) + splits - 1) // splits
        return f(rounds) * (f(0.72) * f(blocks) + f(2) if width == 512 else f(0.40) * f(blocks))
    return min(us(s, 512) for s in range(1, most + 1)) < min(us(s, 256) for s in range(1, most + 1))


def _products(T, V, H):
    """Which products of a training call run wide: (logits of the forward, hidden gradient, weight gradient, logits made again)."""
    from mindspeed_b200.ops import linear_cross_entropy as M
    cols, splits, _, words = M._plan(T, H, V, M.PIECE_BYTES, M.SLAB_BYTES, True)
    part = min(cols, words) if words else min(cols, V)
    return _wide(T, V, H), _wide(T, H, min(cols, V), splits), _wide(part, H, T), words < V and _wide(T, min(cols, V - words), H)


#: T, V, H, logits kept (of how many words), the products that are wide.  The last tile's second half lies past the last word, past the last
#: column of H, or ends inside.
CASES = [(200, 20000, 1728, 0, (True, False, False, True)), (200, 20000, 1728, 20000, (True, False, False, False)),
         (1945, 9748, 272, 0, (False, False, True, False)), (1612, 2086, 2088, 2086, (False, False, True, False)),
         (2235, 3795, 1856, 0, (True, True, True, True)), (2235, 3795, 1856, 3795, (True, True, True, False)),
         (2175, 3440, 1896, 0, (True, True, True, True)), (2060, 2066, 2184, 2066, (True, False, True, False)),
         (4425, 3688, 880, 3688, (False, True, False, False))]


@pytest.fixture(params=CASES, ids=lambda c: "-".join(map(str, c[:4])))
def case(request, monkeypatch):
    from mindspeed_b200.ops import linear_cross_entropy as M
    T, V, H, kept, wide = request.param
    monkeypatch.setattr(M, "KEEP_LEAST", 256)
    monkeypatch.setattr(M, "KEEP_BYTES", 4 * ((T + 7) // 8 * 8) * (kept + 255))
    if not kept:
        monkeypatch.setattr(M, "KEEP_BYTES", 0)
    assert M._plan(T, H, V, M.PIECE_BYTES, M.SLAB_BYTES, True)[3] == kept
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert _products(T, V, H) == wide
    return T, V, H


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("ignored", [0.0, 0.4])
def test_cross_entropy_on_wide_tiles(case, dtype, ignored):
    T, V, H = case
    h, w, fav, g, gen = _inputs(T, V, H, dtype)
    labels = torch.where(torch.rand(T, generator=gen, device="cuda") < ignored, -100, fav)
    _compare(_ce(h, w, labels, g), h, w, _ce_target(labels), 1.0, g)


@pytest.mark.parametrize("K", [5, 40])
def test_distillation_on_wide_tiles(case, K):
    """Short lists beside the product (up to 2048 tokens) and sorted ones from the accumulators; the last words are listed too."""
    T, V, H = case
    h, w, fav, g, gen = _inputs(T, V, H, BF16)
    idx = torch.randint(0, V, (T, K), generator=gen, device="cuda")
    idx[:, 0], idx[:, 1], idx[:, 2] = fav, V - 1, max(0, V - 1 - V % 256)
    idx[:, 4] = idx[:, 3]
    idx = torch.where(torch.rand(T, K, generator=gen, device="cuda") < 0.1, -1, idx)
    idx[7] = -1
    a = torch.randn(T, K, generator=gen, device="cuda") * 3
    _compare(_kd(h, w, a, idx, 2.0, g), h, w, _kd_target(idx, a, 2.0), 2.0, g)


def _into_main_grad(h, w, labels, g, start, **kw):
    from mindspeed_b200.ops.linear_cross_entropy import linear_cross_entropy
    p = torch.nn.Parameter(w.clone())
    p.main_grad = start.clone()
    hg = h.clone().requires_grad_(True)
    loss = linear_cross_entropy(hg, p, labels, accumulate_main_grad=True, **kw)
    loss.backward(g)
    assert p.grad is None and p.grad_added_to_main_grad
    return loss.detach(), hg.grad, p.main_grad


def _compare_main_grad(got, h, w, labels, g, start):
    want, tol = _reference(h, w, *_ce_target(labels), 1.0, g)
    _within(got[0], want[0], tol[0], "loss")
    _within(got[1], want[1], tol[1], "d hidden")
    total = want[2] + start.double()
    _within(got[2], total, tol[2] + total.abs() * 2.0 ** -23, "main_grad")


def test_main_grad_on_wide_tiles(case):
    T, V, H = case
    h, w, fav, g, gen = _inputs(T, V, H, BF16)
    labels = torch.where(torch.rand(T, generator=gen, device="cuda") < 0.3, -100, fav)
    start = torch.randn(V, H, generator=gen, device="cuda")
    _compare_main_grad(_into_main_grad(h, w, labels, g, start), h, w, labels, g, start)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,V,H,words", [(300, 3000, 136, 3000), (300, 3000, 136, 512), (1030, 777, 64, 777), (1, 900, 64, 900), (40, 2049, 72, 2049),
                                         (64, 600, 200, 600), (100, 1300, 1664, 1300)])
@pytest.mark.parametrize("ignored", [0.0, 0.5, 2.0])
def test_main_grad_of_kept_logits(T, V, H, words, ignored, dtype, monkeypatch):
    """Gradients of kept logits (in two terms for up to 64 tokens) added to main_grad, in one piece and in several; rows of the scratch that
    no token has hold NaN."""
    from mindspeed_b200.ops import linear_cross_entropy as M
    h, w, fav, g, gen = _inputs(T, V, H, dtype)
    labels = torch.where(torch.rand(T, generator=gen, device="cuda") < ignored, -100, fav)
    start = torch.randn(V, H, generator=gen, device="cuda")
    monkeypatch.setattr(M, "KEEP_WIDTH", 64)
    monkeypatch.setattr(M, "KEEP_LEAST", 256)
    monkeypatch.setattr(M, "KEEP_BYTES", 4 * ((T + 7) // 8 * 8) * (words + 255 if words == V else words))
    for piece in (M.PIECE_BYTES, 2 * T * 300):
        monkeypatch.setattr(M, "PIECE_BYTES", piece)
        assert M._plan(T, H, V, M.PIECE_BYTES, M.SLAB_BYTES, True)[3] == words
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        poison = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 16, 1 << 18, 1 << 20, 1 << 22, 1 << 22)]
        del poison
        got = _into_main_grad(h, w, labels, g, start)
        _compare_main_grad(got, h, w, labels, g, start)
        if ignored == 2.0:
            assert torch.equal(got[2], start) and not got[1].any() and not got[0].any()


def test_small_steps_follow_the_gradient():
    """Central differences along directions that are small enough for the bound to be below half of the slope: at most four entries of a token
    and two of a word move, by one unit in their grid and along the gradient's own sign.  Bounds: the third derivative of log-sum-exp along
    dz is at most 2 max |dz|^3; u = 2^-8 of each gradient entry for the roundings of dz, of the result, and one more for their product; and
    the losses' own errors."""
    from mindspeed_b200.ops.linear_cross_entropy import linear_cross_entropy
    T, V, H = 16, 200, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randint(-8, 9, (V, H), generator=gen, device="cuda") / 64).to(BF16)
    h = (torch.randint(-16, 17, (T, H), generator=gen, device="cuda") / 16).to(BF16)
    lab = torch.randint(0, V, (T,), generator=gen, device="cuda")
    one = torch.ones(T, device="cuda")
    _, gh, gw = _ce(h, w, lab, one)
    own = _reference(h, w, *_ce_target(lab), 1.0, one)[1][0].sum() * 1.1              # of the losses at either end

    def largest(grad, k, unit):
        at = grad.float().abs().topk(k, 1)[1]
        return torch.zeros_like(grad, dtype=torch.float32).scatter_(1, at, unit) * grad.float().sign()

    def along(e, dh, dw):
        hh, ww = (h.float() + e * dh).to(BF16), (w.float() + e * dw).to(BF16)
        assert torch.equal(hh.float(), h.float() + e * dh) and torch.equal(ww.float(), w.float() + e * dw)
        return linear_cross_entropy(hh, ww, lab).double().sum()

    dirh, dirw = largest(gh, 4, 1 / 16), largest(gw, 2, 1 / 64)
    for dh, dw, slope in ((dirh, 0 * dirw, (gh.double() * dirh).sum()), (0 * dirh, dirw, (gw.double() * dirw).sum())):
        diff = (along(1, dh, dw) - along(-1, dh, dw)) / 2
        step = (dh.double().abs() @ w.double().abs().t() + h.double().abs() @ dw.double().abs().t()).amax(1)
        tol = float((step ** 3 / 3).sum() + 3 * 2.0 ** -8 * ((gh.double() * dh).abs().sum() + (gw.double() * dw).abs().sum()) + own)
        assert tol < 0.5 * float(slope)
        assert abs(float(diff - slope)) <= tol
