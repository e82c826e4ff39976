"""Balance loss of a mixture-of-experts router with its per-expert counts (csrc/kernels/balance_loss.cu).

``router_balance_loss(logits, routing_map, topk, coeff)`` gives what ``moe_utils.switch_load_balancing_loss_func`` (``batch_size=1``) or
``sequence_load_balancing_loss_func`` (``batch_size=b``) make of the scores, the scores themselves included: one pass over logits and
map forward, one backward.  On a CPU it runs as eager PyTorch.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import loader
from ._dtypes import CODE, code
from .linear_cross_entropy import _on_device

_F = ctypes.c_float
MAX_EXPERTS = 1024


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, routing_map, scale, sigmoid, B):
        L = loader.require_lib()
        dev = logits.device
        x, rmap = logits.contiguous(), routing_map.contiguous()
        T, E = x.shape
        S = T // B
        with _on_device(dev):
            blocks = L.msb_balance_blocks(S, B, E)
            n = B * blocks * E
            parts = B * ((E + 31) // 32)
            buf = torch.empty(2 * n + parts + 1, dtype=torch.float32, device=dev)     # sums of p, counts, joined products, ticket
            load = torch.empty(B, E, dtype=torch.float32, device=dev)
            loss = torch.empty((), dtype=torch.float32, device=dev)
            counts = torch.empty(E, dtype=torch.int64, device=dev)
            b = buf.data_ptr()
            P = ctypes.c_void_p
            loader.check(L.msb_balance_forward(loader.p(x), loader.p(rmap), S, B, E, int(sigmoid), _F(scale), code(x.dtype), P(b), P(b + 4 * n),
                                               blocks, loader.p(load), P(b + 8 * n), P(b + 8 * n + 4 * parts), loader.p(loss),
                                               loader.p(counts), P(loader.stream_ptr())), "balance_forward")
        ctx.save_for_backward(x, load)
        ctx.meta = (scale, sigmoid, B)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        if g is None:
            return None, None, None, None, None
        L = loader.require_lib()
        x, load = ctx.saved_tensors
        x = x.contiguous()
        scale, sigmoid, B = ctx.meta
        T, E = x.shape
        with _on_device(x.device):
            g = g.float()
            grad = torch.empty_like(x)
            loader.check(L.msb_balance_backward(loader.p(x), loader.p(load), T // B, B, E, int(sigmoid), _F(scale), loader.p(g), code(x.dtype),
                                                loader.p(grad), ctypes.c_void_p(loader.stream_ptr())), "balance_backward")
        return grad, None, None, None, None


def _balance_ref(logits, routing_map, scale, sigmoid, B):
    T, E = logits.shape
    x = logits if logits.dtype == torch.float64 else logits.float()
    if sigmoid:
        s = torch.sigmoid(x)
        p = s / (s.sum(-1, keepdim=True) + 1e-20)
    else:
        p = torch.softmax(x, dim=-1)
    f = routing_map.reshape(T // B, B, E).sum(0)
    loss = (p.reshape(T // B, B, E).sum(0) * f.to(p.dtype)).sum() * scale
    return loss, f.sum(0)


def router_balance_loss(logits, routing_map, topk, coeff, score_function="softmax", batch_size=1):
    """(balance loss, tokens per expert [E] int64) of router ``logits`` [T, E] and the boolean ``routing_map`` [T, E].

    Tokens are in [sequence, batch] order.  The loss is ``coeff E / (S^2 topk B) sum_b sum_e P_be f_be`` over the ``B = batch_size`` sequences
    of ``S = T / B`` tokens, with P the sum of the scores (``softmax``, or ``sigmoid`` divided by its sum over the experts) and f the number
    of entries of the map; ``batch_size=1`` balances over all tokens together.  Its gradient reaches the logits through P."""
    if logits.dim() != 2 or routing_map.shape != logits.shape:
        raise ValueError(f"router_balance_loss: logits {tuple(logits.shape)} and routing map {tuple(routing_map.shape)} do not fit")
    T, E = logits.shape
    if T == 0 or E == 0 or batch_size < 1 or T % batch_size or topk < 1:
        raise ValueError(f"router_balance_loss: {T} tokens of {E} experts, {batch_size} sequences, top {topk}")
    if score_function not in ("softmax", "sigmoid"):
        raise ValueError(f"router_balance_loss: unknown score function {score_function}")
    if routing_map.dtype != torch.bool or not logits.dtype.is_floating_point:
        raise TypeError(f"router_balance_loss: logits are {logits.dtype}, the routing map {routing_map.dtype}")
    if routing_map.device != logits.device:
        raise ValueError(f"router_balance_loss: logits on {logits.device}, routing map on {routing_map.device}")
    S = T // batch_size
    scale = float(coeff) * E / (float(S) * S * topk * batch_size)
    sigmoid = score_function == "sigmoid"
    if loader.use_kernels(logits):
        if logits.dtype not in CODE:
            raise TypeError(f"router_balance_loss: the sm_100a kernels take fp32, bf16 or fp16, not {logits.dtype}")
        if E > MAX_EXPERTS or T > 1 << 24:
            raise ValueError(f"router_balance_loss: {E} experts (at most {MAX_EXPERTS}), {T} tokens (at most 2^24)")
        return _BalanceLoss.apply(logits, routing_map, scale, sigmoid, int(batch_size))
    return _balance_ref(logits, routing_map, scale, sigmoid, int(batch_size))
