"""Balance loss of a mixture-of-experts router with its per-expert counts (csrc/kernels/balance_loss.cu).

``router_balance_loss(logits, routing_map, topk, coeff)`` gives what ``moe_utils.switch_load_balancing_loss_func`` (``batch_size=1``) or
``sequence_load_balancing_loss_func`` (``batch_size=b``) make of the scores, the scores themselves included: one pass over logits and
map forward, one backward.  On a CPU it runs as eager PyTorch.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import loader
from ._dtypes import CODE, code
from .linear_cross_entropy import _on_device

MAX_EXPERTS = 1024


def _lib():
    L = loader.require_lib()
    if L.msb_balance_forward.argtypes is None:
        P, I, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
        L.msb_balance_backward.argtypes = [P, P, I, I, I, I, F, P, I, P, P]
        L.msb_balance_forward.argtypes = [P, P, I, I, I, I, F, I, P, P, I, P, P, P, P, P, P]
    return L


@functools.lru_cache(maxsize=64)
def _blocks(S, B, E):
    return _lib().msb_balance_blocks(S, B, E)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, job):
        routing_map, scale, sigmoid, B = job
        L = _lib()
        dev = logits.device
        x, rmap = logits.contiguous(), routing_map.contiguous()
        T, E = x.shape
        S = T // B
        with _on_device(dev):
            blocks = _blocks(S, B, E)
            n = B * blocks * E
            parts = B * ((E + 31) // 32) if blocks else -1
            buf = torch.empty(B * E + 2 * n + parts + 1, dtype=torch.float32, device=dev)   # loads; sums of p, counts, joined products, ticket
            loss = torch.empty((), dtype=torch.float32, device=dev)
            counts = torch.empty(E, dtype=torch.int64, device=dev)
            load = buf.data_ptr()
            at = load + 4 * B * E
            loader.check(L.msb_balance_forward(x.data_ptr(), rmap.data_ptr(), S, B, E, sigmoid, scale, code(x.dtype), at, at + 4 * n, blocks, load,
                                               at + 8 * n, at + 8 * n + 4 * parts, loss.data_ptr(), counts.data_ptr(), loader.stream_ptr()),
                         "balance_forward")
        ctx.save_for_backward(x, buf)
        ctx.meta = (scale, sigmoid, B)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    def backward(ctx, g, _):
        if g is None:
            return None, None
        if torch.is_grad_enabled():
            raise RuntimeError("router_balance_loss has no second derivative (create_graph)")
        L = _lib()
        x, buf = ctx.saved_tensors
        x = x.contiguous()
        scale, sigmoid, B = ctx.meta
        T, E = x.shape
        with _on_device(x.device):
            grad = torch.empty_like(x)
            loader.check(L.msb_balance_backward(x.data_ptr(), buf.data_ptr(), T // B, B, E, sigmoid, scale, g.data_ptr(), code(x.dtype),
                                                grad.data_ptr(), loader.stream_ptr()), "balance_backward")
        return grad, None


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
        if E > MAX_EXPERTS or T > 1 << 24 or batch_size > 65535:
            raise ValueError(f"router_balance_loss: {E} experts (at most {MAX_EXPERTS}), {T} tokens (at most 2^24), {batch_size} sequences (at "
                             f"most 65535)")
        return _BalanceLoss.apply(logits, (routing_map, scale, int(sigmoid), int(batch_size)))
    return _balance_ref(logits, routing_map, scale, sigmoid, int(batch_size))
