"""Output projection and its loss in one operator, which holds a bounded part of the [tokens, vocab] matrix of logits at most
(csrc/kernels/linear_ce_sm100.cu).

  linear_cross_entropy(hidden, weight, labels)                                  per-token cross entropy of softmax(hidden weight^T)
  linear_topk_distillation(hidden, weight, teacher_logits, teacher_indices)     per-token tau^2 KL(teacher's top words || student)

Both take ``hidden`` [..., H] and ``weight`` [V, H] in bf16 or fp16 (H a multiple of 8) and return the loss in fp32 with the leading shape
of ``hidden``; any gradient may come back on it.  Tokens without a label (``ignore_index``) or without a teacher word (all indices negative,
or all teacher logits -inf) have loss 0 and no gradient, whatever their hidden states hold, and cost nothing in the products.

Memory.  From the forward to the backward a call keeps a copy of the hidden states (packed where tokens left), the listed logits and
weights (8 bytes a listed word), and, in training, at most ``KEEP_BYTES`` (2 GiB) of fp32 logits, as far as they go over the vocabulary;
the backward makes the others again.  The backward works on a piece of the vocabulary at a time: 16-bit gradients of its logits
(``PIECE_BYTES``, 512 MiB) and fp32 parts of the hidden gradient (``SLAB_BYTES``, 256 MiB, or one part where that is more).  That can be
more than the 16-bit logits of all tokens (4096 x 129280: 2.8 GB next to 1.1): ``memory_limit`` bounds all of it, in bytes, and what
does not fit is made again.  The least that a call can do with is the copy, one part of the hidden gradient and a piece of 256 words; the
forward's statistics (9 bytes a token and 128 words) come and go before the pieces and are not counted.  Calls of few tokens, at most 64 or
a sixteenth of H, are not limited and keep all logits: an eighth of the weight's bytes (for rows rounded up to 8), or 256 bytes a word.

A label or teacher index beyond the vocabulary gives its token loss NaN and no gradient, and makes ``ops.gemm.check_status`` raise.

With ``group`` the weight holds this rank's slice of the vocabulary (rank r has words [r V, (r + 1) V)), ``hidden`` and the targets are the
same on every rank, the loss is that of the whole vocabulary, and the gradient of ``hidden`` is this rank's part: the caller sums it
over the group (``mappings.copy_to_tensor_model_parallel_region`` or the sequence-parallel gather in front of the operator does).

``accumulate_main_grad`` adds the weight's gradient straight to the fp32 ``weight.main_grad``, as the parallel linears do under gradient
accumulation fusion; autograd then gets none.

On a CPU the same functions run as eager PyTorch.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools

import torch
import torch.distributed as dist

from . import gemm as G
from . import loader
from ._dtypes import code

_P, _I, _LL, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float

#: bytes of the 16-bit logit gradients that the backward holds at a time, and of the fp32 partial results of the hidden gradient
PIECE_BYTES = 512 << 20
SLAB_BYTES = 256 << 20
#: most bytes of fp32 logits that a call keeps from its forward to its backward, which then makes those of the remaining words again.  0 keeps
#: none (but for few tokens).  A kept logit costs what its bytes take, making it again 2 H / 1.3 PFLOP/s: at least KEEP_WIDTH hidden columns
#: (both directions, us, made again -> kept: 1024 x 128256 x 512 579 -> 606, 766 x 50257 x 768 333 -> 316, 2048 x 32000 x 1024 515 -> 485,
#: 2048 x 50000 x 1536 1065 -> 945, 4096 x 129280 x 4096 13000 -> 10700), and at least KEEP_LEAST words, which fill the products' tiles.
KEEP_BYTES = 2 << 30
KEEP_WIDTH = 640
KEEP_LEAST = 8192
MAX_LIST = 1024
#: up to so many tokens the logits are kept whatever H is, and their gradients go into the products in two 16-bit terms
TWO_ROWS = 64


class _Args(ctypes.Structure):
    _fields_ = [("hidden", _P), ("weight", _P), ("idx", _P), ("teacher", _P), ("ldh", _LL), ("ldw", _LL), ("vocab_start", _LL), ("vocab", _LL),
                ("ignore_index", _LL), ("T", _I), ("H", _I), ("V", _I), ("K", _I), ("dtype", _I), ("tau", _F), ("pos", _P), ("rowmap", _P),
                ("count", _P), ("kind", _P), ("sorted", _P), ("packed", _P), ("z", _P), ("q", _P), ("dot", _P), ("ent", _P), ("lse", _P), ("loss", _P),
                ("part", _P), ("part_at", _P), ("zt", _P), ("ldt", _I), ("kept", _I), ("mx", _P), ("sum", _P), ("g", _P), ("g_stride", _LL), ("dz", _P), ("ldz", _LL), ("piece", _I), ("acc", _P),
                ("splits", _I), ("slab_rows", _I), ("dhidden", _P), ("dweight", _P), ("dweight_fp32_add", _I), ("scale", _P), ("status", _P)]


_STAY = contextlib.nullcontext()


def _on_device(dev):
    """Makes ``dev`` the current device for the launches inside; nothing where it is already."""
    return _STAY if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _status(dev):
    if dev not in G._status and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the first call of a process on a device sets up its error words and cannot be captured; run the operator once before")
    return G.status_word(dev)


def _rows(t):
    """``t`` [rows, H] as the kernels read it: unit inner stride, rows on 16-byte boundaries that do not overlap."""
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t
    ld = t.shape[1] if t.shape[0] == 1 else t.stride(0)
    if t.stride(1) != 1 or ld % 8 or ld < t.shape[1] or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _plan(T, H, V, piece_bytes, slab_bytes, train, keep_bytes=None):
    """(columns of a piece, most K splits of the hidden gradient, pitch of kept logits, words whose logits are kept)."""
    return _planned(T, H, V, piece_bytes, slab_bytes, train, KEEP_BYTES if keep_bytes is None else keep_bytes, KEEP_WIDTH, KEEP_LEAST)


def _budget(T, H, V, K, limit):
    """(bytes of a piece, of the hidden gradient's parts, of kept logits) for a call that may hold ``limit`` bytes: an eighth for the parts, a
    quarter for the piece and what is left for logits; the piece gets all of that where none are kept.  Few tokens are not limited: their
    logits are small next to the weight, and pieces of some hundred words would cost many launches."""
    if limit is None or T <= TWO_ROWS or 16 * T <= H:
        return PIECE_BYTES, SLAB_BYTES, KEEP_BYTES
    ldt = (T + 7) // 8 * 8
    least = 512 * ldt                                     # a piece of 256 words
    rest = max(0, limit - (2 * T * H + 8 * T * K + 12 * T + 16))
    slab = min(SLAB_BYTES, limit // 8, max(0, rest - least))
    rest = max(0, rest - max(slab, (T + 31) // 32 * 32 * H * 4))
    piece = min(PIECE_BYTES, limit // 4)
    keep = min(KEEP_BYTES, rest - max(piece, least))
    if keep <= 0 or not _plan(T, H, V, piece, slab, True, keep)[3]:
        piece, keep = min(PIECE_BYTES, rest), 0
    return piece * T // ldt, slab, keep


@functools.lru_cache(maxsize=64)
def _planned(T, H, V, piece_bytes, slab_bytes, train, keep_bytes, keep_width, keep_least):
    """The device chooses among the splits for the rows that stay (choose_splits in the kernel file); more of them than fill the 74 SM pairs
    four times are never better.  The logits of all words are kept where they take, in fp32, at most an eighth of the weight's bytes, or
    64 rows; else, where that is faster, of as many words as go into ``keep_bytes``."""
    cols = min(max(256, piece_bytes // (2 * T) // 256 * 256), (V + 255) // 256 * 256)
    tiles = -(-H // 256)
    splits = max(1, min(64, -(-296 // tiles), slab_bytes // ((T + 31) // 32 * 32 * H * 4)))
    ldt = TWO_ROWS if T <= TWO_ROWS else (T + 7) // 8 * 8
    kept = 0
    if train and (T <= TWO_ROWS or 16 * T <= H):
        kept = V
    elif train and H >= keep_width:
        kept = min(V, keep_bytes // (4 * ldt) // 256 * 256)
        kept = kept if kept >= min(V, keep_least) else 0
    return cols, splits, ldt if kept else 0, kept


def _lib():
    L = loader.require_lib()
    if L.msb_lce_forward.argtypes is None:
        L.msb_lce_backward.argtypes = [ctypes.POINTER(_Args), _P]
        L.msb_lce_rescale.argtypes = [_P, _P, _P, _F, _P, _I, _P]
        L.msb_lce_loss.argtypes = [_P, _P, _P, _P, _P, _P, _F, _I, _P, _P, _P]
        L.msb_lce_forward.argtypes = [ctypes.POINTER(_Args), _P]
    return L


class _Job:
    """One call: its targets and what stays the same in both directions.  (Autograd passes it along as one argument; every argument of a
    function costs host time, and short calls are bound by that.)"""
    __slots__ = ("idx", "teacher", "K", "tau", "ignore_index", "group", "world", "rank", "main_grad", "limit", "train", "plan", "shape")

    def __init__(self, hidden, weight, idx, teacher, K, tau, ignore_index, group, main_grad, limit):
        self.idx, self.teacher, self.K, self.tau, self.ignore_index, self.group = idx, teacher, K, tau, ignore_index, group
        self.limit = limit
        self.world, self.rank = (1, 0) if group is None else (dist.get_world_size(group), dist.get_rank(group))
        self.main_grad = weight if main_grad else None
        self.train = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad)

    def args(self, h, w, idx, teacher, kept):
        """The argument block with what both directions need.  ``kept``: [packed rows | logits of few rows | z, q, lse | pos, rowmap, count],
        4-byte words."""
        (T, H), (V, _) = h.shape, w.shape
        K = self.K
        piece, splits, ldt, words = self.plan
        at = kept.data_ptr()
        z = at + 2 * T * H + 4 * words * ldt
        pos = z + 8 * T * K + 4 * T
        return _Args(hidden=h.data_ptr(), weight=w.data_ptr(), idx=idx.data_ptr(), teacher=None if teacher is None else teacher.data_ptr(),
                     ldh=h.stride(0) if T > 1 else H, ldw=w.stride(0) if V > 1 else H, vocab_start=self.rank * V, vocab=self.world * V,
                     ignore_index=self.ignore_index, T=T, H=H, V=V, K=K, dtype=code(h.dtype), tau=self.tau, packed=at,
                     zt=at + 2 * T * H if ldt else None, ldt=ldt, kept=words, z=z, q=z + 4 * T * K, lse=z + 8 * T * K, pos=pos, rowmap=pos + 4 * T,
                     count=pos + 8 * T, piece=piece, splits=splits, status=_status(h.device).data_ptr())


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, job):
        L = _lib()
        dev = hidden.device
        h, w = _rows(hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])), _rows(weight)
        (T, H), V, K = h.shape, w.shape[0], job.K
        piece_bytes, slab_bytes, keep_bytes = _budget(T, H, V, K, job.limit)
        job.plan = _plan(T, H, V, piece_bytes, slab_bytes, job.train, keep_bytes)
        job.shape = hidden.shape
        _, _, ldt, words = job.plan
        with _on_device(dev):
            kept = torch.empty(T * H // 2 + words * ldt + 2 * T * K + 3 * T + 2, dtype=torch.float32, device=dev)
            parts = (V + 255) // 256 * 2
            lists = 0 if job.teacher is None else 2 * T * K
            scratch = torch.empty(lists + 2 * parts * T + 4 * T + (parts * T + T + 3) // 4, dtype=torch.float32, device=dev)
            loss = torch.empty(hidden.shape[:-1], dtype=torch.float32, device=dev)
            a = job.args(h, w, job.idx, job.teacher, kept)
            a.loss = loss.data_ptr()
            a.sorted = at = scratch.data_ptr()
            a.part = at = at + 4 * lists
            a.dot = at = at + 8 * parts * T
            a.ent = at + 4 * T
            a.part_at = at + 16 * T
            a.kind = at + 16 * T + parts * T
            st = loader.stream_ptr()
            if job.world > 1:
                at = lists + 2 * parts * T
                dot, ent, mx, sm = (scratch[at + i * T:at + (i + 1) * T] for i in range(4))
                a.mx, a.sum = mx.data_ptr(), sm.data_ptr()
            loader.check(L.msb_lce_forward(a, st), "linear_ce_forward")
            if job.world > 1:
                gmx = mx.clone()
                dist.all_reduce(gmx, op=dist.ReduceOp.MAX, group=job.group)
                loader.check(L.msb_lce_rescale(sm.data_ptr(), mx.data_ptr(), gmx.data_ptr(), job.tau, a.count, T, st), "linear_ce_rescale")
                dist.all_reduce(sm, group=job.group)
                dist.all_reduce(dot, group=job.group)
                loader.check(L.msb_lce_loss(gmx.data_ptr(), sm.data_ptr(), dot.data_ptr(), ent.data_ptr(), a.rowmap, a.count, job.tau, T, a.lse,
                                            loss.data_ptr(), st), "linear_ce_loss")
        if job.train:
            # targets that come from inference mode cannot be kept as they are
            ctx.save_for_backward(h, w, *(t.clone() if t is not None and t.is_inference() else t for t in (job.idx, job.teacher)), kept)
            job.idx = job.teacher = None          # the saved ones count: hooks may have moved them
            ctx.job = job
        return loss

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            raise RuntimeError("linear loss operators have no second derivative (create_graph)")
        L = _lib()
        h, w, idx, teacher, kept = ctx.saved_tensors
        job = ctx.job
        need_h, need_w, _ = ctx.needs_input_grad
        dev = h.device
        h, w = _rows(h), _rows(w)
        (T, H), V = h.shape, w.shape[0]
        piece, splits, ldt, words = job.plan
        with _on_device(dev):
            one = not any(g.stride()) or g.numel() == 1      # an expanded scalar, as a sum's backward gives
            if not one and not g.is_contiguous():
                g = g.contiguous()
            two = ldt and T <= TWO_ROWS
            ldz = 0 if words == V else min(piece, (V + 7) // 8 * 8)
            slab_rows = 2 * TWO_ROWS if two else (T + 31) // 32 * 32
            dz_words = max(min(piece, words) * (2 if two else 1) * ldt, T * ldz) // 2
            scratch = torch.empty(dz_words + (splits * slab_rows * H if need_h else 0) + 2, dtype=torch.float32, device=dev)
            a = job.args(h, w, idx, teacher, kept)
            a.g, a.g_stride = g.data_ptr(), 0 if one else 1
            a.dz = at = scratch.data_ptr()
            a.ldz, a.slab_rows = ldz, slab_rows
            dh = dw = None
            if h.dtype == torch.float16:
                a.scale = at + 4 * (scratch.numel() - 2)
            if need_h:
                dh = torch.empty(job.shape, dtype=h.dtype, device=dev)
                a.acc, a.dhidden = at + 4 * dz_words, dh.data_ptr()
            param = job.main_grad
            if need_w:
                if param is not None:
                    a.dweight, a.dweight_fp32_add = param.main_grad.data_ptr(), 1
                else:
                    dw = torch.empty(V, H, dtype=h.dtype, device=dev)
                    a.dweight = dw.data_ptr()
            loader.check(L.msb_lce_backward(a, loader.stream_ptr()), "linear_ce_backward")
        if need_w and param is not None:
            param.grad_added_to_main_grad = True
            cb = getattr(param, "_main_grad_ready_cb", None)
            if cb is not None:
                cb(param)
        return dh, dw, None


class _SumOverGroup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, group):
        x = x.clone()
        dist.all_reduce(x, group=group)
        return x

    @staticmethod
    def backward(ctx, g):
        return g, None


def _linear_loss_ref(hidden, weight, idx, q, ent, tau, group):
    """Eager form: ``idx``, ``q`` [T, K] with q = 0 in unused places, ``ent`` [T] = sum q log q; rows whose q are all 0 are left out."""
    world = 1 if group is None else dist.get_world_size(group)
    rank = 0 if group is None else dist.get_rank(group)
    V = weight.shape[0]
    keep = (q.sum(1) != 0).nonzero().squeeze(1)          # (a teacher's NaN stays in)
    x = hidden.reshape(-1, hidden.shape[-1]).index_select(0, keep)
    idx, q, ent_k = idx.index_select(0, keep), q.index_select(0, keep), ent.index_select(0, keep)
    z = (x.float() @ weight.float().t()) / tau
    with torch.no_grad():
        m = z.amax(1, keepdim=True)
        if world > 1:
            dist.all_reduce(m, op=dist.ReduceOp.MAX, group=group)
    s = torch.exp(z - m).sum(1)
    local = idx - rank * V
    here = (local >= 0) & (local < V) & (q > 0)
    picked = torch.where(here, z.gather(1, local.clamp(0, V - 1)), torch.zeros_like(q))
    dot = (q * picked).sum(1)
    if world > 1:
        s, dot = _SumOverGroup.apply(s, group), _SumOverGroup.apply(dot, group)
    loss = (ent_k + (m.squeeze(1) - dot) + torch.log(s)) * (tau * tau)
    out = torch.zeros(ent.shape[0], dtype=torch.float32, device=hidden.device).index_put((keep,), loss)
    return out.reshape(hidden.shape[:-1])


def _check(name, hidden, weight, target, accumulate_main_grad, memory_limit):
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{name}: hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} do not fit")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"{name}: empty weight {tuple(weight.shape)}")
    if hidden.dtype != weight.dtype or not hidden.dtype.is_floating_point:
        raise TypeError(f"{name}: hidden is {hidden.dtype}, weight {weight.dtype}")
    if target.dtype.is_floating_point or target.dtype.is_complex or target.dtype == torch.bool:
        raise TypeError(f"{name}: labels and indices are integers, not {target.dtype}")
    if not (hidden.device == weight.device == target.device):
        raise ValueError(f"{name}: hidden on {hidden.device}, weight on {weight.device}, targets on {target.device}")
    if memory_limit is not None and not memory_limit >= 0:
        raise ValueError(f"{name}: memory_limit is a number of bytes or None, not {memory_limit}")
    if accumulate_main_grad:
        mg = getattr(weight, "main_grad", None)
        if mg is None or mg.dtype != torch.float32 or mg.shape != weight.shape or not mg.is_contiguous() or mg.device != weight.device:
            raise ValueError(f"{name}: accumulate_main_grad needs a contiguous fp32 main_grad of the weight's shape")
    if hidden.is_cuda:
        if hidden.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{name}: the sm_100a kernels take bf16 or fp16, not {hidden.dtype}")
        if hidden.shape[-1] % 8:
            raise ValueError(f"{name}: the hidden size {hidden.shape[-1]} is not a multiple of 8")
        if accumulate_main_grad and weight.main_grad.data_ptr() % 16:
            raise ValueError(f"{name}: main_grad is not on a 16-byte boundary")
        if hidden.numel() // hidden.shape[-1] >= 2 ** 31 - 256 or weight.shape[0] >= 2 ** 31 - 256:
            raise ValueError(f"{name}: more than 2^31 tokens or words")


def _none(hidden, weight):
    """Loss of no tokens: shape [..., 0], zero gradients."""
    return hidden.float().sum(-1) + weight[:0].float().sum()


def _main_grad_hook(weight):
    """The eager form's weight for ``accumulate_main_grad``: its gradient goes to main_grad instead of autograd."""
    w = weight.detach().requires_grad_(weight.requires_grad)
    if weight.requires_grad:
        def add(grad):
            weight.main_grad.add_(grad)
            weight.grad_added_to_main_grad = True
            cb = getattr(weight, "_main_grad_ready_cb", None)
            if cb is not None:
                cb(weight)
            return grad
        w.register_hook(add)
    return w


def linear_cross_entropy(hidden, weight, labels, ignore_index=-100, group=None, accumulate_main_grad=False, memory_limit=None):
    """Cross entropy of ``softmax(hidden @ weight.T)`` against ``labels`` [...], per token, fp32."""
    _check("linear_cross_entropy", hidden, weight, labels, accumulate_main_grad, memory_limit)
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: labels {tuple(labels.shape)} for hidden {tuple(hidden.shape)}")
    if labels.numel() == 0:
        return _none(hidden, weight)
    idx = labels if labels.dtype == torch.int64 and labels.is_contiguous() else labels.long().contiguous()
    if loader.use_kernels(hidden):
        return _LinearLoss.apply(hidden, weight, _Job(hidden, weight, idx, None, 1, 1.0, int(ignore_index), group, accumulate_main_grad,
                                                       None if memory_limit is None else int(memory_limit)))
    idx = idx.reshape(-1)
    world = 1 if group is None else dist.get_world_size(group)
    kept = idx != ignore_index
    if bool(((idx < 0) | (idx >= world * weight.shape[0]))[kept].any()):
        raise IndexError("linear_cross_entropy: a label outside the vocabulary")
    w = _main_grad_hook(weight) if accumulate_main_grad else weight
    q = kept.float().unsqueeze(1)
    return _linear_loss_ref(hidden, w, idx.unsqueeze(1), q, torch.zeros_like(q[:, 0]), 1.0, group)


def linear_topk_distillation(hidden, weight, teacher_logits, teacher_indices, temperature=1.0, group=None, accumulate_main_grad=False,
                             memory_limit=None):
    """``temperature^2 KL(q || p)`` per token, fp32: q is the softmax of ``teacher_logits`` [..., K] at the temperature over the listed words
    ``teacher_indices`` [..., K] (negative: unused place; a word may be listed more than once), p the student's softmax over the whole
    vocabulary.  The teacher gets no gradient."""
    name = "linear_topk_distillation"
    _check(name, hidden, weight, teacher_indices, accumulate_main_grad, memory_limit)
    K = teacher_indices.shape[-1] if teacher_indices.dim() else 0
    if teacher_logits.shape != teacher_indices.shape or teacher_indices.shape[:-1] != hidden.shape[:-1]:
        raise ValueError(f"{name}: teacher logits {tuple(teacher_logits.shape)} and indices {tuple(teacher_indices.shape)} "
                         f"for hidden {tuple(hidden.shape)}")
    if not 1 <= K <= MAX_LIST:
        raise ValueError(f"{name}: {K} listed words a token (1 to {MAX_LIST})")
    if not teacher_logits.dtype.is_floating_point or teacher_logits.device != hidden.device:
        raise ValueError(f"{name}: teacher logits are {teacher_logits.dtype} on {teacher_logits.device}")
    tau = float(temperature)
    if not 0.0 < tau < float("inf"):
        raise ValueError(f"{name}: the temperature must be positive, got {temperature}")
    if teacher_indices.numel() == 0:
        return _none(hidden, weight)
    idx = teacher_indices.reshape(-1, K).long().contiguous()
    a = teacher_logits.detach().reshape(-1, K).float().contiguous()
    if loader.use_kernels(hidden):
        return _LinearLoss.apply(hidden, weight, _Job(hidden, weight, idx, a, K, tau, 0, group, accumulate_main_grad,
                                                       None if memory_limit is None else int(memory_limit)))
    world = 1 if group is None else dist.get_world_size(group)
    if bool((idx >= world * weight.shape[0]).any()):
        raise IndexError(f"{name}: a teacher index outside the vocabulary")
    used = (idx >= 0) & (a != float("-inf"))
    logq = torch.where(used, a / tau, torch.full_like(a, float("-inf")))
    logq = logq - torch.logsumexp(logq, 1, keepdim=True)
    q = torch.where(used, torch.exp(logq), torch.zeros_like(a))
    ent = torch.where(q > 0, q * logq, torch.zeros_like(a)).sum(1)
    w = _main_grad_hook(weight) if accumulate_main_grad else weight
    return _linear_loss_ref(hidden, w, idx, q, ent, tau, group)
