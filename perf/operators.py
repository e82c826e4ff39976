"""What the loss operators are measured on: the output projection with its cross entropy, the same projection with a distillation loss
from a teacher's top logits, and the balance loss of a mixture-of-experts router, each with its gradients.

``run`` is one forward (and, where the case trains, one backward) pass: through the framework's entry points where ``own`` is set, and
otherwise as elementary torch operations in fp32.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_IGNORE = -100


def listed():
    return [
        # -- cross entropy of the output projection
        # one token of a small model: the last position of a scored prompt; latency counts
        dict(name="ce-one-token", op="ce", tokens=1, vocab=32000, hidden=1024, dtype="bf16", ignored=0.0, train=True),
        # a fine-tuning micro-batch of a small model in fp16: odd sizes, a quarter of the labels is padding
        dict(name="ce-odd-fp16", op="ce", tokens=1021, vocab=50257, hidden=768, dtype="fp16", ignored=0.25, train=True),
        # scoring without gradients: 4096 tokens against a 32000-word vocabulary, hidden 5120
        dict(name="ce-score", op="ce", tokens=4096, vocab=32000, hidden=5120, dtype="bf16", ignored=0.0, train=False),
        # instruction tuning: 4096 tokens, the prompts' labels (60 %) are ignored
        dict(name="ce-prompts", op="ce", tokens=4096, vocab=32000, hidden=4096, dtype="bf16", ignored=0.6, train=True),
        # a short last micro-batch against a large vocabulary: few rows, 128256 words
        dict(name="ce-short-rows", op="ce", tokens=96, vocab=128256, hidden=4096, dtype="bf16", ignored=0.0, train=True),
        # pretraining: one sequence of 8192 tokens, 128256 words, hidden 4096 (the largest call)
        dict(name="ce-train-8k", op="ce", tokens=8192, vocab=128256, hidden=4096, dtype="bf16", ignored=0.0, train=True),
        # -- distillation from the teacher's top logits
        # three tokens with eight candidates each
        dict(name="kd-few", op="kd", tokens=3, vocab=32000, hidden=1024, topk=8, tau=1.0, dtype="bf16", ignored=0.0, train=True),
        # odd sizes in fp16, lists with unused places
        dict(name="kd-odd-fp16", op="kd", tokens=777, vocab=50257, hidden=1000, topk=33, tau=2.0, dtype="fp16", ignored=0.1, train=True),
        # a distillation micro-batch: one sequence of 4096 tokens, 129280 words, 64 teacher logits a token
        dict(name="kd-train-4k", op="kd", tokens=4096, vocab=129280, hidden=4096, topk=64, tau=2.0, dtype="bf16", ignored=0.0, train=True),
        # -- balance loss of a router
        # a short batch over eight experts, top 2
        dict(name="balance-short", op="bal", tokens=512, experts=8, topk=2, score="softmax", batch=1, dtype="fp32"),
        # four sequences of 1024 tokens over 64 experts, top 6, sigmoid scores, loss per sequence
        dict(name="balance-sequences", op="bal", tokens=4096, experts=64, topk=6, score="sigmoid", batch=4, dtype="fp32"),
        # a long batch over 256 experts, top 8
        dict(name="balance-long", op="bal", tokens=65536, experts=256, topk=8, score="softmax", batch=1, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ce", "ce", "kd", "bal"])
    if op == "bal":
        experts = _log_int(rng, 2, 512)
        batch = rng.choice([1, 1, 2, 3, 4])
        tokens = _log_int(rng, 1, 65536 * 256 // max(256, experts) // batch) * batch
        return dict(op="bal", tokens=tokens, experts=experts, topk=min(experts, rng.choice([1, 2, 4, 6, 8])),
                    score=rng.choice(["softmax", "sigmoid"]), batch=batch, dtype=rng.choice(["fp32", "fp32", "bf16"]))
    limit = 8192 * 128256 * 4096 if op == "ce" else 4096 * 129280 * 4096
    while True:
        tokens, vocab = _log_int(rng, 1, 8192 if op == "ce" else 4096), _log_int(rng, 1000, 131072)
        hidden = 8 * _log_int(rng, 16, 640)
        if tokens * vocab * hidden <= limit:
            break
    case = dict(op=op, tokens=tokens, vocab=vocab, hidden=hidden, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                ignored=rng.choice([0.0, 0.0, 0.25, 0.6]), train=rng.random() < 0.8)
    if op == "kd":
        case.update(topk=rng.randint(1, 128), tau=rng.choice([1.0, 2.0, 4.0]))
    return case


def _kept(case):
    """Tokens that have a label or a teacher list."""
    return case["tokens"] - int(case["tokens"] * case["ignored"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt = "cuda", _DTYPES[case["dtype"]]
    n = case["tokens"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "bal":
        E = case["experts"]
        # some experts are liked by most tokens, as in a router before it is balanced
        logits = (randn(n, E) + 0.5 * randn(E)).to(dt)
        idx = logits.float().topk(case["topk"], dim=1)[1]
        rmap = torch.zeros(n, E, dtype=torch.bool, device=dev).scatter_(1, idx, True)
        return dict(case=case, logits=logits.requires_grad_(True), routing_map=rmap, coeff=0.01, g=torch.ones((), device=dev))

    V, H = case["vocab"], case["hidden"]
    weight = (randn(V, H) * 0.02).to(dt)
    keep = torch.ones(n, dtype=torch.bool, device=dev)
    keep[torch.randperm(n, generator=gen, device=dev)[:n - _kept(case)]] = False
    # hidden states after the final norm (unit variance) that favour one word each: logits of that word between 0 and 15
    favourite = torch.randint(0, V, (n,), generator=gen, device=dev)
    rows = weight.index_select(0, favourite).float()
    strength = 15.0 * torch.rand(n, 1, generator=gen, device=dev)
    hidden = (randn(n, H) + strength * rows / rows.pow(2).sum(1, keepdim=True)).to(dt)
    # gradients of a weighted mean over the kept tokens; fp16 trains under a loss scale
    g = (0.5 + torch.rand(n, generator=gen, device=dev)) / max(1, _kept(case))
    if case["dtype"] == "fp16":
        g = g * 1024.0
    state = dict(case=case, hidden=hidden.requires_grad_(case["train"]), weight=weight.requires_grad_(case["train"]), g=g)
    if case["op"] == "ce":
        other = torch.randint(0, V, (n,), generator=gen, device=dev)
        labels = torch.where(torch.rand(n, generator=gen, device=dev) < 0.7, favourite, other)
        state["labels"] = torch.where(keep, labels, torch.full_like(labels, _IGNORE))
    else:
        K = case["topk"]
        # distinct words a token: the favourite first, then words a random odd stride apart
        step = torch.randint(0, max(1, V // K), (n, 1), generator=gen, device=dev) + 1
        idx = (favourite.unsqueeze(1) + step * torch.arange(K, device=dev)) % V
        gaps = torch.rand(n, K, generator=gen, device=dev)
        gaps[:, 0] = 0.0
        idx = torch.where(keep.unsqueeze(1), idx, torch.full_like(idx, -1))
        if K > 2:                     # nucleus-style lists: the last places of some tokens are unused
            short = (torch.rand(n, 1, generator=gen, device=dev) < 0.3) & (torch.arange(K, device=dev) >= (K + 1) // 2)
            idx = torch.where(short, torch.full_like(idx, -1), idx)
        state["teacher_logits"] = (14.0 - gaps.cumsum(1)).contiguous()
        state["teacher_indices"] = idx.contiguous()
    return state


# ---------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------
def _plain_linear(state, targets, q, const, tau, train):
    """Loss sum_k q_k (const - z_k / tau + lse) and gradients, with the whole [tokens, vocab] matrix in fp32."""
    h, w = state["hidden"].detach().float(), state["weight"].detach().float()
    z = h @ w.t()
    if tau != 1.0:
        z = z / tau
    m = z.amax(dim=1, keepdim=True)
    valid = q.sum(1) > 0
    picked = (z.gather(1, targets.clamp(min=0)) - m) * q
    e = torch.exp(z - m)
    del z
    s = e.sum(dim=1, keepdim=True)
    loss = (const + torch.log(s).squeeze(1) - picked.sum(1)) * (tau * tau)
    out = {"loss": torch.where(valid, loss, torch.zeros_like(loss))}
    if train:
        p = e.div_(s)
        p.scatter_add_(1, targets.clamp(min=0), -q)
        p.mul_((state["g"] * valid * tau).unsqueeze(1))
        out["grad_hidden"] = (p @ w).to(state["hidden"].dtype)
        out["grad_weight"] = (p.t() @ h).to(state["weight"].dtype)
    return out


def _plain_ce(state):
    t = state["labels"].unsqueeze(1)
    q = (t != _IGNORE).float()
    return _plain_linear(state, t, q, 0.0, 1.0, state["case"]["train"])


def _plain_kd(state):
    idx, tau = state["teacher_indices"], state["case"]["tau"]
    valid = idx >= 0
    a = torch.where(valid, state["teacher_logits"] / tau, torch.full_like(state["teacher_logits"], -1e30))
    a = a - a.amax(1, keepdim=True)
    e = torch.exp(a) * valid
    total = e.sum(1, keepdim=True).clamp(min=1e-30)
    q = e / total
    const = (q * (torch.where(valid, a, torch.zeros_like(a)) - torch.log(total))).sum(1)
    return _plain_linear(state, idx, q, const, tau, state["case"]["train"])


def _plain_balance(state):
    c = state["case"]
    x, rmap = state["logits"].detach().float(), state["routing_map"]
    n, E = x.shape
    B, S = c["batch"], n // c["batch"]
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
        slope = p
    else:
        sg = 1.0 / (1.0 + torch.exp(-x))
        total = sg.sum(1, keepdim=True) + 1e-20
        p = sg / total
        slope = sg * (1.0 - sg) / total
    P = p.view(S, B, E).sum(0)
    counts = rmap.view(S, B, E).sum(0)
    f = counts.float()
    scale = state["coeff"] * E / (S * S * c["topk"] * B)
    loss = (P * f).sum() * scale
    fr = f.unsqueeze(0).expand(S, B, E).reshape(n, E)
    grad = slope * (fr - (p * fr).sum(1, keepdim=True)) * (scale * state["g"])
    return {"loss": loss, "tokens_per_expert": counts.sum(0), "grad_logits": grad.to(state["logits"].dtype)}


# ---------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------
def _own_linear(state, loss):
    out = {"loss": loss.detach()}
    if state["case"]["train"]:
        gh, gw = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["g"])
        out["grad_hidden"], out["grad_weight"] = gh, gw
    return out


def _own_ce(state):
    from mindspeed_b200.ops.linear_cross_entropy import linear_cross_entropy
    return _own_linear(state, linear_cross_entropy(state["hidden"], state["weight"], state["labels"], ignore_index=_IGNORE))


def _own_kd(state):
    from mindspeed_b200.ops.linear_cross_entropy import linear_topk_distillation
    return _own_linear(state, linear_topk_distillation(state["hidden"], state["weight"], state["teacher_logits"],
                                                       state["teacher_indices"], temperature=state["case"]["tau"]))


def _own_balance(state):
    from mindspeed_b200.ops.balance_loss import router_balance_loss
    c = state["case"]
    loss, counts = router_balance_loss(state["logits"], state["routing_map"], c["topk"], state["coeff"], score_function=c["score"],
                                       batch_size=c["batch"])
    (grad,) = torch.autograd.grad(loss, (state["logits"],), state["g"])
    return {"loss": loss.detach(), "tokens_per_expert": counts, "grad_logits": grad}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"ce": _own_ce, "kd": _own_kd, "bal": _own_balance}[op](state)
    return {"ce": _plain_ce, "kd": _plain_kd, "bal": _plain_balance}[op](state)


def work(case):
    n = case["tokens"]
    size = _DTYPES[case["dtype"]].itemsize
    if case["op"] == "bal":
        E = case["experts"]
        # logits and map read, gradient written; an exponential, a normalisation and two products an entry each way
        return {"bytes": n * E * (2 * size + 1) + 8 * E, "flops": 10 * n * E}
    kept, V, H = _kept(case), case["vocab"], case["hidden"]
    K = case.get("topk", 1)
    nbytes = kept * H * size + V * H * size + n * 4 + n * K * (8 if case["op"] == "ce" else 12)
    flops = 2 * kept * V * H
    if case["train"]:
        nbytes += n * H * size + V * H * size + n * 4
        flops *= 3
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "bal":
        x = state["logits"].detach().double()
        n, E = x.shape
        B, S = case["batch"], n // case["batch"]
        seq = torch.arange(n, device=x.device) % B
        member = (seq.unsqueeze(0) == torch.arange(B, device=x.device).unsqueeze(1)).double()
        load = member @ state["routing_map"].double()
        scale = state["coeff"] * E / (float(S) * S * case["topk"] * B)
        per_row = load.index_select(0, seq)
        if case["score"] == "softmax":
            p = torch.softmax(x, dim=1)
            grad = p * (per_row - (p * per_row).sum(1, keepdim=True))
        else:
            sg = torch.sigmoid(x)
            norm = sg.sum(1, keepdim=True) + 1e-20
            p = sg / norm
            grad = sg * torch.sigmoid(-x) / norm * (per_row - (p * per_row).sum(1, keepdim=True))
        return {"loss": ((member @ p) * load).sum() * scale, "tokens_per_expert": load.sum(0).long(),
                "grad_logits": grad * scale * state["g"].double()}
    h, w, g = state["hidden"].detach().double(), state["weight"].detach().double(), state["g"].double()
    tau = case.get("tau", 1.0)
    n = h.shape[0]
    if case["op"] == "ce":
        idx = state["labels"].unsqueeze(1)
        logq = torch.where(idx == _IGNORE, -math.inf, 0.0).double()
    else:
        idx = state["teacher_indices"]
        logq = torch.where(idx < 0, -math.inf, state["teacher_logits"].double() / tau)
        logq = logq - torch.logsumexp(logq, dim=1, keepdim=True)
        logq = torch.where(idx < 0, torch.full_like(logq, -math.inf), logq)
    q = torch.exp(logq)
    loss = torch.zeros(n, dtype=torch.float64, device=h.device)
    gh, gw = torch.zeros_like(h), torch.zeros_like(w)
    for s in range(0, n, 1024):
        rows = slice(s, min(n, s + 1024))
        logp = torch.log_softmax(h[rows] @ w.t() / tau, dim=1)
        at = logp.gather(1, idx[rows].clamp(min=0))
        terms = torch.where(q[rows] > 0, q[rows] * (logq[rows] - at), torch.zeros_like(at))
        loss[rows] = tau * tau * terms.sum(1)
        if case["train"]:
            d = torch.exp(logp) * q[rows].sum(1, keepdim=True)
            d.scatter_add_(1, idx[rows].clamp(min=0), -q[rows])
            d *= tau * g[rows].unsqueeze(1)
            gh[rows] = d @ w
            gw += d.t() @ h[rows]
    out = {"loss": loss}
    if case["train"]:
        out["grad_hidden"], out["grad_weight"] = gh, gw
    return out
