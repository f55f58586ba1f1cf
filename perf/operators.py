"""Cases, plain forms and 64-bit values of the training-loss operators of ``lpmm.functional``:

* ``topk_distillation`` / ``topk_distillation_with_grad``: the divergence of a student's distribution over the whole
  vocabulary from a teacher's distribution over its K stored top logits, with its gradient;
* ``balance_loss`` / ``balance_loss_with_grad``: the load-balance loss of a router and the tokens each expert was given,
  for a whole batch or per sequence, with its gradient.

``own`` selects what ``run`` computes with: False the plain form (elementary torch operations), True the package.
"""
import math
import os
import sys

import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "low-bit-optimizers_b200")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    def distill(name, rows, vocab, k, dtype, how, temperature=1.0, padded=0, reduction="mean"):
        return dict(name=name, op="distill", rows=rows, vocab=vocab, k=k, dtype=dtype, how=how, temperature=temperature,
                    padded=padded, reduction=reduction)

    def balance(name, tokens, experts, k, dtype, how, score="softmax", sequences=0, padded=0, dropped=0):
        return dict(name=name, op="balance", tokens=tokens, experts=experts, k=k, dtype=dtype, how=how, score=score,
                    sequences=sequences, padded=padded, dropped=dropped)

    return [
        # one optimizer step's worth of tokens on the 32000-entry vocabulary of the LLaMA-shaped list, a tenth of them
        # padding (weight 0); the loss and its gradient in one call, as a loop without autograd over the loss takes them
        distill("distill_grad_32000_bf16", 16384, 32000, 64, "bf16", "with_grad", 2.0, padded=1638),
        # the odd vocabulary of the GPT-2-shaped list in fp32, through loss.backward()
        distill("distill_train_50257_fp32", 4096, 50257, 32, "fp32", "autograd"),
        # evaluation: one loss per token, no gradient
        distill("distill_eval_32000_fp16", 8192, 32000, 100, "fp16", "forward", 1.5, reduction="none"),
        # a wide vocabulary with many stored teacher logits
        distill("distill_grad_131072_bf16", 2048, 131072, 256, "bf16", "with_grad", 1.0, reduction="sum"),
        # a handful of rows: what is left of a micro-batch, where one row has to be shared by many SMs
        distill("distill_grad_few_rows", 7, 50257, 50, "bf16", "with_grad", 2.0, padded=1),
        # a single row, evaluation: the smallest call
        distill("distill_eval_one_row", 1, 32000, 16, "fp32", "forward"),
        # a layer's router in fp32 through loss.backward()
        balance("balance_train_64_fp32", 16384, 64, 2, "fp32", "autograd"),
        # many fine-grained experts, a large batch in bf16
        balance("balance_grad_256_bf16", 131072, 256, 8, "bf16", "with_grad", padded=4096),
        # the loss per sequence for a packed batch (two empty sequences, padding behind the last one), sigmoid scores
        balance("balance_sequences_128", 32768, 128, 4, "fp32", "autograd", "sigmoid", sequences=26, dropped=200),
        # odd numbers of tokens and experts; loss and counts only
        balance("balance_eval_60_odd", 65537, 60, 4, "fp32", "forward", padded=1000),
        # the router of a few tokens
        balance("balance_grad_few_tokens", 48, 8, 2, "fp16", "with_grad"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    how = rng.choice(["with_grad", "autograd", "forward"])
    if rng.random() < 0.5:
        vocab = _spread(rng, 1000, 131072)
        if rng.random() < 0.5:  # a vocabulary padded to a multiple of 64, else as it falls
            vocab = max(1024, vocab // 64 * 64)
        rows = _spread(rng, 1, min(16384, (1 << 29) // (vocab * SIZES[dtype])))
        return dict(op="distill", rows=rows, vocab=vocab, k=_spread(rng, 1, 512), dtype=dtype, how=how,
                    temperature=rng.choice([1.0, 1.0, 0.5, 2.0, round(rng.uniform(0.7, 4.0), 3)]),
                    padded=rng.choice([0, rows // 10, rows // 3]),
                    reduction=rng.choice(["mean", "sum"] if how == "autograd" else ["mean", "sum", "none"]))
    experts, sequences = _spread(rng, 2, 512), rng.choice([0, 0, _spread(rng, 1, 64)])
    if sequences and dtype == "fp16":  # sequences of one token and of thousands together leave fp16's range
        dtype = "bf16"
    if rng.random() < 0.5:
        experts = max(8, experts // 8 * 8)
    tokens = _spread(rng, 1, min(262144, (1 << 25) // experts))
    return dict(op="balance", tokens=tokens, experts=experts, k=rng.randint(1, max(1, min(8, experts // 2))), dtype=dtype, how=how,
                score=rng.choice(["softmax", "sigmoid"]), sequences=sequences,
                padded=rng.choice([0, tokens // 16]), dropped=rng.choice([0, tokens // 50]))


def _loss_scale(case):
    """The loss scale that fp16 training keeps its gradients in range with; 1 for the other types."""
    if case["dtype"] != "fp16":
        return 1.0
    if case["op"] == "distill":
        return 1024.0 * (case["rows"] if case["reduction"] == "mean" else 1)
    return 2.0 * case["tokens"]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    if case["op"] == "distill":
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        logits = torch.randn(rows, vocab, generator=g, device=dev).mul_(2.5)
        teacher = torch.randn(rows, vocab, generator=g, device=dev).add_(logits)  # a teacher that agrees in part
        top, idx = teacher.topk(min(k, vocab), dim=-1)
        del teacher
        weights = None
        if case["padded"]:
            weights = torch.ones(rows, device=dev)
            weights[torch.randperm(rows, generator=g, device=dev)[:case["padded"]]] = 0.0
        return dict(case=case, logits=logits.to(dtype).requires_grad_(case["how"] == "autograd"),
                    top=top.to(torch.bfloat16), idx=idx.to(torch.int32), weights=weights)
    n, e, k = case["tokens"], case["experts"], case["k"]
    liked = torch.randn(e, generator=g, device=dev)  # some experts are asked more often than others
    logits = torch.randn(n, e, generator=g, device=dev).add_(liked).to(dtype)
    idx = logits.float().topk(k, dim=-1).indices
    if case["dropped"]:  # assignments that a full expert refused
        idx[torch.randint(n, (case["dropped"],), generator=g, device=dev), 0] = -1
    valid = None
    if case["padded"]:
        valid = torch.ones(n, dtype=torch.bool, device=dev)
        valid[torch.randperm(n, generator=g, device=dev)[:case["padded"]]] = False
    offsets = None
    if case["sequences"]:
        s = case["sequences"]
        cuts = torch.randint(0, n + 1, (s + 1,), generator=g, device=dev).sort().values
        cuts[0] = 0
        if s >= 8:  # empty sequences, next to one another and at the end
            cuts[3] = cuts[4]
            cuts[s - 1] = cuts[s]
        offsets = cuts.to(torch.int32)
    return dict(case=case, logits=logits.requires_grad_(case["how"] == "autograd"), idx=idx, valid=valid, offsets=offsets)


def run(state):
    case = state["case"]
    if case["op"] == "distill":
        return _distill_own(case, state) if own else _distill_plain(case, state)
    return _balance_own(case, state) if own else _balance_plain(case, state)


def _distill_own(case, state):
    from lpmm import functional as F
    args = (state["logits"], state["top"], state["idx"])
    kw = dict(temperature=case["temperature"], weights=state["weights"], reduction=case["reduction"])
    if case["how"] == "with_grad":
        loss, grad = F.topk_distillation_with_grad(*args, grad_scale=_loss_scale(case), **kw)
        return {"loss": loss, "grad": grad}
    loss = F.topk_distillation(*args, **kw)
    if case["how"] == "autograd":
        return {"loss": loss.detach(), "grad": torch.autograd.grad(loss * _loss_scale(case), state["logits"])[0]}
    return {"loss": loss}


@torch.no_grad()
def _distill_plain(case, state):
    t = case["temperature"]
    x = state["logits"].float() / t
    u = state["top"].float() / t
    at = state["idx"].long()
    p = torch.exp(u - u.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    x = x - x.amax(-1, keepdim=True)
    lse = torch.exp(x).sum(-1, keepdim=True).log()
    rows = (p * (p.log() - (x.gather(-1, at) - lse))).sum(-1) * (t * t)
    w = state["weights"]
    if w is not None:
        rows = rows * w
    scale = 1.0
    if case["reduction"] == "mean":
        scale = 1.0 / (w.sum() if w is not None else float(rows.numel()))
    loss = rows if case["reduction"] == "none" else rows.sum() * scale
    if case["how"] == "forward":
        return {"loss": loss}
    q = torch.exp(x - lse).scatter_add_(-1, at, -p) * t
    if w is not None:
        q = q * w[:, None]
    return {"loss": loss, "grad": (q * (scale * _loss_scale(case))).to(state["logits"].dtype)}


def _balance_own(case, state):
    from lpmm import functional as F
    kw = dict(score=case["score"], valid=state["valid"], offsets=state["offsets"])
    if case["how"] == "with_grad":
        loss, counts, grad = F.balance_loss_with_grad(state["logits"], state["idx"],
                                                      grad_scale=_loss_scale(case) / max(case["sequences"], 1), **kw)
        return {"loss": loss, "counts": counts, "grad": grad}
    loss, counts = F.balance_loss(state["logits"], state["idx"], **kw)
    if case["how"] == "autograd":
        grad = torch.autograd.grad(loss.mean() * _loss_scale(case), state["logits"])[0]
        return {"loss": loss.detach(), "counts": counts, "grad": grad}
    return {"loss": loss, "counts": counts}


@torch.no_grad()
def _balance_plain(case, state):
    x, idx = state["logits"].float(), state["idx"]
    n, e = x.shape
    k, s = idx.shape[1], max(case["sequences"], 1)
    top = x.amax(-1, keepdim=True)
    if case["score"] == "sigmoid":
        fall = torch.exp(-x.abs())
        p = torch.exp(x.clamp(max=0.0) - top.clamp(max=0.0)) / (1.0 + fall)
    else:
        p = torch.exp(x - top)
    p = p / p.sum(-1, keepdim=True)
    # the sequence of every row; s for rows that belong to none (padding, behind the last sequence)
    seg = torch.zeros(n, dtype=torch.int64, device=x.device)
    if state["offsets"] is not None:
        rows = torch.arange(n, device=x.device)
        seg = (state["offsets"].long()[None, :] <= rows[:, None]).sum(-1) - 1
        seg = torch.where(seg < 0, s, seg)
    if state["valid"] is not None:
        seg = torch.where(state["valid"], seg, s)
    size = torch.zeros(s + 1, dtype=torch.int64, device=x.device).scatter_add_(0, seg, torch.ones_like(seg))
    cell = torch.where(idx >= 0, seg[:, None] * e + idx, s * e).reshape(-1)
    counts = torch.zeros((s + 1) * e, dtype=torch.int64, device=x.device).scatter_add_(0, cell, torch.ones_like(cell))
    counts = counts.view(s + 1, e)
    mass = torch.zeros(s + 1, e, dtype=torch.float64, device=x.device).index_add_(0, seg, p.double())
    factor = float(e) / (float(k) * size.clamp(min=1).double().square())
    factor[s] = 0.0
    loss = ((counts * mass).sum(-1) * factor)[:s].float()
    one = state["offsets"] is None
    out = {"loss": loss[0] if one else loss, "counts": counts[0] if one else counts[:s]}
    if case["how"] == "forward":
        return out
    c = counts.float()[seg]
    grad = p * (c - (c * p).sum(-1, keepdim=True)) * (factor * (_loss_scale(case) / s)).float()[seg][:, None]
    if case["score"] == "sigmoid":
        grad = grad * torch.where(x >= 0, fall, 1.0) / (1.0 + fall)
    out["grad"] = grad.to(state["logits"].dtype)
    return out


def work(case):
    b = SIZES[case["dtype"]]
    grads = case["how"] != "forward"
    if case["op"] == "distill":
        live, cells = case["rows"] - case["padded"], case["rows"] * case["vocab"]
        k = min(case["k"], case["vocab"])
        # a row of weight 0 is not read; its gradient is written
        return {"bytes": live * case["vocab"] * b + live * k * (2 + 4) + case["rows"] * 4 * (2 if case["padded"] else 1)
                + (cells * b if grads else 0), "flops": live * case["vocab"] * (8 if grads else 4)}
    live, e, s = case["tokens"] - case["padded"], case["experts"], max(case["sequences"], 1)
    return {"bytes": live * e * b + live * case["k"] * 8 + (case["tokens"] if case["padded"] else 0) + s * (e * 8 + 4)
            + (case["tokens"] * e * b if grads else 0), "flops": live * e * (10 if grads else 5)}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _distill_exact(case, state) if case["op"] == "distill" else _balance_exact(case, state)


def _distill_exact(case, state):
    """T^2 KL(teacher || student) and its derivative w T (q - p), some rows at a time."""
    x, temp = state["logits"].detach(), case["temperature"]
    rows, vocab = x.shape
    w = state["weights"].double() if state["weights"] is not None else torch.ones(rows, dtype=torch.float64, device=x.device)
    share = 1.0 / w.sum() if case["reduction"] == "mean" else torch.ones((), dtype=torch.float64, device=x.device)
    loss = torch.empty(rows, dtype=torch.float64, device=x.device)
    grad = torch.empty(rows, vocab, dtype=torch.float64, device=x.device) if case["how"] != "forward" else None
    some = max(1, (1 << 26) // vocab)
    for a in range(0, rows, some):
        b = min(rows, a + some)
        logq = torch.log_softmax(x[a:b].double() / temp, -1)
        logp = torch.log_softmax(state["top"][a:b].double() / temp, -1)
        at = state["idx"][a:b].long()
        loss[a:b] = w[a:b] * temp ** 2 * (logp.exp() * (logp - torch.gather(logq, 1, at))).sum(1)
        if grad is not None:
            dense = torch.zeros_like(logq)
            dense[torch.arange(b - a, device=x.device)[:, None], at] = logp.exp()
            grad[a:b] = (logq.exp() - dense) * (w[a:b] * temp * share * _loss_scale(case))[:, None]
    out = {"loss": loss if case["reduction"] == "none" else loss.sum() * share}
    if grad is not None:
        out["grad"] = grad
    return out


def _balance_exact(case, state):
    """sum_e f_e P_e per sequence, f_e = E count_e / (k n), P_e the mean score, and its derivative by the chain rule."""
    x, idx = state["logits"].detach().double(), state["idx"]
    n, e = x.shape
    k = idx.shape[1]
    if case["score"] == "sigmoid":
        score = torch.sigmoid(x)
        slope = score * torch.sigmoid(-x)
        total = score.sum(1, keepdim=True)
        p = score / total
    else:
        p = torch.softmax(x, 1)
    ends = [0, n] if state["offsets"] is None else state["offsets"].tolist()
    live = torch.ones(n, dtype=torch.bool, device=x.device) if state["valid"] is None else state["valid"]
    losses, counts, grad = [], [], torch.zeros_like(x)
    for a, b in zip(ends[:-1], ends[1:]):
        keep = live[a:b]
        size = int(keep.sum())
        asked = idx[a:b][keep]
        c = torch.bincount(asked[asked >= 0], minlength=e)
        counts.append(c)
        if size == 0:
            losses.append(torch.zeros((), dtype=torch.float64, device=x.device))
            continue
        f = c.double() * e / (k * size)
        losses.append((f * p[a:b][keep].mean(0)).sum())
        up = f / size / (len(ends) - 1) * _loss_scale(case)  # of the mean over the sequences by each p
        if case["score"] == "sigmoid":
            d = (up - (up * p[a:b]).sum(1, keepdim=True)) / total[a:b] * slope[a:b]
        else:
            d = p[a:b] * (up - (up * p[a:b]).sum(1, keepdim=True))
        grad[a:b] = torch.where(keep[:, None], d, torch.zeros_like(d))
    one = state["offsets"] is None
    out = {"loss": losses[0] if one else torch.stack(losses), "counts": None}
    if case["how"] != "forward":
        out["grad"] = grad
    return out
