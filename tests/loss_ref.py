"""Plain 64-bit restatements of the training losses, and the error bounds that the tests hold the kernels to."""
import torch

U32 = 2.0 ** -24  # half a step of fp32, relative


def distill_ref(x, t, idx, temp, w=None):
    """Per row (loss, G-free parts of the gradient): ``(loss [n], q [n, v], p [n, v])`` in fp64; gradient = w T (q - p).
    Rows of weight 0 or without entries give zeros."""
    x, t, idx = x.double().cpu(), t.double().cpu(), idx.long().cpu()
    n, v = x.shape
    w = torch.ones(n, dtype=torch.float64) if w is None else w.double().cpu()
    loss, q, p = torch.zeros(n, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64)
    for r in range(n):
        there = (idx[r] >= 0) & (t[r] != -float("inf"))
        if w[r] == 0 or not there.any():
            continue
        pr = torch.softmax(t[r][there] / temp, 0)
        logq = torch.log_softmax(x[r] / temp, 0)
        at = idx[r][there]
        term = torch.where(pr > 0, pr * (pr.log() - logq[at]), torch.zeros_like(pr))
        loss[r] = w[r] * temp ** 2 * term.sum()
        q[r] = logq.exp()
        p[r].index_add_(0, at, pr)
    return loss, q, p


def distill_row_bound(vocab, temp, w=1.0, spread=60.0):
    """Absolute error of one row's loss.  log s: an exponential is off by 2^-22 and by 3 roundings of its argument (at most
    `spread` in size where it matters), a partial sum has at most vocab / 128 + 64 additions; the K terms are off by a few
    roundings of numbers up to `spread`."""
    return temp * temp * abs(w) * U32 * (vocab / 128 + 64 + 4 + 6 * spread)


def distill_grad_bound(ref, q, p, scale, vocab, dtype, spread=60.0):
    """Elementwise: q and p are each off by the relative error of an exponential and of a sum (as above), the difference is
    rounded once to fp32 and once to the type; below the type's smallest normal number half a step is absolute.  An
    exponential below 2^-126, fp32's smallest normal number, is 0: with sums of at least 1 that is less than 2^-126 of q and
    of p, times w T (at most 1024 here): 2 * 2^-126 * 2^10 = 2^-115."""
    step = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # the step of the denormal range
    return abs(scale) * ((q + p) * U32 * (vocab / 128 + 64 + 16 + 8 * spread) + 2.0 ** -115) + step * 1.001 * ref.abs() + tiny


def balance_ref(x, idx, score="softmax", valid=None, offsets=None):
    """``(loss [s], counts [s, e], grad of sum(loss) [n, e], size [n, e] of the gradient's two terms)`` in fp64."""
    x, idx = x.double().cpu(), idx.long().cpu()
    n, e = x.shape
    k = idx.shape[1]
    live = torch.ones(n, dtype=torch.bool) if valid is None else valid.cpu()
    ends = [0, n] if offsets is None else offsets.cpu().tolist()
    losses, counts = [], []
    grad, size = torch.zeros(n, e, dtype=torch.float64), torch.zeros(n, e, dtype=torch.float64)
    for a, b in zip(ends[:-1], ends[1:]):
        rows = torch.arange(a, b)[live[a:b]]
        c = torch.bincount(idx[rows][idx[rows] >= 0], minlength=e)
        counts.append(c)
        m = len(rows)
        if m == 0:
            losses.append(torch.zeros((), dtype=torch.float64))
            continue
        if score == "softmax":
            p, slope = torch.softmax(x[rows], 1), 1.0
        else:
            p, slope = torch.softmax(torch.nn.functional.logsigmoid(x[rows]), 1), torch.sigmoid(-x[rows])
        f = e * c.double() / (k * m)
        losses.append((f * p.mean(0)).sum())
        dot = (f * p).sum(1, keepdim=True)
        grad[rows] = p * (f - dot) * slope / m
        size[rows] = p * (f + dot) * slope / m
    return torch.stack(losses), torch.stack(counts), grad, size


def balance_loss_bound(loss, tokens, experts, spread=40.0):
    """A score is off by an exponential's error (2^-22, 3 roundings of an argument up to `spread`) and its sum's; the sums over
    tokens have at most tokens / 64 + 512 additions of numbers of one sign."""
    return loss.abs() * U32 * (16 + 6 * spread + experts / 32 + 32 + tokens / 64 + 512) + 1e-30


def balance_grad_bound(ref, size, scale, experts, dtype, spread=40.0):
    step = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return abs(scale) * size * U32 * (32 + 12 * spread + experts) + step * 1.001 * ref.abs() + tiny
