"""The training losses on a B200 where values, lengths or calls leave the ordinary: against the 64-bit restatements of
``loss_ref.py`` with their bounds, and against themselves."""
import threading

import pytest
import torch

from gpu_helpers import device
from loss_ref import U32, balance_loss_bound
from test_gpu_losses import (DT, F, INF, REGIMES, balance_inputs, check_balance, check_distill, check_distill_copies, close, distill_inputs,
                             same_bits)

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------------------------------------
# columns at a mask's finite value
# ----------------------------------------------------------------------------------------------
def masked_inputs(vocab, k, dtype, fill):
    """Twelve rows with columns at `fill`; the entries lie where the student has ordinary logits."""
    x, t, idx = distill_inputs(12, vocab, k, dtype, seed=21)
    g = torch.Generator().manual_seed(22)
    low = torch.finfo(DT[dtype]).min if fill == "lowest" else fill
    live = torch.ones(12, vocab, dtype=torch.bool)
    live[0, :vocab * 3 // 5] = False            # a thread's first columns
    live[1, :-9] = False                        # all but the last ones
    live[2, 9:] = False                         # all but the first ones
    live[3, ::2] = False                        # every other one
    live[4, vocab // 4:vocab // 2 + 64] = False  # whole parts of a cluster
    live[6] = torch.rand(vocab, generator=g) < 0.1
    live[6, 0] = True
    live[8, :-1] = False                        # all but one
    live[9] = live[1]
    live[11, vocab // 2:] = False
    for r in range(12):
        at = torch.arange(vocab)[live[r]]
        idx[r] = at[torch.randint(len(at), (k,), generator=g)]  # some of them several times
    x[~live.to(device())] = low
    x[5] = low                                  # nothing but masked columns: uniform
    x[9, :vocab // 2] = low / 2                 # two mask values
    x[10, idx[10, 0]] = abs(low)                # the largest one far above the others: certain
    t[10, 1:] = -INF
    w = torch.ones(12, device=device())
    w[3], w[11] = 0.5, -2.0
    return x, t, idx, w


@pytest.mark.parametrize("fill", [-1e9, -1e10, -1e12, -1e20, -1e30, "lowest"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("copies, vocab", REGIMES)
def test_distillation_finite_masks(copies, vocab, dtype, fill):
    x, t, idx, w = masked_inputs(vocab, 8, dtype, fill)
    for temp in (0.25, 0.5, 1.0, 2.0, 5.0, 8.0, 20.0, 100.0):
        check_distill_copies(copies, x, t, idx, temp, w, "none")


@pytest.mark.parametrize("fill", [-1e10, -1e30])
@pytest.mark.parametrize("copies, vocab", REGIMES)
def test_distillation_finite_masks_many_entries(copies, vocab, fill):
    x, t, idx, w = masked_inputs(vocab, 300, "bf16", fill)
    for temp in (1.0, 5.0):
        check_distill_copies(copies, x, t, idx, temp, w, "sum")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("copies, vocab", REGIMES)
def test_distillation_rows_of_minus_infinity_at_high_temperatures(copies, vocab, dtype):
    """No distribution, whatever the temperature: NaN, and the other rows as they are."""
    x, t, idx = distill_inputs(12, vocab, 4, dtype, seed=23)
    x[7] = -INF
    for temp in (1.0, 8.0, 1024.0):
        check_distill_copies(copies, x, t, idx, temp, torch.ones(12, device=device()), "none")


# ----------------------------------------------------------------------------------------------
# what the caller does with the counts
# ----------------------------------------------------------------------------------------------
# one CTA, a cluster, several launches whose last CTA adds up, more sequences than that
@pytest.mark.parametrize("tokens, experts, sequences", [(48, 8, 0), (48, 8, 3), (3000, 64, 0), (3000, 64, 5), (30000, 64, 0),
                                                        (30000, 64, 7), (30000, 64, 100)])
def test_balance_gradient_does_not_read_the_returned_counts(tokens, experts, sequences):
    x, idx = balance_inputs(tokens, experts, 2, "fp32", seed=24)
    offsets = torch.linspace(0, tokens, sequences + 1, device=device()).long() if sequences else None
    ends = [0, tokens] if offsets is None else offsets.tolist()
    want_counts = torch.stack([torch.bincount(idx[a:b].reshape(-1), minlength=experts) for a, b in zip(ends[:-1], ends[1:])])
    assert torch.equal(F().balance_loss_with_grad(x, idx, offsets=offsets)[1].view(-1, experts), want_counts)
    x.requires_grad_()
    grads, losses = [], []
    for change in (lambda c: None, lambda c: c.data.mul_(2),  # as a collective over ranks leaves them, past autograd's record
                   lambda c: c.zero_()):
        loss, counts = F().balance_loss(x, idx, offsets=offsets)
        assert torch.equal(counts.view(-1, experts), want_counts)
        losses.append(loss.detach())
        change(counts)
        grads.append(torch.autograd.grad(loss.sum(), x)[0])
    assert grads[0].any()
    for same in (grads, losses):
        assert same_bits(same[0], same[1]) and same_bits(same[0], same[2])


# ----------------------------------------------------------------------------------------------
# many tokens: what is added in fp32 has a bound of its own
# ----------------------------------------------------------------------------------------------
def many_tokens(row, tokens, k=1):
    """`tokens` times the same row of logits (one in memory), and experts drawn at random."""
    g = torch.Generator(device=device()).manual_seed(26)
    idx = torch.randint(row.numel(), (tokens, k), device=device(), generator=g, dtype=torch.int32)
    return row.to(device())[None].expand(tokens, -1), idx


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [1 << 23, 1 << 26])
def test_balance_loss_of_many_even_tokens(tokens, score):
    """All scores 1 / 248, loss exactly 1.  Exponentials of 0, sums of 1 and (for sigmoid, all 0.5) of 0.5 are exact; a reciprocal
    is off by 2 roundings, a product by one, at most 512 additions of a run by one each, 5 across the lanes, the whole numbers by less
    than one, the result by one; for sigmoid 3 more for 0.5."""
    x, idx = many_tokens(torch.zeros(248, dtype=torch.bfloat16), tokens)
    loss, counts = F().balance_loss(x, idx, score)
    close(loss, torch.ones((), dtype=torch.float64), (512 + 2 + 1 + 5 + 1 + 1 + 3) * U32)
    assert torch.equal(counts, torch.bincount(idx[:, 0], minlength=248))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens, cuts", [(1 << 26, None), (9000001, [5, 4000000, 4000003, 9000000])])
def test_balance_loss_of_many_tokens(tokens, cuts, score):
    row = torch.randn(248, generator=torch.Generator().manual_seed(27)).bfloat16()
    x, idx = many_tokens(row, tokens, 2)
    offsets = None if cuts is None else torch.tensor(cuts, device=device())
    loss, counts = F().balance_loss(x, idx, score, offsets=offsets)
    x64 = row.double()
    p = torch.softmax(x64 if score == "softmax" else torch.nn.functional.logsigmoid(x64), 0)
    c = counts.double().cpu().view(-1, 248)
    ref = (248 * c / c.sum(1, keepdim=True) * p).sum(1).view(loss.shape)
    close(loss, ref, balance_loss_bound(ref, 0, 248))  # its constant part has the 512 additions of a run


# ----------------------------------------------------------------------------------------------
# weights that cancel
# ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [4, 40, 160, 256, 258])
@pytest.mark.parametrize("vocab", [700, 10000, 40000])
def test_distillation_mean_over_weights_that_cancel(rows, vocab):
    """Their sum is 1.5 and exact in double, in any order; in fp32 it would be 0: loss and gradient have the same mean."""
    x, t, idx = distill_inputs(rows, vocab, 5, "bf16", seed=28)
    w = torch.tensor([3.0, -3.0]).repeat(rows // 2)
    w[:4] = torch.tensor([2.0 ** 25, -2.0 ** 25, 1.0, 0.5])
    assert w.double().sum() == 1.5
    check_distill(x, t, idx, 2.0, w.to(device()), "mean")


# ----------------------------------------------------------------------------------------------
# two host threads at a time
# ----------------------------------------------------------------------------------------------
# calls that take one kernel with different amounts of shared memory: short rows, a ring of small chunks, one of large chunks,
# clusters
@pytest.mark.parametrize("sizes", [((300, 1000, 8), (300, 4000, 8)), ((200, 12000, 8), (200, 20000, 250)),
                                   ((160, 40000, 8), (160, 60000, 1000)), ((160, 131072, 8), (160, 100000, 1000))])
def test_distillation_from_two_threads(sizes):
    inputs = [distill_inputs(*s, "bf16", seed=25 + i) for i, s in enumerate(sizes)]
    want = [F().topk_distillation_with_grad(*v, reduction="none") for v in inputs]
    torch.cuda.synchronize()
    errors = []

    def work(v, ref):
        try:
            torch.cuda.set_device(device())
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(2000):
                    got = F().topk_distillation_with_grad(*v, reduction="none")
            stream.synchronize()
            assert all(same_bits(a, b) for a, b in zip(ref, got))
        except Exception as e:  # noqa: BLE001 - handed to the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(v, w)) for v, w in zip(inputs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


# ----------------------------------------------------------------------------------------------
# captured passes of every size
# ----------------------------------------------------------------------------------------------
def captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [v.clone() for v in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    return graph, want, got


def check_replays(step, x, other):
    """A replay has the bits of the ordinary call, twice, and those of the other inputs once they lie in the same memory."""
    graph, want, got = captured(step)
    for _ in range(2):
        for v in got:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(want, got))
    with torch.no_grad():
        x.copy_(other)
    want = [v.clone() for v in step()]
    graph.replay()
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(want, got))


# rows of their own, a ring of each size, clusters, few rows; the sum of the weights inside the kernel and before it
@pytest.mark.parametrize("rows, vocab", [(300, 700), (200, 12000), (300, 12000), (300, 40000), (160, 131072), (300, 131072), (7, 50257)])
def test_distillation_captured(rows, vocab):
    x, t, idx = distill_inputs(rows, vocab, 9, "bf16", seed=29)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(30)).to(device())
    check_replays(lambda: F().topk_distillation_with_grad(x, t, idx, 2.0, w), x, x * 0.5)
    x.requires_grad_()

    def train():
        loss = F().topk_distillation(x, t, idx, 2.0, w)
        return loss.detach(), torch.autograd.grad(loss, x)[0]
    check_replays(train, x, x.detach() * 0.5)


@pytest.mark.parametrize("tokens, experts, sequences", [(48, 8, 0), (3000, 64, 5), (30000, 64, 0), (30000, 64, 100)])
def test_balance_captured(tokens, experts, sequences):
    x, idx = balance_inputs(tokens, experts, 2, "bf16", seed=31)
    offsets = torch.linspace(0, tokens, sequences + 1, device=device()).long() if sequences else None
    check_replays(lambda: F().balance_loss_with_grad(x, idx, offsets=offsets), x, x * 0.5)
    x.requires_grad_()

    def train():
        loss, counts = F().balance_loss(x, idx, offsets=offsets)
        return loss.detach(), counts, torch.autograd.grad(loss.sum(), x)[0]
    check_replays(train, x, x.detach() * 0.5)


# ----------------------------------------------------------------------------------------------
# many experts per token
# ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("tokens, experts, k", [(70, 2, 5), (100, 33, 33), (45, 700, 500), (1000, 64, 1024), (3000, 100, 31)])
def test_balance_many_chosen(tokens, experts, k):
    g = torch.Generator().manual_seed(32)
    x = torch.randn(tokens, experts, generator=g).to(device())
    idx = torch.randint(-1, experts, (tokens, k), generator=g).int().to(device())
    valid = (torch.rand(tokens, generator=g) < 0.8).to(device())
    check_balance(x, idx, "softmax", valid, torch.tensor([0, tokens // 3, tokens], device=device()), grad_scale=float(tokens))
    check_balance(x, idx, "sigmoid", None, None, grad_scale=float(tokens))
