"""The training losses on a B200 against 64-bit restatements (``loss_ref.py``), whose bounds count roundings."""
import math

import pytest
import torch

from gpu_helpers import device
from loss_ref import (U32, balance_grad_bound, balance_loss_bound, balance_ref, distill_grad_bound, distill_ref,
                      distill_row_bound)

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
INF = float("inf")


def F():
    from lpmm import functional
    return functional


def close(got, ref, bound, what=""):
    got = got.double().cpu()
    nan = torch.isnan(ref)
    assert torch.equal(nan, torch.isnan(got)), f"{what}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), f"{what}: infinities"
    fine = ~nan & ~inf
    off = (got - ref).abs()
    worst = (off - bound)[fine]
    assert worst.numel() == 0 or bool((worst <= 0).all()), f"{what}: off by {off[fine].max():.3g}, {int((worst > 0).sum())} beyond the bound"


def same_bits(a, b):
    return a.dtype == b.dtype and torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


# ----------------------------------------------------------------------------------------------
# distillation
# ----------------------------------------------------------------------------------------------
def distill_inputs(rows, vocab, k, dtype, seed=0, idx_dtype=torch.int64, tdtype=torch.float32, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * scale).to(DT[dtype]).to(device())
    t = (torch.randn(rows, k, generator=g) * 2).to(tdtype).to(device())
    if k <= vocab:
        idx = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]) if rows else torch.zeros(0, k)
    else:  # more entries than columns: some columns several times
        idx = torch.randint(vocab, (rows, k), generator=g)
    return x, t, idx.to(idx_dtype).to(device())


def check_distill(x, t, idx, temp=1.0, w=None, reduction="sum", scale=1.0, grad_scale=1.0):
    """All three forms against the restatement, and against one another."""
    vocab, dtype = x.shape[-1], x.dtype
    loss, q, p = distill_ref(x.reshape(-1, vocab), t.reshape(-1, t.shape[-1]), idx.reshape(-1, t.shape[-1]), temp,
                             None if w is None else w.reshape(-1))
    n = loss.numel()
    wd = torch.ones(n, dtype=torch.float64) if w is None else w.reshape(-1).double().cpu()
    norm = 1.0
    if reduction == "mean":
        norm = 0.0 if n == 0 or wd.sum() == 0 else float(1.0 / wd.sum())
    rb = torch.tensor([distill_row_bound(vocab, temp, float(a)) for a in wd], dtype=torch.float64)
    ref = loss.view(x.shape[:-1]) if reduction == "none" else loss.sum() * norm
    # a sum of rows adds a rounding to fp32 for every row's loss and one at the end
    lb = rb.view(x.shape[:-1]) if reduction == "none" else rb.sum() * abs(norm) + 4 * U32 * loss.abs().sum() * abs(norm)
    coef = (wd * temp * norm).view(-1, 1)
    gref = (coef * (q - p)).view(x.shape)
    gb = distill_grad_bound(gref * grad_scale, (coef.abs() * q).view(x.shape), (coef.abs() * p).view(x.shape), grad_scale,
                            vocab, dtype)
    f = F()
    kw = dict(temperature=temp, weights=w, reduction=reduction)
    with torch.no_grad():
        only = f.topk_distillation(x, t, idx, **kw)
    close(only, ref, lb, "loss")
    both, grad = f.topk_distillation_with_grad(x, t, idx, grad_scale=grad_scale, **kw)
    assert grad.dtype == dtype and grad.shape == x.shape and both.dtype == torch.float32
    close(both, ref, lb, "loss of with_grad")
    close(grad, gref * grad_scale, gb, "grad of with_grad")
    leaf = x.detach().clone() if x.is_contiguous() else x.detach()
    leaf.requires_grad_()
    out = f.topk_distillation(leaf, t, idx, **kw)
    (auto,) = torch.autograd.grad(out.sum() * grad_scale, leaf)
    close(out.detach(), ref, lb, "loss through autograd")
    close(auto, gref * grad_scale, gb, "grad through autograd")
    return both, grad


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows, vocab, k", [
    (1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 8, 1), (3, 9, 4), (2, 31, 5), (7, 128, 16), (40, 1000, 64), (3, 4097, 33),
    (2, 32000, 64), (3, 50257, 100), (1, 131075, 1024), (300, 515, 9), (1, 3, 7), (700, 260, 300), (5, 2048, 256), (9, 2049, 257),
    (33, 8192, 40), (6, 8193, 1000), (3, 1024, 31), (310, 8200, 12), (640, 16391, 65), (200, 40003, 1024), (160, 70001, 33),
])
def test_distillation_sizes(dtype, rows, vocab, k):
    x, t, idx = distill_inputs(rows, vocab, k, dtype, seed=rows + vocab)
    check_distill(x, t, idx, temp=1.0, reduction="sum")


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("temp", [0.5, 2.0, 3.7])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_distillation_temperature_weights_reduction(dtype, temp, reduction):
    x, t, idx = distill_inputs(37, 777, 20, dtype, seed=3, idx_dtype=torch.int32, tdtype=torch.bfloat16)
    w = torch.rand(37, generator=torch.Generator().manual_seed(1)).to(device())
    w[::5] = 0
    check_distill(x, t, idx, temp, w, reduction, grad_scale=1.0 if reduction == "none" else 0.25)
    check_distill(x, t, idx, temp, None, reduction)


@pytest.mark.parametrize("idx_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, vocab, k", [(9, 500, 33), (9, 500, 130), (9, 500, 260), (7, 9000, 70), (150, 9000, 70)])
def test_distillation_types_of_the_entries(rows, vocab, k, tdtype, idx_dtype):
    x, t, idx = distill_inputs(rows, vocab, k, "bf16", seed=17, idx_dtype=idx_dtype, tdtype=tdtype)
    idx[:, 1::5] = -1
    t[:, 2::7] = -INF
    check_distill(x, t, idx, 1.5, None, "sum")


@pytest.mark.parametrize("rows", [255, 256, 257, 600])
@pytest.mark.parametrize("vocab", [700, 10000])
def test_distillation_mean_over_weights(rows, vocab):
    x, t, idx = distill_inputs(rows, vocab, 5, "fp32", seed=18)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(2)).to(device())
    w[::7] = 0
    check_distill(x, t, idx, 2.0, w, "mean")
    check_distill(x, t, idx, 2.0, None, "mean")


# (copies of the twelve rows, columns): each kernel, the vocabulary within one CTA's columns and shared by a cluster
REGIMES = [(1, 1001), (150, 1001), (1, 4095), (1, 20011), (13, 9003), (26, 30001), (13, 70003)]


@pytest.mark.parametrize("copies, vocab", REGIMES)
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("k", [8, 90, 300])
def test_distillation_masks_and_absent_entries(copies, vocab, dtype, k):
    x, t, idx = distill_inputs(12, vocab, k, dtype, seed=5)
    low = torch.finfo(DT[dtype]).min
    idx[0, 3:] = -1          # a shorter list
    idx[1] = -1              # none at all
    t[2] = -INF              # none at all
    t[3, 1:] = -INF          # one
    idx[4, 1] = idx[4, 0]    # the same index twice
    idx[5] = idx[5, 0]       # many times
    idx[6] = torch.arange(k, device=device())
    x[6, k + vocab // 2:] = -INF  # columns that the student may not use ...
    x[7, :] = low
    x[7, 17] = 0.0
    idx[7, 0] = 17
    t[7, 1:] = -INF
    x[8, :] = low            # all of the lowest value: uniform
    x[9, idx[9, 0]] = -INF   # ... an entry among them: infinite loss
    x[10], idx[10, 0] = float("nan"), 5
    w = torch.ones(12, device=device())
    w[10] = 0                # a padded row may hold anything
    w[11] = -2.0
    for temp, reduction in ((1.0, "none"), (1.0, "sum"), (2.0, "none")):
        check_distill_copies(copies, x, t, idx, temp, w, reduction)


def check_distill_copies(copies, x, t, idx, temp, w, reduction):
    """Twelve different rows, so many times that another kernel takes them.  Every copy keeps the bounds; copies that lie alike to
    the 16-byte boundaries, by which a row is cut into vectors and so its sums into parts, have the same bits."""
    if copies == 1:
        check_distill(x, t, idx, temp, w, reduction)
        return
    f, n = F(), x.shape[0]
    loss, q, p = distill_ref(x, t, idx, temp, w)
    rb = torch.tensor([distill_row_bound(x.shape[1], temp, float(a)) for a in w], dtype=torch.float64)
    coef = (w.double().cpu() * temp).view(-1, 1)
    gref = coef * (q - p)
    gb = distill_grad_bound(gref, coef.abs() * q, coef.abs() * p, 1.0, x.shape[1], x.dtype)
    many = [v.repeat(copies, *[1] * (v.dim() - 1)) for v in (x, t, idx, w)]
    got, grad = f.topk_distillation_with_grad(*many[:3], temp, many[3], "none")
    leaf = many[0].requires_grad_()
    out = f.topk_distillation(leaf, *many[1:3], temp, many[3], reduction)
    (auto,) = torch.autograd.grad(out.sum(), leaf)
    rows = out if reduction == "none" else f.topk_distillation(leaf.detach(), *many[1:3], temp, many[3], "none")
    for v, ref, bound in ((got, loss, rb), (rows, loss, rb), (grad, gref, gb), (auto, gref, gb)):
        v = v.detach().view(copies, n, -1)
        alike = 16 // math.gcd(16, n * x.shape[1] * x.element_size())
        assert all(same_bits(v[0], v[c]) for c in range(alike, copies, alike)), "copies of a row differ"
        for c in range(min(alike, copies)):
            close(v[c], ref.view(n, -1), bound.view(n, -1))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_distillation_rows_of_nan_and_infinity_keep_to_themselves(dtype):
    x, t, idx = distill_inputs(6, 300, 4, dtype, seed=6)
    x[1, 7] = float("nan")
    x[2, 9] = INF
    x[3] = -INF
    t[4, 2] = float("nan")
    loss, grad = F().topk_distillation_with_grad(x, t, idx, reduction="none")
    for r in range(6):
        if r in (0, 5):
            assert loss[r].isfinite() and grad[r].isfinite().all()
        else:
            assert loss[r].isnan() and grad[r].isnan().all(), r
    check_distill(x[[0, 5]], t[[0, 5]], idx[[0, 5]], 1.0, None, "none")


@pytest.mark.parametrize("idx_dtype", [torch.int32, torch.int64])
def test_distillation_index_out_of_range_is_nan_and_not_followed(idx_dtype):
    x, t, idx = distill_inputs(5, 100, 3, "fp32", seed=7, idx_dtype=idx_dtype)
    idx[1, 2] = 100
    idx[3, 0] = torch.iinfo(idx_dtype).max
    idx[4, 0] = torch.iinfo(idx_dtype).min  # negative: absent
    loss, grad = F().topk_distillation_with_grad(x, t, idx, reduction="none")
    leaf = x.clone().requires_grad_()
    out = F().topk_distillation(leaf, t, idx, reduction="none")
    (auto,) = torch.autograd.grad(out.sum(), leaf)
    for r in range(5):
        bad = r in (1, 3)
        assert bool(loss[r].isnan()) == bool(out[r].isnan()) == bad
        for g in (grad, auto):
            assert bool(g[r].isnan().all()) == bad and bool(g[r].isnan().any()) == bad
    keep = [0, 2, 4]
    check_distill(x[keep], t[keep], idx[keep], 1.0, None, "none")


@pytest.mark.parametrize("make", [
    lambda b: b[:, :-1], lambda b: b[:, 1:], lambda b: b[..., :-3], lambda b: b[..., 1:], lambda b: b.transpose(0, 1),
    lambda b: b[0, 0].expand(4, 5, b.shape[-1]), lambda b: b.transpose(1, 2),
    lambda b: b[:, ::2, 3:], lambda b: b[None],
], ids=["first tokens", "later tokens", "padded columns", "off the boundary", "transposed rows", "expanded", "columns not dense",
        "every other", "four axes"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_distillation_strides(make, dtype):
    g = torch.Generator().manual_seed(8)
    x = make((torch.randn(4, 5, 203, generator=g) * 2).to(DT[dtype]).to(device()))
    lead, v = x.shape[:-1], x.shape[-1]
    n = lead.numel()
    t = torch.randn(n, 6, generator=g).view(*lead, 6).to(device())
    idx = torch.stack([torch.randperm(v, generator=g)[:min(6, v)] for _ in range(n)])
    if v < 6:
        idx = torch.randint(v, (n, 6), generator=g)
    idx = idx.view(*lead, 6).to(device())
    check_distill(x, t, idx, 1.5, None, "sum")
    check_distill(x, t.transpose(-1, -2).contiguous().transpose(-1, -2), idx.expand(idx.shape), 1.5, None, "mean")


def test_distillation_of_nothing():
    f = F()
    x = torch.randn(0, 10, device=device(), requires_grad=True)
    t, idx = torch.zeros(0, 2, device=device()), torch.zeros(0, 2, dtype=torch.int64, device=device())
    for reduction in ("sum", "mean"):
        loss = f.topk_distillation(x, t, idx, reduction=reduction)
        assert loss.item() == 0.0
        assert torch.autograd.grad(loss, x)[0].shape == (0, 10)
    assert f.topk_distillation(x, t, idx, reduction="none").shape == (0,)
    loss, grad = f.topk_distillation_with_grad(x, t, idx)
    assert loss.item() == 0.0 and grad.shape == (0, 10)
    x, t, idx = distill_inputs(4, 50, 3, "bf16")
    loss, grad = f.topk_distillation_with_grad(x, t, idx, weights=torch.zeros(4, device=device()))  # mean over no weight
    assert loss.item() == 0.0 and not grad.any()
    one = f.topk_distillation(x[0], t[0], idx[0], reduction="none")
    assert one.shape == ()
    close(one, distill_ref(x[:1], t[:1], idx[:1], 1.0)[0][0], distill_row_bound(50, 1.0))


def test_distillation_gradient_against_differences():
    """Along d of +-1, third derivative per row at most 0.77 / T^3 T^2 (third central moment of a variable in [-1, 1])."""
    for temp in (1.0, 2.0):
        x, t, idx = distill_inputs(5, 33, 4, "fp32", seed=9)
        _, grad = F().topk_distillation_with_grad(x, t, idx, temp, reduction="sum")
        d = torch.where(grad >= 0, 1.0, -1.0)
        h = 2.0 ** -5
        with torch.no_grad():
            up, down = (F().topk_distillation(x + s * h * d, t, idx, temp, reduction="none").double().sum().item() for s in (1, -1))
        tol = 5 * (h * h / 6 * 0.77 / temp + 1.5 * distill_row_bound(33, temp) / h)
        assert abs((up - down) / (2 * h) - (grad.double() * d).sum().item()) < tol


def test_distillation_is_the_same_each_time_and_in_every_form():
    x, t, idx = distill_inputs(50, 5003, 40, "bf16", seed=10)
    w = torch.rand(50, device=device())
    runs = [F().topk_distillation_with_grad(x, t, idx, 2.0, w, "mean") for _ in range(3)]
    assert all(same_bits(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@pytest.mark.parametrize("rows, vocab", [(67200, 32000), (2150000, 1000)])  # 2.15e9 elements
def test_distillation_rows_beyond_32_bit_offsets(rows, vocab):
    x = torch.empty(rows, vocab, dtype=torch.bfloat16, device=device())
    for a in range(0, rows, rows // 8):
        x[a:a + rows // 8].normal_(generator=torch.Generator(device=device()).manual_seed(a))
    g = torch.Generator(device=device()).manual_seed(1)
    t = torch.randn(rows, 8, device=device(), generator=g)
    idx = torch.randint(vocab, (rows, 8), device=device(), generator=g)
    loss, grad = F().topk_distillation_with_grad(x, t, idx, 1.0, reduction="none")
    edge = 2 ** 31 // vocab
    for r in (0, rows // 2, edge - 1, edge, rows - 1):
        ref, q, p = distill_ref(x[r:r + 1], t[r:r + 1], idx[r:r + 1], 1.0)
        close(loss[r], ref[0], distill_row_bound(vocab, 1.0))
        close(grad[r:r + 1], q - p, distill_grad_bound(q - p, q, p, 1.0, vocab, torch.bfloat16))


@pytest.mark.parametrize("temp", [2.0 ** -10, 0.01, 100.0, 1024.0])
@pytest.mark.parametrize("rows, vocab", [(5, 700), (200, 700), (5, 20000), (160, 20000)])
def test_distillation_far_temperatures(rows, vocab, temp):
    """Arguments of exponentials up to 25 / T in size: that is the spread of the bounds."""
    x, t, idx = distill_inputs(rows, vocab, 6, "fp32", seed=14)
    loss, q, p = distill_ref(x, t, idx, temp)
    got, grad = F().topk_distillation_with_grad(x, t, idx, temp, reduction="none")
    spread = 60.0 + 25.0 / temp
    close(got, loss, distill_row_bound(vocab, temp, spread=spread))
    close(grad, temp * (q - p), distill_grad_bound(temp * (q - p), q, p, temp, vocab, torch.float32, spread=spread))


def test_distillation_second_backward_and_changed_inputs():
    x, t, idx = distill_inputs(7, 900, 5, "fp32", seed=15)
    leaf = x.clone().requires_grad_()
    loss = F().topk_distillation(leaf, t, idx, 2.0, reduction="none")
    up = torch.linspace(-1, 2, 7, device=device())
    (a,) = torch.autograd.grad(loss, leaf, up, retain_graph=True)
    (b,) = torch.autograd.grad(loss, leaf, up)
    assert same_bits(a, b)
    _, q, p = distill_ref(x, t, idx, 2.0)
    coef = (2.0 * up).double().cpu().view(-1, 1)
    close(a, coef * (q - p), distill_grad_bound(coef * (q - p), coef.abs() * q, coef.abs() * p, 1.0, 900, torch.float32))
    loss = F().topk_distillation(leaf, t, idx)
    t.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_distillation_weights_of_other_types():
    x, t, idx = distill_inputs(9, 300, 4, "bf16", seed=16)
    mask = torch.arange(9, device=device()) % 3 != 0
    want = F().topk_distillation_with_grad(x, t, idx, weights=mask.float())
    for w in (mask, mask.int(), mask.double(), mask.bfloat16(), torch.stack([mask, mask], 1)[:, 0]):
        got = F().topk_distillation_with_grad(x, t, idx, weights=w)
        assert all(same_bits(a, b) for a, b in zip(want, got))


def test_distillation_on_another_stream_and_in_graphs():
    f = F()
    x, t, idx = distill_inputs(9, 2050, 7, "bf16", seed=11)
    w = torch.rand(9, device=device())
    want = f.topk_distillation_with_grad(x, t, idx, 1.0, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = f.topk_distillation_with_grad(x, t, idx, 1.0, w)
    side.synchronize()
    assert all(same_bits(a, b) for a, b in zip(want, got))
    # two graphs over different inputs, replayed in turn and at the same time
    x2 = x * 0.5
    want2 = f.topk_distillation_with_grad(x2, t, idx, 1.0, w)
    graphs, outs = [], []
    for inp in (x, x2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(f.topk_distillation_with_grad(inp, t, idx, 1.0, w))
        graphs.append(gr)
    for _ in range(3):
        for o in outs:
            o[1].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert all(same_bits(a, b) for a, b in zip(want, outs[0]))
        assert all(same_bits(a, b) for a, b in zip(want2, outs[1]))
    x.copy_(x2)  # a replay reads what the inputs hold now
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(want2, outs[0]))


def test_distillation_training_pass_in_a_graph():
    f = F()
    x, t, idx = distill_inputs(6, 1111, 5, "fp32", seed=12)
    x.requires_grad_()

    def step():
        loss = f.topk_distillation(x, t, idx, 2.0)
        return loss.detach(), torch.autograd.grad(loss, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [v.clone() for v in step()]
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    got[1].zero_()
    gr.replay()
    torch.cuda.synchronize()
    assert all(same_bits(a, b) for a, b in zip(want, got))


# ----------------------------------------------------------------------------------------------
# load balance
# ----------------------------------------------------------------------------------------------
def balance_inputs(tokens, experts, k, dtype, seed=0, idx_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(tokens, experts, generator=g) * 1.5 + torch.randn(experts, generator=g)).to(DT[dtype])
    idx = x.float().topk(k, dim=-1).indices
    return x.to(device()), idx.to(idx_dtype).to(device())


def check_balance(x, idx, score="softmax", valid=None, offsets=None, grad_scale=1.0):
    e = x.shape[-1]
    flat = x.reshape(-1, e)
    loss, counts, gref, size = balance_ref(flat, idx.reshape(-1, idx.shape[-1]), score,
                                           None if valid is None else valid.reshape(-1), offsets)
    if offsets is None:
        loss, counts = loss[0], counts[0]
    lb = balance_loss_bound(loss, flat.shape[0], e)
    gref, size = gref.view(x.shape) * grad_scale, size.view(x.shape)
    gb = balance_grad_bound(gref, size, grad_scale, e, x.dtype)
    f = F()
    kw = dict(score=score, valid=valid, offsets=offsets)
    with torch.no_grad():
        only, c0 = f.balance_loss(x, idx, **kw)
    both, c1, grad = f.balance_loss_with_grad(x, idx, grad_scale=grad_scale, **kw)
    leaf = (x.detach().clone() if x.is_contiguous() else x.detach()).requires_grad_()
    out, c2 = f.balance_loss(leaf, idx, **kw)
    (auto,) = torch.autograd.grad(out.sum() * grad_scale, leaf)
    for got, what in ((only, "loss"), (both, "loss of with_grad"), (out.detach(), "loss through autograd")):
        assert got.dtype == torch.float32 and got.shape == loss.shape
        close(got, loss, lb, what)
    for c in (c0, c1, c2):
        assert c.dtype == torch.int64 and torch.equal(c.cpu(), counts)
    for got, what in ((grad, "grad of with_grad"), (auto, "grad through autograd")):
        assert got.dtype == x.dtype and got.shape == x.shape
        close(got, gref, gb, what)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens, experts, k", [
    (1, 1, 1), (1, 8, 2), (5, 2, 1), (48, 8, 2), (33, 60, 4), (100, 64, 2), (257, 100, 7), (1000, 128, 4), (65, 256, 8),
    (300, 441, 5), (129, 512, 8), (70, 1000, 3), (40, 1023, 2), (90, 1024, 8), (9473, 16, 2), (20011, 24, 3),
])
def test_balance_sizes(tokens, experts, k, score, dtype):
    x, idx = balance_inputs(tokens, experts, k, dtype, seed=tokens)
    check_balance(x, idx, score, grad_scale=float(tokens))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens, cuts", [
    (50, [0, 50]), (50, [0, 1, 2, 3, 50]), (50, [5, 5, 5, 20, 20, 41]), (50, [0, 0, 0]), (50, [50, 50]), (700, [0, 300, 700]),
    (700, list(range(0, 701))), (5000, [3, 40, 41, 1000, 1000, 3777, 4990]), (10000, [0, 10000]), (10000, [0, 4999, 5000, 9999]),
])
def test_balance_sequences(tokens, cuts, score):
    x, idx = balance_inputs(tokens, 40, 3, "fp32", seed=len(cuts), idx_dtype=torch.int32)
    for dt in (torch.int32, torch.int64):
        check_balance(x, idx, score, offsets=torch.tensor(cuts, dtype=dt, device=device()), grad_scale=50.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_many_sequences(score):
    """More sequences than offsets are kept in shared memory: some empty, some of one token, some of hundreds."""
    g = torch.Generator().manual_seed(11)
    sizes = torch.randint(0, 8, (3000,), generator=g)
    sizes[::500] = 300
    cuts = torch.cat([torch.tensor([2]), 2 + sizes.cumsum(0)])
    x, idx = balance_inputs(int(cuts[-1]) + 5, 20, 2, "fp32", seed=12)
    check_balance(x, idx, score, offsets=cuts.to(device()), grad_scale=10.0)


def test_balance_tokens_beyond_32_bit_offsets():
    tokens, experts = 8400000, 256  # 2.15e9 logits
    g = torch.Generator(device=device()).manual_seed(1)
    x = torch.empty(tokens, experts, dtype=torch.bfloat16, device=device())
    for a in range(0, tokens, tokens // 8):
        x[a:a + tokens // 8].normal_(generator=g)
    idx = torch.randint(experts, (tokens, 1), device=device(), generator=g, dtype=torch.int32)
    loss, counts, grad = F().balance_loss_with_grad(x, idx, grad_scale=float(tokens))
    assert torch.equal(counts, torch.bincount(idx[:, 0], minlength=experts))
    mass = torch.zeros(experts, dtype=torch.float64, device=device())
    for a in range(0, tokens, tokens // 40):
        mass += torch.softmax(x[a:a + tokens // 40].double(), 1).sum(0)
    f = experts * counts.double() / tokens
    ref = (f * mass).sum().cpu() / tokens
    close(loss, ref, balance_loss_bound(ref, tokens // 2368, experts))  # tokens per warp: what is added in fp32
    edge = 2 ** 31 // experts
    for r in (0, edge - 1, edge, tokens - 1):
        p = torch.softmax(x[r:r + 1].double(), 1)
        dot = (f * p).sum(1, keepdim=True)
        want, size = p * (f - dot), p * (f + dot)
        close(grad[r:r + 1], want.cpu(), balance_grad_bound(want.cpu(), size.cpu(), 1.0, experts, torch.bfloat16))


def test_balance_masks_drops_and_repeated_experts():
    x, idx = balance_inputs(2000, 32, 4, "fp32", seed=3)
    g = torch.Generator().manual_seed(4)
    valid = (torch.rand(2000, generator=g) < 0.7).to(device())
    x[~valid] = float("nan")              # what is masked may hold anything
    x[~valid, ::3] = INF
    idx[::9, 0] = -1                      # dropped
    idx[~valid] = 10 ** 6                 # not looked at either
    idx[1::7, 1] = idx[1::7, 2]           # an expert twice for one token
    x[valid, 5] = -INF                    # an expert that nobody may use
    x[10, :] = torch.finfo(torch.float32).min  # all alike, at the lowest value
    valid[10], x[10] = True, torch.finfo(torch.float32).min
    idx[10] = torch.arange(4, device=device())
    for score in ("softmax", "sigmoid"):
        if score == "sigmoid":
            x[10] = -80.0                 # sigmoids of 1e-35
        check_balance(x, idx, score, valid, grad_scale=2000.0)
        check_balance(x, idx, score, valid, torch.tensor([1, 7, 600, 600, 1500, 1990], device=device()), grad_scale=100.0)
    check_balance(x, idx, "softmax", torch.zeros_like(valid))


def test_balance_sequence_without_valid_tokens():
    x, idx = balance_inputs(100, 8, 2, "bf16", seed=5)
    valid = torch.ones(100, dtype=torch.bool, device=device())
    valid[20:40] = False
    check_balance(x, idx, "softmax", valid, torch.tensor([0, 20, 40, 100], device=device()), grad_scale=10.0)


def test_balance_bad_rows_bad_indices_bad_offsets():
    f = F()
    x, idx = balance_inputs(100, 8, 2, "fp32", seed=6)
    offsets = torch.tensor([0, 30, 60, 100], device=device())
    idx[35, 1] = 8
    idx[36, 0] = torch.iinfo(torch.int64).max
    for call in ("with_grad", "autograd"):
        leaf = x.clone().requires_grad_()
        if call == "with_grad":
            loss, counts, grad = f.balance_loss_with_grad(leaf, idx, offsets=offsets)
        else:
            loss, counts = f.balance_loss(leaf, idx, offsets=offsets)
            (grad,) = torch.autograd.grad(loss.sum(), leaf)
        assert loss.isnan().tolist() == [False, True, False]
        assert grad[30:60].isnan().all() and not grad[:30].isnan().any() and not grad[60:].isnan().any()
        assert counts.sum(1).tolist() == [60, 58, 80]
    idx[35, 1] = idx[36, 0] = 0
    x[3, 2] = float("nan")
    loss, counts, grad = f.balance_loss_with_grad(x, idx, offsets=offsets)
    assert loss.isnan().tolist() == [True, False, False] and grad[3].isnan().all() and not grad[4:].isnan().any()
    for cuts in ([0, 60, 30, 100], [-1, 30, 100], [0, 30, 101], [100, 0], [2 ** 40, 7, -2 ** 40]):
        loss, _, grad = f.balance_loss_with_grad(x, idx, offsets=torch.tensor(cuts, device=device()))
        assert loss.isnan().all() and grad.shape == x.shape


@pytest.mark.parametrize("make", [
    lambda b: b[:, :-1], lambda b: b[:, 1:], lambda b: b[..., :-3], lambda b: b[..., 1:], lambda b: b.transpose(0, 1),
    lambda b: b[0, 0].expand(4, 50, b.shape[-1]), lambda b: b.transpose(1, 2)[..., :40], lambda b: b[None],
], ids=["first tokens", "later tokens", "padded columns", "off the boundary", "transposed rows", "expanded", "columns not dense",
        "four axes"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_balance_strides(make, dtype):
    g = torch.Generator().manual_seed(8)
    x = make(torch.randn(4, 50, 64, generator=g).to(DT[dtype]).to(device()))
    idx = torch.randint(x.shape[-1], x.shape[:-1] + (3,), generator=g).to(device())
    valid = (torch.rand(x.shape[:-1], generator=g) < 0.8).to(device())
    check_balance(x, idx, "softmax", valid, grad_scale=200.0)
    check_balance(x, idx.transpose(-1, -2).contiguous().transpose(-1, -2), "sigmoid", grad_scale=200.0)


def test_balance_of_nothing():
    f = F()
    x = torch.randn(0, 8, device=device(), requires_grad=True)
    idx = torch.zeros(0, 2, dtype=torch.int64, device=device())
    loss, counts = f.balance_loss(x, idx)
    assert loss.item() == 0.0 and counts.tolist() == [0] * 8
    assert torch.autograd.grad(loss, x)[0].shape == (0, 8)
    loss, counts, grad = f.balance_loss_with_grad(x, idx, offsets=torch.zeros(4, dtype=torch.int32, device=device()))
    assert loss.tolist() == [0.0] * 3 and counts.shape == (3, 8) and not counts.any() and grad.shape == (0, 8)


def test_balance_gradient_against_differences():
    """Along d of +-1 a score's third derivative is at most 15 times the score, so the loss's at most 15 times the loss."""
    x, idx = balance_inputs(64, 16, 2, "fp32", seed=9)
    for score, most in (("softmax", 15.0), ("sigmoid", 60.0)):  # log sigmoid adds its own three derivatives, each below 1
        loss, _, grad = F().balance_loss_with_grad(x, idx, score)
        d = torch.where(grad >= 0, 1.0, -1.0)
        h = 2.0 ** -6
        with torch.no_grad():
            up, down = (F().balance_loss(x + s * h * d, idx, score)[0].double().item() for s in (1, -1))
        tol = most * h * h / 6 * 1.1 * loss.item() + float(balance_loss_bound(loss.double(), 64, 16)) * 1.2 / h
        assert abs((up - down) / (2 * h) - (grad.double() * d).sum().item()) < tol


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens, experts", [(64, 8), (8192, 16), (20000, 125)])
def test_balance_of_an_even_router(tokens, experts, score):
    """Even counts: no gradient at all.  One assignment moved: the gradient is that of counts (1, -1, 0, ...), to a few roundings
    of its own size and not of the counts'."""
    x = torch.randn(tokens, experts, generator=torch.Generator().manual_seed(13)).to(device())
    idx = (torch.arange(tokens, device=device()) % experts)[:, None]
    if tokens % experts == 0:
        _, counts, grad = F().balance_loss_with_grad(x, idx, score, grad_scale=float(tokens))
        assert counts.unique().numel() == 1 and not grad.any()
    idx[0] = 1
    check_balance(x, idx, score, grad_scale=float(tokens))
    _, counts, grad = F().balance_loss_with_grad(x, idx, score, grad_scale=float(tokens))
    x64 = x.double().cpu()
    logp = torch.log_softmax(x64 if score == "softmax" else torch.nn.functional.logsigmoid(x64), 1)
    p, c = logp.exp(), (counts - counts[0]).double().cpu()
    slope = 1.0 if score == "softmax" else torch.sigmoid(-x64)
    dot = (c * p).sum(1, keepdim=True)
    ref = experts / tokens * p * (c - dot) * slope
    close(grad, ref, balance_grad_bound(ref, experts / tokens * p * (c.abs() + (c.abs() * p).sum(1, keepdim=True)) * slope, 1.0,
                                        experts, torch.float32))


def test_balance_counts_do_not_take_part_in_autograd():
    x, idx = balance_inputs(20, 8, 2, "fp32")
    loss, counts = F().balance_loss(x.requires_grad_(), idx)
    assert loss.requires_grad and not counts.requires_grad
    (a,) = torch.autograd.grad(loss * 3.0, x, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x)
    assert torch.allclose(a, 3 * b, rtol=4 * U32, atol=0)


def test_balance_same_each_time_on_streams_and_in_graphs():
    f = F()
    x, idx = balance_inputs(5000, 96, 6, "bf16", seed=10)
    cuts = torch.tensor([0, 100, 2500, 2501, 5000], device=device())
    for offsets in (None, cuts):
        want = f.balance_loss_with_grad(x, idx, offsets=offsets)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = f.balance_loss_with_grad(x, idx, offsets=offsets)
        side.synchronize()
        assert all(same_bits(a, b) for a, b in zip(want, got))
        x2 = (x * 0.5).contiguous()
        want2 = f.balance_loss_with_grad(x2, idx, offsets=offsets)
        graphs, outs = [], []
        for inp in (x, x2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                outs.append(f.balance_loss_with_grad(inp, idx, offsets=offsets))
            graphs.append(gr)
        for _ in range(3):
            for o in outs:
                o[0].zero_(), o[1].zero_(), o[2].zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                graphs[1].replay()
            graphs[0].replay()
            torch.cuda.synchronize()
            assert all(same_bits(a, b) for a, b in zip(want, outs[0]))
            assert all(same_bits(a, b) for a, b in zip(want2, outs[1]))


# ----------------------------------------------------------------------------------------------
# as they are used together, and before the optimizer step
# ----------------------------------------------------------------------------------------------
def test_losses_before_an_optimizer_step():
    """A teacher's top logits kept as 8-bit codes, a student whose loss is distillation plus balance, its weights stepped."""
    import lpmm
    f = F()
    torch.manual_seed(0)
    dev, n, h, e, v, k = device(), 64, 96, 8, 640, 16
    hidden = torch.randn(n, h, device=dev)
    head, router = (torch.nn.Parameter(torch.randn(o, h, device=dev) * 0.1) for o in (v, e))
    stored = torch.randn(n, k, device=dev).sort(-1, descending=True).values
    idx = torch.stack([torch.randperm(v, device=dev)[:k] for _ in range(n)])
    md = dict(quant_type="nonlinear", b=8, signed=True, round_type="real-nearest", scale_type="group", gp_sz=128,
              qmap=f.create_general_qmap("nonlinear", 8, True).to(dev))
    codes, made = f.vectorwise_quant(stored, **md)
    teacher = f.vectorwise_dequant(codes, **dict(md, **made, shape=stored.shape))
    assert (teacher - stored).abs().max() < 0.15
    opt = lpmm.optim.AdamW([head, router], lr=1e-2, fused=True)
    for _ in range(2):
        logits, routed = hidden @ head.t(), hidden @ router.t()
        chosen = routed.detach().topk(2).indices
        main = f.topk_distillation(logits, teacher, idx, temperature=2.0)
        aux, counts = f.balance_loss(routed, chosen)
        opt.zero_grad()
        (main + 0.01 * aux).backward()
        assert counts.sum().item() == 2 * n
        # the weights' gradients against 64 bits: g^T hidden, an inner product over n rows of fp32
        _, q, p = distill_ref(logits.detach(), teacher, idx, 2.0)
        x64 = hidden.double().cpu()
        bound = distill_grad_bound((q - p) * 2 / n, q * 2 / n, p * 2 / n, 1.0, v, torch.float32)
        ref = ((q - p) * 2 / n).t() @ x64
        slack = (n + 4) * U32 * (((q - p) * 2 / n).abs().t() @ x64.abs())
        close(head.grad, ref, bound.t() @ x64.abs() + slack, "head")
        _, _, g, size = balance_ref(routed.detach(), chosen)
        bound = balance_grad_bound(0.01 * g, size, 0.01, e, torch.float32)
        close(router.grad, (0.01 * g).t() @ x64, bound.t() @ x64.abs() + (n + 4) * U32 * ((0.01 * g).abs().t() @ x64.abs()), "router")
        # the form without autograd gives the same gradients
        _, grad = f.topk_distillation_with_grad(logits, teacher, idx, temperature=2.0)
        close(grad, (q - p) * 2 / n, distill_grad_bound((q - p) * 2 / n, q * 2 / n, p * 2 / n, 1.0, v, torch.float32))
        before = [w.detach().clone() for w in (head, router)]
        opt.step()
        assert all(bool((a != b.detach()).any()) for a, b in zip(before, (head, router)))
