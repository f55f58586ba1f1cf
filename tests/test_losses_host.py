"""Host side of the training losses, without a GPU: which buffers the forms share, which calls are refused."""
import pytest
import torch
from torch.autograd import forward_ad

from lpmm import _native as N
from lpmm import functional as F
from lpmm import losses as L


@pytest.fixture
def host(monkeypatch):
    """The public functions on CPU tensors: the CUDA check is left out and launches are recorded."""
    calls = []
    monkeypatch.setattr(L, "_check_cuda", lambda t, name: None)
    monkeypatch.setattr(L, "_launch", lambda fn, args, device: calls.append((fn.__name__, args)))
    return calls


@pytest.mark.parametrize("offsets", [None, torch.tensor([0, 2, 6])])
def test_returned_counts_are_not_what_backward_reads(host, offsets):
    x, idx = torch.randn(6, 8, requires_grad=True), torch.zeros(6, 2, dtype=torch.int64)
    loss, counts = F.balance_loss(x, idx, offsets=offsets)
    name, forward = host.pop()
    assert name == "lpmm_b200_balance_forward" and forward.counts_out == counts.data_ptr()
    cells = 8 * (1 if offsets is None else 2)
    assert counts.numel() == cells and counts.untyped_storage().nbytes() == 8 * cells
    assert not counts.data_ptr() <= forward.counts < counts.data_ptr() + 8 * cells
    counts.zero_()
    loss.sum().backward()
    name, backward = host.pop()
    assert name == "lpmm_b200_balance_backward"
    assert (backward.counts, backward.factor, backward.counts_out) == (forward.counts, forward.factor, None)


def test_returned_counts_keep_no_workspace(host):
    x, idx = torch.randn(6, 8), torch.zeros(6, 2, dtype=torch.int64)
    for call in (F.balance_loss, F.balance_loss_with_grad):
        counts = call(x, idx)[1]
        assert counts.untyped_storage().nbytes() == 64
        assert host.pop()[1].counts_out == counts.data_ptr()


@pytest.mark.parametrize("name", ["logits", "teacher_logits", "weights", "router_logits"])
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("leaf", [False, True])
def test_tensors_with_a_forward_tangent_are_refused(host, name, grad_mode, leaf):
    kw = dict(logits=torch.randn(3, 10), teacher_logits=torch.randn(3, 2), teacher_idx=torch.zeros(3, 2, dtype=torch.int64),
              weights=torch.ones(3))
    call = F.topk_distillation
    if name == "router_logits":
        call, kw = F.balance_loss, dict(router_logits=torch.randn(3, 10), expert_idx=torch.zeros(3, 2, dtype=torch.int64))
    if leaf:
        kw["logits" if name != "router_logits" else name].requires_grad_()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = dict(kw, **{name: forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))})
        with pytest.raises(RuntimeError, match=f"{name} carries a forward-mode tangent"):
            call(**dual)
        assert not host, "nothing may be launched"
        call(**kw)  # without a tangent it is an ordinary call
        assert len(host) == 1


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("shape", [(0, 10), (2, 0, 10)])
def test_backward_of_no_rows(monkeypatch, reduction, shape):
    """Through the library's own checks; without rows the backward pass launches nothing."""
    monkeypatch.setattr(L, "_check_cuda", lambda t, name: None)
    status = []

    def launch(fn, args, device):
        if fn is N.lib.lpmm_b200_distill_backward:
            status.append(fn(args, None))
            N.check(status[-1])
    monkeypatch.setattr(L, "_launch", launch)
    x = torch.randn(shape, requires_grad=True)
    t, idx = torch.zeros(*shape[:-1], 2), torch.zeros(*shape[:-1], 2, dtype=torch.int64)
    loss = F.topk_distillation(x, t, idx, reduction=reduction)
    (grad,) = torch.autograd.grad(loss.sum(), x)
    assert grad.shape == shape and status == [0]
