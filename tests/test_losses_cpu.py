"""Host side of the training losses, without a GPU: what is refused, what the C structures are given, the row layout."""
import ctypes

import pytest
import torch

from lpmm import _native as N
from lpmm import functional as F
from lpmm import losses as L


@pytest.fixture
def host(monkeypatch):
    """The checks of the public functions on CPU tensors: the CUDA check is left out and launches are recorded."""
    calls = []
    monkeypatch.setattr(L, "_check_cuda", lambda t, name: None)
    monkeypatch.setattr(L, "_launch", lambda fn, args, device: calls.append((fn.__name__, args)))
    return calls


def _distill(rows=(3,), v=10, k=2):
    return torch.randn(*rows, v), torch.randn(*rows, k), torch.zeros(*rows, k, dtype=torch.int64)


def test_cpu_tensors_are_refused():
    x, t, i = _distill()
    for call in (F.topk_distillation, F.topk_distillation_with_grad):
        with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
            call(x, t, i)
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        F.topk_distillation(x.requires_grad_(), t, i)
    for call in (F.balance_loss, F.balance_loss_with_grad):
        with pytest.raises(RuntimeError, match="router_logits must be a CUDA tensor"):
            call(torch.randn(4, 8), torch.zeros(4, 2, dtype=torch.int64))


@pytest.mark.parametrize("what, change, error, text", [
    ("type of the logits", dict(logits=torch.randn(3, 10).double()), RuntimeError, "type of logits"),
    ("no columns", dict(logits=torch.randn(3, 0)), RuntimeError, "at least one column"),
    ("not a tensor", dict(logits=[1.0]), TypeError, "must be a tensor"),
    ("type of the index", dict(teacher_idx=torch.zeros(3, 2, dtype=torch.int16)), RuntimeError, "type of teacher_idx"),
    ("type of the teacher", dict(teacher_logits=torch.zeros(3, 2).double()), RuntimeError, "type of teacher_logits"),
    ("rows", dict(teacher_idx=torch.zeros(4, 2, dtype=torch.int64), teacher_logits=torch.zeros(4, 2)), RuntimeError, "must be"),
    ("broadcast rows", dict(teacher_idx=torch.zeros(1, 2, dtype=torch.int64), teacher_logits=torch.zeros(1, 2)), RuntimeError,
     "must be"),
    ("shapes differ", dict(teacher_idx=torch.zeros(3, 3, dtype=torch.int64)), RuntimeError, "must be"),
    ("no entries", dict(teacher_idx=torch.zeros(3, 0, dtype=torch.int64), teacher_logits=torch.zeros(3, 0)), RuntimeError,
     "teacher logits per row"),
    ("too many entries", dict(teacher_idx=torch.zeros(3, 1025, dtype=torch.int64), teacher_logits=torch.zeros(3, 1025)),
     RuntimeError, "teacher logits per row"),
    ("temperature 0", dict(temperature=0.0), ValueError, "temperature"),
    ("temperature NaN", dict(temperature=float("nan")), ValueError, "temperature"),
    ("temperature inf", dict(temperature=float("inf")), ValueError, "temperature"),
    ("negative temperature", dict(temperature=-1.0), ValueError, "temperature"),
    ("reduction", dict(reduction="batchmean"), ValueError, "reduction"),
    ("weights' shape", dict(weights=torch.ones(3, 1)), RuntimeError, "weights must be"),
    ("weights' type", dict(weights=torch.ones(3, dtype=torch.complex64)), RuntimeError, "type of weights"),
    ("weights as a list", dict(weights=[1.0, 1.0, 1.0]), RuntimeError, "weights must be a tensor"),
])
def test_distillation_refuses(host, what, change, error, text):
    x, t, i = _distill()
    kw = dict(logits=x, teacher_logits=t, teacher_idx=i)
    kw.update(change)
    for call in (F.topk_distillation, F.topk_distillation_with_grad):
        with pytest.raises(error, match=text):
            call(**kw)
    assert not host, "nothing may be launched"


def test_constants_that_want_a_gradient_are_refused(host):
    x, t, i = _distill()
    with pytest.raises(RuntimeError, match="teacher_logits are constants"):
        F.topk_distillation(x, t.requires_grad_(), i)
    with pytest.raises(RuntimeError, match="weights are constants"):
        F.topk_distillation(x, t.detach(), i, weights=torch.ones(3).requires_grad_())
    with torch.no_grad():
        F.topk_distillation(x, t, i)
    assert len(host) == 1


@pytest.mark.parametrize("what, change, error, text", [
    ("type", dict(router_logits=torch.randn(4, 8).double()), RuntimeError, "type of router_logits"),
    ("no experts", dict(router_logits=torch.randn(4, 0)), RuntimeError, "columns"),
    ("too many experts", dict(router_logits=torch.randn(4, 1025)), RuntimeError, "columns"),
    ("index type", dict(expert_idx=torch.zeros(4, 2, dtype=torch.uint8)), RuntimeError, "type of expert_idx"),
    ("index rows", dict(expert_idx=torch.zeros(5, 2, dtype=torch.int64)), RuntimeError, "expert_idx must be"),
    ("index without k", dict(expert_idx=torch.zeros(4, dtype=torch.int64)), RuntimeError, "expert_idx must be"),
    ("k of 0", dict(expert_idx=torch.zeros(4, 0, dtype=torch.int64)), RuntimeError, "expert_idx must be"),
    ("score", dict(score="tanh"), ValueError, "score"),
    ("valid's type", dict(valid=torch.ones(4)), RuntimeError, "type of valid"),
    ("valid's shape", dict(valid=torch.ones(4, 1, dtype=torch.bool)), RuntimeError, "valid must be"),
    ("offsets' type", dict(offsets=torch.zeros(3)), RuntimeError, "type of offsets"),
    ("offsets' shape", dict(offsets=torch.zeros(2, 2, dtype=torch.int64)), RuntimeError, "one-dimensional"),
    ("one offset", dict(offsets=torch.zeros(1, dtype=torch.int64)), RuntimeError, "one-dimensional"),
])
def test_balance_refuses(host, what, change, error, text):
    kw = dict(router_logits=torch.randn(4, 8), expert_idx=torch.zeros(4, 2, dtype=torch.int64))
    kw.update(change)
    for call in (F.balance_loss, F.balance_loss_with_grad):
        with pytest.raises(error, match=text):
            call(**kw)
    assert not host


def _rows_of(t, inner, outer, step):
    """First elements of the rows that the layout names, read from the storage."""
    inner = max(inner, 1)
    flat = t.as_strided((t.untyped_storage().nbytes() // t.element_size(),), (1,), 0)
    rows = t.numel() // t.shape[-1]
    at = [t.storage_offset() + (r // inner) * outer + (r % inner) * step for r in range(rows)]
    return flat[torch.tensor(at, dtype=torch.int64)] if rows else flat[:0]


@pytest.mark.parametrize("make, copied", [
    (lambda: torch.randn(5, 7), False),
    (lambda: torch.randn(5, 9)[:, :7], False),
    (lambda: torch.randn(4, 6, 7)[:, :-1], False),
    (lambda: torch.randn(4, 6, 7)[:, 1:], False),
    (lambda: torch.randn(4, 6, 7).transpose(0, 1), False),
    (lambda: torch.randn(1, 7).expand(5, 7), False),
    (lambda: torch.randn(2, 3, 4, 7), False),
    (lambda: torch.randn(2, 3, 4, 8)[..., 1:], True),
    (lambda: torch.randn(7, 5).t(), True),
    (lambda: torch.randn(14)[::2], True),
    (lambda: torch.randn(7), False),
    (lambda: torch.randn(5, 3)[:, 1:2], False),
    (lambda: torch.randn(0, 7), False),
    (lambda: torch.randn(3, 0, 7).transpose(0, 1), False),
])
def test_row_layout(make, copied):
    t = make()
    got, inner, outer, step = L._row_strides(t)
    assert (got is not t) == copied and inner >= 1
    assert torch.equal(_rows_of(got, inner, outer, step), t.reshape(-1, t.shape[-1])[:, 0])


@pytest.mark.parametrize("make", [
    lambda b: b, lambda b: b[:, :-1], lambda b: b[:, 1:], lambda b: b[..., :-3], lambda b: b[..., 1:], lambda b: b.transpose(0, 1),
    lambda b: b[0, 0].expand(4, 5, 203), lambda b: b.transpose(1, 2), lambda b: b[:, ::2, 3:], lambda b: b[None],
    lambda b: b[1, 2], lambda b: b[:, 1], lambda b: b[:0], lambda b: b[:, :1, 5:6], lambda b: b.reshape(-1)[1:].view(1, -1),
    lambda b: b.transpose(0, 1)[:, 1:],
])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_layout(make, dtype):
    """The gradient's rows are where the structure says, apart, inside their storage, and like the logits' rows to 16 bytes."""
    t = make(torch.zeros(4, 5, 203, dtype=dtype))
    got, inner, outer, step = L._row_strides(t)
    d = N.Distill(logits=got.data_ptr(), inner=inner, outer_stride=outer, inner_stride=step, rows=got.numel() // got.shape[-1])
    g = L._grad_of(got, d)
    assert g.shape == t.shape and g.dtype == dtype
    flat = g.as_strided((g.untyped_storage().nbytes() // g.element_size(),), (1,), 0).fill_(-1)
    g.copy_((torch.arange(g.numel()) % 251).view(g.shape))
    assert torch.equal(g.reshape(-1).float(), torch.arange(g.numel()).remainder(251).float())
    assert torch.equal(_rows_of(g, inner, d.grad_outer_stride, d.grad_inner_stride), g.reshape(-1, g.shape[-1])[:, 0])
    wide = 16 // t.element_size()
    if d.rows:
        assert d.grad == g.data_ptr() and (got.data_ptr() - d.grad) % 16 == 0
    assert (outer - d.grad_outer_stride) % wide == 0 and (step - d.grad_inner_stride) % wide == 0
    assert flat.numel() <= g.numel() + wide * (d.rows + 2 + d.rows // max(inner, 1))


def test_structures_as_the_library_gets_them(host):
    x, t, i = _distill((2, 3), 10, 4)
    F.topk_distillation_with_grad(x[:, :2], t[:, :2], i[:, :2].int(), temperature=2.0, weights=torch.ones(2, 2, dtype=torch.bool),
                                  reduction="sum", grad_scale=3.0)
    name, d = host.pop()
    assert name == "lpmm_b200_distill_forward_backward"
    assert (d.rows, d.inner, d.outer_stride, d.inner_stride, d.vocab, d.k) == (4, 2, 30, 10, 10, 4)
    assert (d.dtype, d.teacher_dtype, d.index_bits, d.reduction) == (N.DTYPE_FP32, N.DTYPE_FP32, 32, N.REDUCE_SUM)
    assert (d.temperature, d.grad_scale) == (2.0, 3.0) and d.weights and d.work % 16 == 0
    F.balance_loss(torch.randn(6, 8).bfloat16(), torch.zeros(6, 2, dtype=torch.int32), score="sigmoid",
                   offsets=torch.tensor([0, 2, 6]))
    name, b = host.pop()
    assert name == "lpmm_b200_balance_forward"
    assert (b.tokens, b.experts, b.k, b.sequences) == (6, 8, 2, 2)
    assert (b.dtype, b.index_bits, b.offset_bits, b.score) == (N.DTYPE_BF16, 32, 64, N.SCORE_SIGMOID)


def test_library_refuses_bad_arguments_before_any_launch():
    lib, ref = N.lib, ctypes.byref
    assert lib.lpmm_b200_distill_work_floats(3) == 19 and lib.lpmm_b200_distill_work_floats(-1) == -2
    assert lib.lpmm_b200_balance_work_bytes(0, 1) == -2 and lib.lpmm_b200_balance_work_bytes(1025, 1) == -2
    assert lib.lpmm_b200_balance_work_bytes(1, 1) > 0
    forms = (lib.lpmm_b200_distill_forward, lib.lpmm_b200_distill_backward, lib.lpmm_b200_distill_forward_backward)
    good = dict(rows=1, inner=1, outer_stride=8, vocab=8, k=1, index_bits=32, temperature=1.0, grad_scale=1.0)
    for fn in forms:
        assert fn(None, None) == -1
        for change, status in ((dict(rows=-1), -2), (dict(inner=0), -2), (dict(vocab=0), -2), (dict(k=0), -2), (dict(dtype=3), -3),
                               (dict(teacher_dtype=-1), -3), (dict(index_bits=16), -3), (dict(reduction=3), -3),
                               (dict(temperature=0.0), -2), (dict(temperature=float("nan")), -2), (dict(k=1025), -6),
                               (dict(vocab=(1 << 30) + 1), -6), (dict(rows=1 << 28), -6), (dict(), -1)):
            assert fn(ref(N.Distill(**dict(good, **change))), None) == status, (fn.__name__, change)
    # work off its boundary
    some = (ctypes.c_float * 64)()
    at = ctypes.addressof(some)
    d = N.Distill(**dict(good, logits=at, grad=at, teacher=at, index=at, upstream=at, loss=at, work=(at + 15) // 16 * 16 + 4))
    assert all(fn(ref(d), None) == -2 for fn in forms)
    # a gradient that lies otherwise to the 16-byte boundaries than the logits
    room = (at + 15) // 16 * 16
    for change in (dict(grad=room + 4), dict(grad_outer_stride=9)):
        d = N.Distill(**dict(dict(good, logits=room, grad=room, teacher=at, index=at, upstream=at, loss=at, work=room,
                                  grad_outer_stride=8), **change))
        assert all(fn(ref(d), None) == -2 for fn in forms[1:])
    forms = (lib.lpmm_b200_balance_forward, lib.lpmm_b200_balance_backward, lib.lpmm_b200_balance_forward_backward)
    good = dict(tokens=1, inner=1, outer_stride=8, experts=8, k=1, sequences=1, index_bits=64)
    for fn in forms:
        assert fn(None, None) == -1
        for change, status in ((dict(tokens=-1), -2), (dict(inner=0), -2), (dict(experts=0), -2), (dict(k=0), -2),
                               (dict(sequences=0), -2), (dict(sequences=2), -3), (dict(dtype=7), -3), (dict(index_bits=8), -3),
                               (dict(score=2), -3), (dict(offsets=at, offset_bits=0), -3), (dict(experts=1025), -6),
                               (dict(k=1025), -6), (dict(tokens=(1 << 30) + 1), -6), (dict(), -1)):
            assert fn(ref(N.Balance(**dict(good, **change))), None) == status, (fn.__name__, change)
