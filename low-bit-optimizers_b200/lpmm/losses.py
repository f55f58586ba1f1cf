"""Training losses with their gradients, on the CUDA library (no counterpart in the reference, whose work begins at
``p.grad``): distillation from a teacher's stored top logits, and a router's load-balance loss with the number of
assignments per expert.  Reached as ``lpmm.functional.topk_distillation`` and so on.

Each comes as a differentiable function and as a ``..._with_grad`` form that returns loss and gradient of one call:
the logits are then read once instead of twice, and nothing of autograd runs.  Both launch on torch's current stream
of the logits' device and synchronise nothing.
"""
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as N

_DTYPES = {torch.float32: N.DTYPE_FP32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_FP16}
_BITS = {torch.int32: 32, torch.int64: 64}
_REDUCTIONS = {"none": N.REDUCE_NONE, "sum": N.REDUCE_SUM, "mean": N.REDUCE_MEAN}
_SCORES = {"softmax": N.SCORE_SOFTMAX, "sigmoid": N.SCORE_SIGMOID}


def _check_cuda(t, name):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor!")


def _check_tensor(t, name, dtypes, like):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, not {type(t).__name__}")
    _check_cuda(t, name)
    if t.device != like.device:
        raise RuntimeError(f"{name} is on {t.device}, the logits are on {like.device}")
    if t.dtype not in dtypes:
        raise RuntimeError(f"The type of {name} is not correct: {t.dtype}")


# -1 while no forward-mode level is open: there are no dual tensors then
_dual_level = (lambda: forward_ad._current_level) if hasattr(forward_ad, "_current_level") else (lambda: 0)


def _refuse_tangents(tensors):
    """The differentiable forms have no forward-mode derivative: a dual tensor would lose its tangent in silence."""
    for t, name in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} carries a forward-mode tangent, which is not supported: only the backward pass is")


def _row_strides(t):
    """``(tensor, inner, outer_stride, inner_stride)`` of the rows of ``t`` (its last axis, which is dense): row r
    begins at element ``(r // inner) * outer_stride + (r % inner) * inner_stride``.  A layout that two strides cannot
    say, or a last axis that is not dense, is copied."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, 1, n, 0
    if t.dim() == 1:
        return t.detach().contiguous(), 1, n, 0
    if t.stride(-1) == 1 or n == 1:
        if t.dim() == 2:
            return t, 1, t.stride(0), 0
        if t.dim() == 3:
            return (t, t.shape[1], t.stride(0), t.stride(1)) if t.shape[1] > 1 else (t, 1, t.stride(0), 0)
    return t.detach().contiguous(), 1, n, 0


def _grad_of(logits, d):
    """A tensor for the gradient of ``logits`` (the tensor that ``d`` describes), its strides in ``d``.  Contiguous where
    that puts every row to the 16-byte boundaries as the logits' row lies to them, which the kernels' wide accesses
    need; else with up to 16 bytes between rows."""
    n, at = logits.shape[-1], d.logits or 0
    if at % 16 == 0 and logits.is_contiguous():
        grad = torch.empty_like(logits)
        d.grad, d.grad_outer_stride, d.grad_inner_stride = grad.data_ptr(), d.outer_stride, d.inner_stride
        return grad
    size = logits.element_size()
    off, wide = at % 16 // size, 16 // size
    if d.inner == 1:
        inner, outer = 0, n + (d.outer_stride - n) % wide
        odd = outer != n
    else:
        inner = n + (d.inner_stride - n) % wide
        outer = d.inner * inner + (d.outer_stride - d.inner * inner) % wide
        odd = inner != n or outer != d.inner * n
    if off or odd:
        rows = -(-d.rows // d.inner)
        grad = torch.empty(off + rows * outer, dtype=logits.dtype, device=logits.device)
        if odd:  # two or three axes: others are contiguous
            strides = (outer, 1) if logits.dim() == 2 else (outer, inner or n, 1)
            grad = grad.as_strided(logits.shape, strides, off)
        else:
            grad = grad[off:].view(logits.shape)
    else:
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
    d.grad, d.grad_outer_stride, d.grad_inner_stride = grad.data_ptr(), outer, inner
    return grad


# the handle of a device's current stream; building a Stream object for it takes ten times as long
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _launch(fn, args, device):
    if device.index == torch.cuda.current_device():
        N.check(fn(args, _stream_of(device.index)))
    else:
        with torch.cuda.device(device):
            N.check(fn(args, _stream_of(device.index)))


# ----------------------------------------------------------------------------------------------
# distillation from a teacher's stored top logits
# ----------------------------------------------------------------------------------------------
def _distill_args(logits, teacher_logits, teacher_idx, temperature, weights, reduction):
    """Checked arguments -> ``(struct, tensors that the struct points to, rows, leading shape)``."""
    _check_tensor(logits, "logits", _DTYPES, logits)
    _check_tensor(teacher_logits, "teacher_logits", _DTYPES, logits)
    _check_tensor(teacher_idx, "teacher_idx", _BITS, logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError("logits must have at least one column")
    lead = logits.shape[:-1]
    if teacher_idx.shape != teacher_logits.shape or teacher_idx.dim() != logits.dim() or teacher_idx.shape[:-1] != lead:
        raise RuntimeError(f"teacher_logits and teacher_idx must be {tuple(lead)} + (k,), got "
                           f"{tuple(teacher_logits.shape)} and {tuple(teacher_idx.shape)}")
    k = teacher_idx.shape[-1]
    if not 1 <= k <= N.DISTILL_MAX_K:
        raise RuntimeError(f"1 to {N.DISTILL_MAX_K} teacher logits per row are supported, got {k}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', not {reduction!r}")
    temperature = float(temperature)
    if not N.DISTILL_MIN_T <= temperature <= N.DISTILL_MAX_T:
        raise ValueError(f"temperature must lie in [{N.DISTILL_MIN_T}, {N.DISTILL_MAX_T}], got {temperature}")
    if weights is not None:
        if not isinstance(weights, torch.Tensor) or weights.device != logits.device:
            raise RuntimeError("weights must be a tensor on the logits' device")
        if weights.shape != lead:
            raise RuntimeError(f"weights must be {tuple(lead)}, got {tuple(weights.shape)}")
        if weights.is_complex():
            raise RuntimeError(f"The type of weights is not correct: {weights.dtype}")
        if weights.dtype != torch.float32 or not weights.is_contiguous():
            weights = weights.to(torch.float32).contiguous()
    logits, inner, outer_stride, inner_stride = _row_strides(logits)
    teacher, idx = teacher_logits.contiguous(), teacher_idx.contiguous()
    d = N.Distill()
    d.logits, d.teacher, d.index = logits.data_ptr(), teacher.data_ptr(), idx.data_ptr()
    d.weights = None if weights is None else weights.data_ptr()
    d.rows = rows = logits.numel() // logits.shape[-1]
    d.inner, d.outer_stride, d.inner_stride = inner, outer_stride, inner_stride
    d.vocab, d.k = logits.shape[-1], k
    d.dtype, d.teacher_dtype, d.index_bits = _DTYPES[logits.dtype], _DTYPES[teacher.dtype], _BITS[idx.dtype]
    d.reduction, d.temperature, d.grad_scale = _REDUCTIONS[reduction], temperature, 1.0
    return d, (logits, teacher, idx, weights), rows, lead


def _distill_outputs(d, rows, lead, device):
    work = torch.empty(4 + 5 * rows, dtype=torch.float32, device=device)
    loss = torch.empty(lead if d.reduction == N.REDUCE_NONE else (), dtype=torch.float32, device=device)
    d.work, d.loss = work.data_ptr(), loss.data_ptr()
    return loss, work


class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_logits, teacher_idx, temperature, weights, reduction):
        d, kept, rows, lead = _distill_args(logits, teacher_logits, teacher_idx, temperature, weights, reduction)
        loss, work = _distill_outputs(d, rows, lead, logits.device)
        _launch(N.lib.lpmm_b200_distill_forward, d, logits.device)
        ctx.save_for_backward(logits, teacher_logits, teacher_idx, weights)
        ctx.work, ctx.how = work, (temperature, reduction)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        logits, teacher_logits, teacher_idx, weights = ctx.saved_tensors
        temperature, reduction = ctx.how
        with torch.no_grad():
            d, kept, rows, lead = _distill_args(logits, teacher_logits, teacher_idx, temperature, weights, reduction)
        grad = _grad_of(kept[0], d)
        upstream = upstream.to(torch.float32).contiguous()
        d.work, d.upstream = ctx.work.data_ptr(), upstream.data_ptr()
        _launch(N.lib.lpmm_b200_distill_backward, d, logits.device)
        return grad, None, None, None, None, None


def topk_distillation(logits, teacher_logits, teacher_idx, temperature=1.0, weights=None, reduction="mean"):
    """Divergence of the student's distribution from a teacher known by its top logits; differentiable by ``logits``.

    Per row, with ``p = softmax(teacher_logits / T)`` over the row's K stored entries and ``q = softmax(logits / T)`` over
    the whole vocabulary, the loss is ``weight * T**2 * sum_k p_k (log p_k - log q[teacher_idx_k])``.

    ``logits``: ``[..., V]``, fp32, bf16 or fp16, any strides.  ``teacher_logits``: ``[..., K]``, K up to 1024, any of
    these types; ``teacher_idx``: ``[..., K]``, int32 or int64.  An entry with a negative index or a logit of -inf is
    absent; an index given twice counts with both probabilities.  ``weights``: ``[...]``, one factor per row (a padding
    mask, for instance).  A row of weight 0, or without entries, has loss 0 and gradient 0 whatever its logits hold.
    ``reduction``: ``"none"`` gives ``[...]`` losses, ``"sum"`` their sum, ``"mean"`` the sum over the sum of the
    weights (0 if that is 0).  The loss is fp32, the gradient has the logits' type and is rounded once.

    An index of V or more makes its row's loss and gradient NaN.  Results do not depend on scheduling.  Tensors with
    forward-mode tangents are refused."""
    if _dual_level() >= 0:
        _refuse_tangents(((logits, "logits"), (teacher_logits, "teacher_logits"), (weights, "weights")))
    if torch.is_grad_enabled():
        for t, name in ((teacher_logits, "teacher_logits"), (weights, "weights")):
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise RuntimeError(f"{name} are constants of the loss: detach them")
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _TopkDistillation.apply(logits, teacher_logits, teacher_idx, temperature, weights, reduction)
    d, kept, rows, lead = _distill_args(logits, teacher_logits, teacher_idx, temperature, weights, reduction)
    loss, work = _distill_outputs(d, rows, lead, logits.device)
    _launch(N.lib.lpmm_b200_distill_forward, d, logits.device)
    return loss


def topk_distillation_with_grad(logits, teacher_logits, teacher_idx, temperature=1.0, weights=None, reduction="mean",
                                grad_scale=1.0):
    """``topk_distillation`` and its gradient in one call: ``(loss, grad)``.

    ``grad`` is ``grad_scale`` (a loss scale, a share of the total loss) times the derivative of the loss by ``logits``,
    of the losses' sum with ``reduction="none"``: a new tensor of the logits' shape and type, for ``logits.backward(grad)``
    (contiguous, but with up to 16 bytes between rows where the logits' rows lie to the 16-byte boundaries in another way
    than a contiguous tensor's would).  ``loss`` is not scaled, and neither takes part in autograd."""
    d, kept, rows, lead = _distill_args(logits, teacher_logits, teacher_idx, temperature, weights, reduction)
    loss, work = _distill_outputs(d, rows, lead, logits.device)
    grad = _grad_of(kept[0], d)
    d.grad_scale = float(grad_scale)
    _launch(N.lib.lpmm_b200_distill_forward_backward, d, logits.device)
    return loss, grad


# ----------------------------------------------------------------------------------------------
# load balance of a router
# ----------------------------------------------------------------------------------------------
def _balance_args(router_logits, expert_idx, score, valid, offsets):
    """Checked arguments -> ``(struct, tensors that the struct points to)``."""
    _check_tensor(router_logits, "router_logits", _DTYPES, router_logits)
    _check_tensor(expert_idx, "expert_idx", _BITS, router_logits)
    if router_logits.dim() < 1 or not 1 <= router_logits.shape[-1] <= N.BALANCE_MAX_EXPERTS:
        raise RuntimeError(f"router_logits must have 1 to {N.BALANCE_MAX_EXPERTS} columns")
    lead, experts = router_logits.shape[:-1], router_logits.shape[-1]
    if expert_idx.dim() != router_logits.dim() or expert_idx.shape[:-1] != lead or expert_idx.shape[-1] < 1:
        raise RuntimeError(f"expert_idx must be {tuple(lead)} + (k,), got {tuple(expert_idx.shape)}")
    if expert_idx.shape[-1] > N.BALANCE_MAX_EXPERTS:
        raise RuntimeError(f"at most {N.BALANCE_MAX_EXPERTS} experts per token are supported")
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', not {score!r}")
    b = N.Balance()
    if valid is not None:
        _check_tensor(valid, "valid", (torch.bool,), router_logits)
        if valid.shape != lead:
            raise RuntimeError(f"valid must be {tuple(lead)}, got {tuple(valid.shape)}")
        valid = valid.contiguous()
        b.valid = valid.data_ptr()
    b.sequences = 1
    if offsets is not None:
        _check_tensor(offsets, "offsets", _BITS, router_logits)
        if offsets.dim() != 1 or offsets.numel() < 2:
            raise RuntimeError("offsets must be one-dimensional: the sequences' starts and the last one's end")
        offsets = offsets.contiguous()
        b.offsets, b.offset_bits, b.sequences = offsets.data_ptr(), _BITS[offsets.dtype], offsets.numel() - 1
    logits, b.inner, b.outer_stride, b.inner_stride = _row_strides(router_logits)
    idx = expert_idx.contiguous()
    b.logits, b.index, b.tokens = logits.data_ptr(), idx.data_ptr(), logits.numel() // experts
    b.experts, b.k = experts, idx.shape[-1]
    b.dtype, b.index_bits, b.score, b.grad_scale = _DTYPES[logits.dtype], _BITS[idx.dtype], _SCORES[score], 1.0
    return b, (logits, idx, valid, offsets)


@functools.lru_cache(maxsize=64)
def _balance_work_bytes(experts, sequences):
    nbytes = N.lib.lpmm_b200_balance_work_bytes(experts, sequences)  # a multiple of 16
    if nbytes < 0:
        N.check(int(nbytes))
    return nbytes


def _balance_outputs(b, device):
    """Loss, counts, and the buffer that holds what belongs to the call: counts that the backward pass reads (the caller may do
    with the returned ones as it likes), the workspace behind them and the gradient's factors."""
    s, e = b.sequences, b.experts
    cells = s * e
    nbytes = _balance_work_bytes(e, s)
    buf = torch.empty(cells + nbytes // 8 + (s + 1) // 2, dtype=torch.int64, device=device)
    loss = torch.empty((s,) if b.offsets else (), dtype=torch.float32, device=device)
    at = buf.data_ptr()
    b.counts, b.work, b.factor, b.loss = at, at + 8 * cells, at + 8 * cells + nbytes, loss.data_ptr()
    counts = torch.empty((s, e) if b.offsets else (e,), dtype=torch.int64, device=device)
    b.counts_out = counts.data_ptr()
    return loss, counts, buf


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, router_logits, expert_idx, score, valid, offsets):
        b, kept = _balance_args(router_logits, expert_idx, score, valid, offsets)
        loss, counts, ctx.buf = _balance_outputs(b, router_logits.device)
        _launch(N.lib.lpmm_b200_balance_forward, b, router_logits.device)
        ctx.mark_non_differentiable(counts)
        ctx.save_for_backward(router_logits, expert_idx, valid, offsets)
        ctx.counts, ctx.factor, ctx.score = b.counts, b.factor, score
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream, _):
        router_logits, expert_idx, valid, offsets = ctx.saved_tensors
        b, kept = _balance_args(router_logits, expert_idx, ctx.score, valid, offsets)
        grad = torch.empty_like(router_logits, memory_format=torch.contiguous_format)
        upstream = upstream.to(torch.float32).contiguous()
        b.grad, b.upstream, b.counts, b.factor = grad.data_ptr(), upstream.data_ptr(), ctx.counts, ctx.factor
        _launch(N.lib.lpmm_b200_balance_backward, b, router_logits.device)
        return grad, None, None, None, None


def balance_loss(router_logits, expert_idx, score="softmax", valid=None, offsets=None):
    """Load-balance loss of a mixture's router and the assignments per expert: ``(loss, counts)``; the loss is
    differentiable by ``router_logits``.

    With the scores ``p`` of a token over E experts (``"softmax"`` of its logits, or ``"sigmoid"``: the logits' sigmoids
    divided by their sum) and the k experts that were chosen for it, a sequence of n valid tokens has
    ``loss = sum_e f_e P_e``, ``f_e = E * counts_e / (k * n)`` and ``P_e`` the mean of ``p_e``; even use gives 1.

    ``router_logits``: ``[..., E]``, E up to 1024, fp32, bf16 or fp16, any strides.  ``expert_idx``: ``[..., k]``, int32
    or int64; a negative one is a dropped assignment and is not counted.  ``valid``: bool ``[...]``; a token that is not
    valid takes no part and has gradient 0 whatever its logits hold.  ``offsets``: int32 or int64 ``[S + 1]``, ascending:
    sequence s is the flattened tokens ``offsets[s]`` to ``offsets[s + 1]``, with a loss and counts of its own (``[S]``
    and ``[S, E]``, else scalar and ``[E]``); tokens outside of all sequences take no part, a sequence without valid
    tokens has loss 0.  Loss fp32, counts int64 (the caller's own: nothing reads them later), gradient of the logits'
    type, rounded once.

    An index of E or more makes its sequence's loss and gradient NaN, offsets that descend or leave the range make every
    loss NaN.  Results do not depend on scheduling.  Logits with a forward-mode tangent are refused."""
    if _dual_level() >= 0:
        _refuse_tangents(((router_logits, "router_logits"),))
    if torch.is_grad_enabled() and isinstance(router_logits, torch.Tensor) and router_logits.requires_grad:
        return _BalanceLoss.apply(router_logits, expert_idx, score, valid, offsets)
    b, kept = _balance_args(router_logits, expert_idx, score, valid, offsets)
    loss, counts, buf = _balance_outputs(b, router_logits.device)
    _launch(N.lib.lpmm_b200_balance_forward, b, router_logits.device)
    return loss, counts


def balance_loss_with_grad(router_logits, expert_idx, score="softmax", valid=None, offsets=None, grad_scale=1.0):
    """``balance_loss`` and its gradient in one call: ``(loss, counts, grad)``.

    ``grad`` is ``grad_scale`` times the derivative of the loss (of the losses' sum with ``offsets``) by
    ``router_logits``: a new contiguous tensor of their shape and type.  Nothing takes part in autograd."""
    b, kept = _balance_args(router_logits, expert_idx, score, valid, offsets)
    loss, counts, buf = _balance_outputs(b, router_logits.device)
    grad = torch.empty_like(router_logits, memory_format=torch.contiguous_format)
    b.grad, b.grad_scale = grad.data_ptr(), float(grad_scale)
    _launch(N.lib.lpmm_b200_balance_forward_backward, b, router_logits.device)
    return loss, counts, grad
