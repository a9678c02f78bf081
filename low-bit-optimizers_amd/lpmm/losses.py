"""Terms of a training loss with their gradients: distillation from a teacher's top logits (with the label's cross entropy
from the same pass) and the balance of a router's experts.

The reference has no counterpart.  The optimizers end a training step; these stand where its gradients begin, and a
teacher's values may come in the block-wise codes in which the optimizers keep their states
(`lpmm.functional.vectorwise_quant`).  The kernels are in liblpmm_hip.so; there is no CPU or PyTorch fallback.  Work is
enqueued on torch's current stream of the tensors' device, nothing waits for the GPU, and a call can be recorded
into a graph.
"""
import math

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .cpp_extension._checks import same_device

__all__ = ["balance_loss", "distill_loss"]

_TYPES = {torch.float32: _native.TYPE_F32, torch.float16: _native.TYPE_F16, torch.bfloat16: _native.TYPE_BF16}
_ID_BITS = {torch.int32: 32, torch.int64: 64}
_REDUCTIONS = {"none": _native.REDUCE_NONE, "sum": _native.REDUCE_SUM, "mean": _native.REDUCE_MEAN}


def _require_tensors(**tensors):
    for name, t in tensors.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")


def _require_cuda(**tensors):
    """The tensors' device; checked after everything that can be said without one."""
    for name, t in tensors.items():
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor!")
    return same_device(*[t for t in tensors.values() if t is not None])


def _type_of(t, name):
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise RuntimeError(f"The type of {name} is not float32, float16 or bfloat16: {t.dtype}")
    return kind


def _finite(value, name):
    value = float(value)
    if not math.isfinite(value):
        raise ValueError(f"{name} must be finite, got {value}")
    return value


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _row_strides(t):
    """(tensor, inner, outer stride, inner stride): row n of the flattened leading dimensions starts at
    (n // inner) * outer + (n % inner) * inner stride.  Views such as logits[:, :-1] fit; others are copied."""
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        levels = []  # (length, stride), adjacent dimensions joined
        for length, stride in zip(t.shape[:-1], t.stride()[:-1]):
            if length == 1:
                continue
            if levels and levels[-1][1] == length * stride:
                levels[-1] = (levels[-1][0] * length, stride)
            else:
                levels.append((length, stride))
        if not levels or t.numel() == 0:
            return t, 1, 0, 0
        if len(levels) == 1:
            return t, levels[0][0], 0, levels[0][1]
        if len(levels) == 2:
            return t, levels[1][0], levels[0][1], levels[1][1]
    t = t.contiguous()
    return t, max(1, t.numel() // t.shape[-1]), 0, t.shape[-1]


# --------------------------------------------------------------------------------------
# distillation
# --------------------------------------------------------------------------------------
def _stored_teacher(codes, quant, entries):
    """(scales, map, values per scale, bits) of a teacher stored by vectorwise_quant."""
    from .functional import _NONLINEAR_TYPES, _select_qmap, packed_nbytes

    if quant["scale_type"] != "group":
        raise NotImplementedError(f"scale_type {quant['scale_type']!r}: a stored teacher has scales by 'group'")
    if quant["quant_type"] not in _NONLINEAR_TYPES:
        raise ValueError(f"Not support {quant['quant_type']} quant type.")
    bits, scale, group = int(quant["b"]), quant["max1"], int(quant["scaled_shape"][1])
    qmap = _select_qmap(quant)
    if not 4 <= bits <= 8:
        raise NotImplementedError(f"a stored teacher has codes of 4 to 8 bits, got {bits}")
    if group < 1:
        raise ValueError(f"group size need to be a positive integer, but found {group}")
    _require_tensors(max1=scale, qmap=qmap)
    if codes.dtype != torch.int8 or codes.dim() != 1 or not codes.is_contiguous():
        raise RuntimeError("stored teacher_logits must be the contiguous 1-D int8 tensor of vectorwise_quant")
    if scale.dtype != torch.float32 or not scale.is_contiguous() or qmap.dtype != torch.float32 or not qmap.is_contiguous():
        raise RuntimeError("max1 and qmap of a stored teacher must be contiguous float32 tensors")
    if qmap.numel() < 2 ** bits:
        raise RuntimeError(f"{bits}-bit quantisation maps must have {2 ** bits} entries, got {qmap.numel()}")
    if codes.numel() < packed_nbytes(entries, bits) - 1 or scale.numel() < -(-entries // group):
        raise RuntimeError(f"stored teacher_logits hold fewer than the {entries} values that teacher_ids asks for")
    return scale, qmap, group, bits


class _Distill:
    """One call's tensors and the record that the library reads."""

    __slots__ = ("tensors", "device", "shape", "type", "before", "after", "reduction")

    def new_grad(self):
        return torch.empty(self.shape, dtype=self.type, device=self.device)

    def record(self, row_loss, stats, loss, share, grad):
        b, a = self.before, self.after
        return _native.DISTILL_CALL.pack(*b, row_loss, stats, loss, share, grad, *a)


def _distill_call(logits, teacher_logits, teacher_ids, temperature, labels, teacher_weight, label_weight, ignore_index, reduction,
                  teacher_quant):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    temperature = float(temperature)
    if not 1.0 / 1024 <= temperature <= 1024.0:
        raise ValueError(f"temperature must lie within 1/1024 and 1024, got {temperature}")
    teacher_weight, label_weight = _finite(teacher_weight, "teacher_weight"), _finite(label_weight, "label_weight")
    if labels is None and label_weight != 0.0:
        raise ValueError("label_weight needs labels")
    _require_tensors(logits=logits, teacher_logits=teacher_logits, teacher_ids=teacher_ids, labels=labels)
    kind = _type_of(logits, "logits")
    if logits.dim() < 1 or teacher_ids.dim() < 1:
        raise RuntimeError("logits and teacher_ids must have at least one dimension")
    lead, vocab, topk = logits.shape[:-1], logits.shape[-1], teacher_ids.shape[-1]
    if teacher_ids.shape[:-1] != lead:
        raise RuntimeError(f"teacher_ids of shape {tuple(teacher_ids.shape)} do not belong to logits of shape {tuple(logits.shape)}")
    if vocab < 1 or vocab >= 2 ** 31:
        raise RuntimeError(f"logits must have 1 to 2^31 - 1 values in their last dimension, got {vocab}")
    if topk > _native.DISTILL_MOST:
        raise RuntimeError(f"at most {_native.DISTILL_MOST} teacher entries per row are supported, got {topk}")
    if teacher_ids.dtype not in _ID_BITS:
        raise RuntimeError(f"teacher_ids must be int32 or int64, got {teacher_ids.dtype}")
    scale, qmap, group, bits = None, None, 1, 8
    if teacher_quant is not None:
        scale, qmap, group, bits = _stored_teacher(teacher_logits, teacher_quant, teacher_ids.numel())
        teacher_kind = _native.TYPE_CODES
    else:
        if teacher_logits.shape != teacher_ids.shape:
            raise RuntimeError(f"teacher_logits of shape {tuple(teacher_logits.shape)} do not belong to teacher_ids of shape "
                               f"{tuple(teacher_ids.shape)}")
        teacher_kind = _type_of(teacher_logits, "teacher_logits")
    if labels is not None:
        if labels.dtype != torch.int64:
            raise RuntimeError(f"labels must be int64, got {labels.dtype}")
        if labels.shape != lead:
            raise RuntimeError(f"labels of shape {tuple(labels.shape)} do not belong to logits of shape {tuple(logits.shape)}")
    call = _Distill()
    call.device = _require_cuda(logits=logits, teacher_logits=teacher_logits, teacher_ids=teacher_ids, labels=labels, max1=scale, qmap=qmap)
    call.shape, call.type = logits.shape, logits.dtype
    logits, inner, outer_stride, inner_stride = _row_strides(logits.detach())
    teacher_logits, teacher_ids = teacher_logits.detach().contiguous(), teacher_ids.contiguous()
    labels = None if labels is None else labels.contiguous()
    call.tensors = (logits, teacher_logits, teacher_ids, labels, scale, qmap)
    call.reduction = _REDUCTIONS[reduction]
    call.before = (logits.data_ptr(), teacher_logits.data_ptr(), _ptr(scale), _ptr(qmap), teacher_ids.data_ptr(), _ptr(labels))
    call.after = (math.prod(lead), vocab, topk, inner, outer_stride, inner_stride, group, int(ignore_index), temperature, teacher_weight,
                  label_weight, kind, teacher_kind, _ID_BITS[teacher_ids.dtype], call.reduction, bits)
    return call


def _distill_forward(call, keep, grad):
    """The loss, and the work array that the gradient call needs (rows' statistics, share, rows' losses)."""
    rows = call.after[0]
    none = call.reduction == _native.REDUCE_NONE
    loss = torch.empty(call.shape[:-1] if none else (), dtype=torch.float32, device=call.device)
    stats_len = 4 * rows if keep else 0
    work = torch.empty(stats_len + 1 + (0 if none else rows), dtype=torch.float32, device=call.device)
    at = work.data_ptr()
    share, row_loss = at + 4 * stats_len, at + 4 * stats_len + 4
    record = call.record(loss.data_ptr() if none else row_loss, at if keep else 0, 0 if none else loss.data_ptr(), share, _ptr(grad))
    with torch.cuda.device(call.device):
        st = _native.lib().lpmm_distill_loss(record, _native.current_stream(call.device))
    _native.check(st, "distill_loss")
    return loss, work


class _DistillLoss(torch.autograd.Function):
    """The gradient of a reduced loss is written by the pass that computes the loss, while the row's logits are at hand, for the
    gradient 1 that `loss.backward()` starts from; a backward pass that arrives with another value writes it again from
    the logits.  float16 training scales its loss as a rule, so there (and for the losses of single rows) only the backward
    pass writes it."""

    @staticmethod
    def forward(ctx, logits, call):
        grad = call.new_grad() if call.reduction != _native.REDUCE_NONE and call.type != torch.float16 else None
        loss, work = _distill_forward(call, True, grad)
        ctx.save_for_backward(work, *call.tensors)
        call.tensors = None  # the graph's from here on, which lets go of them after the backward pass
        ctx.call, ctx.grad = call, grad
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        work = ctx.saved_tensors[0]  # also checks that no input was written over since
        call, grad, ctx.grad = ctx.call, ctx.grad, None
        made = grad is not None  # handed out once: a second pass over the graph gets a gradient of its own
        if grad is None:
            grad = call.new_grad()
        stride = 0
        if call.reduction == _native.REDUCE_NONE and any(grad_loss.stride()):
            grad_loss, stride = grad_loss.contiguous(), 1
        at, rows = work.data_ptr(), call.after[0]
        record = call.record(at, at, 0, at + 16 * rows, grad.data_ptr())
        with torch.cuda.device(call.device):
            st = _native.lib().lpmm_distill_loss_grad(record, grad_loss.data_ptr(), stride, made, _native.current_stream(call.device))
        _native.check(st, "distill_loss_grad")
        return grad, None


def distill_loss(logits, teacher_logits, teacher_ids, *, temperature=1.0, labels=None, teacher_weight=1.0, label_weight=0.0,
                 ignore_index=-100, reduction="mean", teacher_quant=None):
    """Distillation from a teacher's top logits, differentiable in `logits`.

    logits: (..., V) float32, float16 or bfloat16; views such as `logits[:, :-1]` are read in place.
    teacher_logits, teacher_ids: (..., K), the teacher's K largest logits of each position and where in the vocabulary they
    are (int32 or int64), K at most 1024, in any order.  A negative id marks an empty entry.  The values are float32, float16 or
    bfloat16, or stored by `vectorwise_quant` with scale_type 'group' and 4 to 8 bits: then teacher_logits is
    the int8 tensor it returned and teacher_quant the keywords with which `vectorwise_dequant` gives the values back.
    labels: (...) int64, optional.

    With T the temperature, q = softmax(logits / T) and p = softmax(teacher_logits / T) over a row's entries, the loss of a row is

        teacher_weight * T^2 * sum_k p_k (log p_k - log q[id_k])  +  label_weight * cross_entropy(logits, label)

    A row without entries (or with values of -infinity only) has the second term alone; a term of weight 0 is not looked at.  Rows whose
    label is ignore_index take no part: loss and gradient are 0 whatever they hold, and 'mean' divides by the number of
    the other rows (the mean of no rows is 0).  An id that occurs several times in a row counts with the sum of its
    probabilities.  Nothing is copied to the host to be checked: an id of V or more, a label outside [0, V) that is not
    ignore_index, and teacher values of NaN or +infinity make the loss and the gradient of their row NaN.

    Returns a float32 tensor: a scalar for reduction 'mean' or 'sum', (...) for 'none'.  No gradient flows to the teacher.  With
    'mean' and 'sum' factors are best put into the two weights: the gradient is then made along with the loss, while a loss
    that is multiplied afterwards has it written once more."""
    call = _distill_call(logits, teacher_logits, teacher_ids, temperature, labels, teacher_weight, label_weight, ignore_index, reduction,
                         teacher_quant)
    if logits.requires_grad and torch.is_grad_enabled():
        return _DistillLoss.apply(logits, call)
    return _distill_forward(call, False, None)[0]


# --------------------------------------------------------------------------------------
# balance of experts
# --------------------------------------------------------------------------------------
class _Balance:
    """One call's tensors and the record that the library reads."""

    __slots__ = ("tensors", "device", "shape", "type", "sizes", "tail")

    def record(self, rows, ids, mask, loss, counts, factors, work, grad):
        return _native.BALANCE_CALL.pack(rows.data_ptr(), _ptr(ids), _ptr(mask), _ptr(loss), _ptr(counts), factors.data_ptr(), _ptr(work),
                                         _ptr(grad), *self.sizes, *self.tail)


def _balance_forward(call):
    groups, tokens, experts = call.sizes[:3]
    loss = torch.empty((), dtype=torch.float32, device=call.device)
    counts = torch.empty(call.shape[:-2] + (experts,), dtype=torch.int64, device=call.device)
    factors = torch.empty(groups * (experts + 2), dtype=torch.float32, device=call.device)
    lib = _native.lib()
    work = torch.empty(lib.lpmm_balance_work_bytes(groups, tokens, experts), dtype=torch.uint8, device=call.device)
    record = call.record(*call.tensors, loss, counts, factors, work, None)
    with torch.cuda.device(call.device):
        st = lib.lpmm_balance_loss(record, _native.current_stream(call.device))
    _native.check(st, "balance_loss")
    return loss, counts, factors


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, router_logits, call):
        loss, counts, factors = _balance_forward(call)
        rows, _, mask = call.tensors
        ctx.save_for_backward(rows, mask, factors)
        call.tensors = None
        ctx.call = call
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None
        rows, mask, factors = ctx.saved_tensors
        call = ctx.call
        grad = torch.empty(call.shape, dtype=call.type, device=call.device)
        record = call.record(rows, None, mask, None, None, factors, None, grad)
        with torch.cuda.device(call.device):
            st = _native.lib().lpmm_balance_loss_grad(record, grad_loss.data_ptr(), _native.current_stream(call.device))
        _native.check(st, "balance_loss_grad")
        return grad, None


def balance_loss(router_logits, expert_ids, *, mask=None, weight=1.0, z_weight=0.0):
    """Loss that spreads a router's tokens over its experts, differentiable in `router_logits`, and the experts' counts.

    router_logits: (N, E) float32, float16 or bfloat16, or (G, N, E) for G groups (sequences, layers) that are balanced each by
    itself; E at most 1024.  expert_ids: (..., k) int32 or int64, the experts that each token goes to; a negative id
    is no pick (a token that was dropped).  mask: (...) bool, the tokens that take part.

    With p = softmax(router_logits), T a group's tokens that take part and c_e the picks of expert e among them, the loss is the mean
    over the groups of

        weight * E * sum_e c_e / (T k) * mean_n p_ne  +  z_weight * mean_n logsumexp(router_logits_n)^2

    1 times `weight` where both picks and probabilities are even.  The counts are constants to the gradient.  A group without tokens
    has loss 0.  An id of E or more makes the loss and its group's gradient NaN.

    Returns (loss, counts): a float32 scalar and the int64 counts, (E,) or (G, E)."""
    weight, z_weight = _finite(weight, "weight"), _finite(z_weight, "z_weight")
    _require_tensors(router_logits=router_logits, expert_ids=expert_ids, mask=mask)
    kind = _type_of(router_logits, "router_logits")
    if router_logits.dim() not in (2, 3):
        raise RuntimeError(f"router_logits must be (tokens, experts) or (groups, tokens, experts), got {tuple(router_logits.shape)}")
    if expert_ids.dim() != router_logits.dim() or expert_ids.shape[:-1] != router_logits.shape[:-1]:
        raise RuntimeError(f"expert_ids of shape {tuple(expert_ids.shape)} do not belong to router_logits of shape "
                           f"{tuple(router_logits.shape)}")
    if expert_ids.dtype not in _ID_BITS:
        raise RuntimeError(f"expert_ids must be int32 or int64, got {expert_ids.dtype}")
    lead = router_logits.shape[:-2]
    tokens, experts, picks = router_logits.shape[-2], router_logits.shape[-1], expert_ids.shape[-1]
    if not 1 <= experts <= _native.BALANCE_MOST:
        raise RuntimeError(f"1 to {_native.BALANCE_MOST} experts are supported, got {experts}")
    if picks > experts:
        raise RuntimeError(f"{picks} picks of {experts} experts")
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != router_logits.shape[:-1]:
            raise RuntimeError(f"mask must be a bool tensor of shape {tuple(router_logits.shape[:-1])}, got {mask.dtype} of shape "
                               f"{tuple(mask.shape)}")
    call = _Balance()
    call.device = _require_cuda(router_logits=router_logits, expert_ids=expert_ids, mask=mask)
    call.shape, call.type = router_logits.shape, router_logits.dtype
    rows = router_logits.detach()
    if rows.stride(-1) != 1 and experts > 1:
        rows = rows.contiguous()
    call.tensors = (rows, expert_ids.contiguous(), None if mask is None else mask.contiguous())
    call.sizes = (lead[0] if lead else 1, tokens, experts, picks, rows.stride(0) if lead else 0, rows.stride(-2))
    call.tail = (weight, z_weight, kind, _ID_BITS[expert_ids.dtype])
    if router_logits.requires_grad and torch.is_grad_enabled():
        return _BalanceLoss.apply(router_logits, call)
    return _balance_forward(call)[:2]
