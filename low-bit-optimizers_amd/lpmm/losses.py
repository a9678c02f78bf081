"""Terms of a training loss with their gradients: distillation from a teacher's top logits (with the label's cross entropy
from the same pass) and the balance of a router's experts.

The reference has no counterpart.  The optimizers end a training step; these stand where its gradients begin, and a
teacher's values may come in the block-wise codes in which the optimizers keep their states
(`lpmm.functional.vectorwise_quant`).  The kernels are in liblpmm_hip.so, their host side in lpmm/_losses.so; there is no
CPU or PyTorch fallback.  Work is enqueued on torch's current stream of the tensors' device, nothing waits for the GPU,
and a call can be recorded into a graph.  Inside `torch.compile` a call runs as it is, between two compiled parts.  Tracers
(`torch.jit.trace`, `make_fx`, fake tensors) and forward-mode derivatives are refused.
"""
import torch

from . import _native

__all__ = ["balance_loss", "distill_loss"]

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}  # LPMM_REDUCE_*


def _require_tensors(**tensors):
    for name, t in tensors.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")


def _stored_teacher(quant):
    """(scales, map, values per scale, bits) of a teacher stored by vectorwise_quant."""
    from .functional import _NONLINEAR_TYPES, _select_qmap

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
    for name, t in (("max1", scale), ("qmap", qmap)):
        if not isinstance(t, torch.Tensor):  # None too: a stored teacher has both
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    return scale, qmap, group, bits


def distill_loss(logits, teacher_logits, teacher_ids, *, temperature=1.0, labels=None, teacher_weight=1.0, label_weight=0.0,
                 ignore_index=-100, reduction="mean", teacher_quant=None):
    """Distillation from a teacher's top logits, differentiable in `logits`.

    logits: (..., V) float32, float16 or bfloat16, fewer than 2^31 rows; views are read in place.  For next tokens pass whole logits and
    shifted labels whose last one is ignore_index: `logits[:, :-1]` is the same loss, but the slice's backward pass writes all of
    the gradient twice more (4 x 2048 x 32000 bf16: 504 us for loss and gradient, 199 from whole logits).
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
    ignore_index (whatever its weight), and teacher values of NaN or +infinity make the loss and the gradient of their row NaN.

    Returns a float32 tensor: a scalar for reduction 'mean' or 'sum', (...) for 'none'.  No gradient flows to the teacher.  With
    'mean' and 'sum' factors are best put into the two weights: the gradient of float32 and bfloat16 logits is then made along with the
    loss, while a loss that is multiplied afterwards has it written once more (378 us instead of 199)."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    scale, qmap, group, bits = (None, None, 1, 8) if teacher_quant is None else _stored_teacher(teacher_quant)
    native = _native.losses()
    try:
        return native.distill_loss(logits, teacher_logits, teacher_ids, temperature, labels, teacher_weight, label_weight, ignore_index,
                                   _REDUCTIONS[reduction], scale, qmap, group, bits)
    except TypeError:
        _require_tensors(logits=logits, teacher_logits=teacher_logits, teacher_ids=teacher_ids, labels=labels)
        raise


def balance_loss(router_logits, expert_ids, *, mask=None, weight=1.0, z_weight=0.0):
    """Loss that spreads a router's tokens over its experts, differentiable in `router_logits`, and the experts' counts.

    router_logits: (N, E) float32, float16 or bfloat16, or (G, N, E) for G groups (sequences, layers) that are balanced each by
    itself; E at most 1024, G at most 65535, G N at most 2^28.  expert_ids: (..., k) int32 or int64, the experts that each
    token goes to, k at most E, N k below 2^31; a negative id is no pick (a token that was dropped).  mask: (...) bool, the tokens that take part.

    With p = softmax(router_logits), T a group's tokens that take part and c_e the picks of expert e among them, the loss is the mean
    over the groups of

        weight * E * sum_e c_e / (T k) * mean_n p_ne  +  z_weight * mean_n logsumexp(router_logits_n)^2

    1 times `weight` where both picks and probabilities are even.  The counts are constants to the gradient.  A group without tokens
    has loss 0.  An id of E or more makes the loss and its group's gradient NaN.

    Returns (loss, counts): a float32 scalar and the int64 counts, (E,) or (G, E)."""
    native = _native.losses()
    try:
        return native.balance_loss(router_logits, expert_ids, mask, weight, z_weight)
    except TypeError:
        _require_tensors(router_logits=router_logits, expert_ids=expert_ids, mask=mask)
        raise
