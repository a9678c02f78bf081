"""The training-loss terms from their definitions, in 64 bits on the CPU, with the magnitudes their rounding errors scale with.

Every function returns values and, beside each, a bound on what 32-bit arithmetic may add to it.  U = 2^-24 is half a step of
float32 relative to the value; the bounds count roundings along the longest path and are not fitted to any result."""
import math
import struct

import torch

# the library's calls (lpmm_distill_call, lpmm_balance_call), and its names for types and reductions
DISTILL_CALL = struct.Struct("<11Q8q3f5i")
BALANCE_CALL = struct.Struct("<8Q6q2f2i")
TYPE_F32, TYPE_F16, TYPE_BF16, TYPE_CODES = range(4)
REDUCE_NONE, REDUCE_SUM, REDUCE_MEAN = range(3)

U = 2.0 ** -24
TINY = 2.0 ** -126  # an exponential below the smallest normal float32 is 0, in the kernels and on the hardware: an absolute error of at most this
SMALLEST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step of the smallest numbers


def step(dtype):
    """Half a step of `dtype` relative to the value; float32 results carry it in the bounds already."""
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def _softmax(z):
    """(softmax, log of the sum after the largest value is taken off, differences to the largest value)"""
    d = z - z.amax(dim=-1, keepdim=True)
    s = torch.exp(d).sum(dim=-1, keepdim=True)
    return torch.exp(d) / s, torch.log(s), d


def _sum_error(q, d, vocab):
    """Relative error of a sum of vocab exponentials: every term's argument has three roundings (difference, constant, product) of
    |d| each and the exponential itself is off by two half steps; the additions: vocab / 512 in a thread's own sum, which is
    rescaled as often as its largest value grows (at most once for every 4 values), then 6 + 8 to join threads and waves."""
    arguments = (q * d.abs().nan_to_num(posinf=0.0)).sum(dim=-1, keepdim=True)
    return U * (3 * arguments + 2 + vocab / 512 * 1.25 + 16 + 3)


def distill(logits, teacher, ids, temperature=1.0, labels=None, wt=1.0, wl=0.0, ignore=-100, reduction="mean", grad_loss=None):
    """(loss, its bound, gradient for grad_loss, its bound); float64, bounds without the output's own rounding."""
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    rows, topk = math.prod(lead), ids.shape[-1]
    x, t, i = logits.double().reshape(rows, vocab), teacher.double().reshape(rows, topk), ids.reshape(rows, topk)
    y = None if labels is None else labels.reshape(rows)
    counts = torch.ones(rows, dtype=torch.bool) if y is None else y != ignore
    loss, bound = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    grad, gbound = torch.zeros_like(x), torch.zeros_like(x)
    for n in range(rows):
        if not counts[n]:
            continue
        held = i[n] >= 0
        tn, at = t[n][held], i[n][held]
        if wt != 0 and tn.numel() and tn.max() > -math.inf:
            q, log_s, d = _softmax(x[n] / temperature)
            e_s = _sum_error(q, d, vocab)
            p, log_total, td = _softmax(tn / temperature)
            terms = torch.where(p > 0, p * (torch.where(p > 0, td, 0.0) - log_total - d[at] + log_s), 0.0)
            # log p: difference, scaling, logarithm of a sum of at most 1024 terms; p itself: the same through the exponential
            e_p = U * (4 * td.abs().nan_to_num(posinf=0.0) + 24)
            size = torch.where(p > 0, p * (td.abs().nan_to_num(posinf=0.0) + log_total.abs() + d[at].abs().nan_to_num(posinf=0.0) + log_s.abs()), 0.0)
            loss[n] += wt * temperature ** 2 * terms.sum()
            bound[n] += abs(wt) * temperature ** 2 * (U * 32 * size.sum() + e_s.squeeze(-1) + (e_p * size).sum() + (U * 24 * p).sum())
            grad[n] += wt * temperature * q
            grad[n].index_add_(0, at, -wt * temperature * p)
            gbound[n] += abs(wt) * temperature * (q * (U * (3 * d.abs().nan_to_num(posinf=0.0) + 8) + e_s) + TINY)
            gbound[n].index_add_(0, at, abs(wt) * temperature * (p * (e_p + U * 8) + TINY))
        if y is not None and wl != 0:
            q, log_s, d = _softmax(x[n])
            e_s = _sum_error(q, d, vocab)
            loss[n] += wl * (log_s.squeeze(-1) - d[y[n]])
            bound[n] += abs(wl) * (U * 8 * (log_s.abs().squeeze(-1) + d[y[n]].abs()) + e_s.squeeze(-1))
            grad[n] += wl * q
            grad[n, y[n]] -= wl
            gbound[n] += abs(wl) * (q * (U * (3 * d.abs().nan_to_num(posinf=0.0) + 8) + e_s) + TINY)
            gbound[n, y[n]] += abs(wl) * U * 8
    share = 1.0
    if reduction == "mean":
        share = 1.0 / max(1, int(counts.sum()))
    g = torch.full((rows,), 1.0, dtype=torch.float64)
    if grad_loss is not None:
        g = grad_loss.double().reshape(-1).expand(rows) if rows else g
    grad, gbound = grad * (g * share).unsqueeze(1), gbound * (g * share).abs().unsqueeze(1) + 4 * U * (grad * (g * share).unsqueeze(1)).abs()
    if reduction == "none":
        return loss.view(lead), bound.view(lead) + 4 * U * loss.abs().view(lead), grad.view(logits.shape), gbound.view(logits.shape)
    return (loss * share).sum(), (bound * share).sum() + 4 * U * (loss * share).abs().sum(), grad.view(logits.shape), gbound.view(logits.shape)


def balance(logits, ids, mask=None, weight=1.0, z_weight=0.0, grad_loss=1.0):
    """(loss, its bound, counts, gradient for grad_loss, its bound)"""
    shape, experts, picks = logits.shape, logits.shape[-1], ids.shape[-1]
    groups, tokens = math.prod(shape[:-2]), shape[-2]
    r = logits.double().reshape(groups, tokens, experts)
    i = ids.reshape(groups, tokens, picks)
    seen = torch.ones(groups, tokens, dtype=torch.bool) if mask is None else mask.reshape(groups, tokens)
    loss, bound = 0.0, 0.0
    counts = torch.zeros(groups, experts, dtype=torch.int64)
    grad, gbound = torch.zeros_like(r), torch.zeros_like(r)
    for g in range(groups):
        rows = r[g][seen[g]]
        T = rows.shape[0]
        picked = i[g][seen[g]].reshape(-1)
        counts[g] = torch.bincount(picked[picked >= 0], minlength=experts)[:experts]
        if T == 0:
            continue
        p, log_s, d = _softmax(rows)
        lse = (log_s + rows.amax(dim=-1, keepdim=True)).squeeze(-1)
        size = d.abs().nan_to_num(posinf=0.0)
        # a probability: three roundings of |d| in the argument, the exponential, a sum over at most 1024 experts (16 in a lane, 6 exchanges),
        # the reciprocal, the product
        e_s = U * (3 * (p * size).sum(dim=-1, keepdim=True) + 26)
        e_p = p * (U * (3 * size + 6) + e_s) + TINY
        share = weight * experts * counts[g].double() / (T * T * max(1, picks))
        # sums over tokens: a thread adds every fourth of its group's at most, then waves are joined (70 at most); the rest is in 64 bits
        e_sum = U * (T / 4 + 70)
        # logsumexp: the logarithm, the addition of the largest value
        e_lse = e_s.squeeze(-1) + U * 4 * (lse.abs() + rows.amax(dim=-1).abs() + log_s.squeeze(-1).abs())
        loss += ((share * p.sum(dim=0)).sum() + z_weight * (lse ** 2).sum() / T) / groups
        bound += ((share.abs() * (e_p.sum(dim=0) + e_sum * p.sum(dim=0))).sum() + abs(z_weight) * (2 * lse.abs() * e_lse).sum() / T) / groups
        f, h = share / groups, 2 * z_weight / (T * groups)
        dot = (f * p).sum(dim=-1, keepdim=True)
        e_dot = (f.abs() * (e_p + 26 * U * p)).sum(dim=-1, keepdim=True)
        inner = f - dot + h * lse.unsqueeze(1)
        e_inner = 4 * U * (f.abs() + dot.abs() + (h * lse.unsqueeze(1)).abs()) + e_dot + abs(h) * e_lse.unsqueeze(1)
        grad[g][seen[g]] = grad_loss * p * inner
        gbound[g][seen[g]] = abs(grad_loss) * (e_p * inner.abs() + p * e_inner + 4 * U * (p * inner).abs())
    loss = torch.as_tensor(loss, dtype=torch.float64)
    bound = torch.as_tensor(bound, dtype=torch.float64) + 4 * U * loss.abs()
    return loss, bound, counts.view(shape[:-2] + (experts,)), grad.view(shape), gbound.view(shape)


def assert_within(got, want, bound, what, dtype=None):
    """got within `bound` of want, plus half a step of got's type; infinities and NaN have to be the same."""
    dtype = got.dtype if dtype is None else dtype
    g, w = got.detach().cpu().double(), want
    assert g.shape == w.shape, f"{what}: {tuple(g.shape)} for {tuple(w.shape)}"
    w = torch.where(w.abs() > torch.finfo(dtype).max, w * math.inf, w)  # past the type's largest number its rounding is infinity
    fine = torch.isfinite(w)
    assert torch.equal(fine, torch.isfinite(g)), f"{what}: finite values differ in place"
    assert torch.equal(torch.isnan(w), torch.isnan(g)) and torch.equal(w[~fine].nan_to_num(1.0), g[~fine].nan_to_num(1.0)), f"{what}: infinities"
    far = (g - w).abs() - (bound + step(dtype) * (w.abs() + bound) + SMALLEST[dtype])
    far = torch.where(fine, far, 0.0)
    worst = far.reshape(-1).argmax() if far.numel() else 0
    assert not far.numel() or far.max() <= 0, (f"{what}: {g.reshape(-1)[worst]:.9g} for {w.reshape(-1)[worst]:.9g}, bound {bound.reshape(-1)[worst]:.3g}, "
                                              f"at {int(worst)}; {int((far > 0).sum())} of {far.numel()}")
