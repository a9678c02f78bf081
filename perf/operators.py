"""The terms of a training loss that the package computes beside its optimizer steps, as they are measured.

A pass is what a training loop does at its loss once per step: the loss of a batch and its gradient with respect to
the logits; or, where a model is evaluated, the loss of every token.  `prepare` makes what the model and the data
loader have left by then, `run` is the loss call and the backward pass through it.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100  # label of prompt and padding tokens
GROUP = 128  # values per scale of stored teacher logits
HALF_SCALE = 8192.0  # training in half precision scales its loss, so that small gradients do not vanish


# ---- cases -------------------------------------------------------------------------------------
def _distill(name=None, *, batch, seq, vocab, topk, dtype="bf16", temperature=1.0, labels=True, shift=False, bits=0, train=True):
    case = dict(op="distill", batch=batch, seq=seq, vocab=vocab, topk=topk, dtype=dtype, temperature=temperature, labels=labels,
                shift=shift, bits=bits, train=train)
    return dict(case, name=name) if name else case


def _balance(name=None, *, groups=0, tokens, experts, picks, dtype="fp32", mask=False, z_weight=0.0):
    case = dict(op="balance", groups=groups, tokens=tokens, experts=experts, picks=picks, dtype=dtype, mask=mask, z_weight=z_weight)
    return dict(case, name=name) if name else case


def listed():
    return [
        # fine-tuning on four sequences of 2048 tokens with a 32000-entry vocabulary, each position's logits against the
        # next token: the views that a causal model's loss takes of its logits, and the largest case
        _distill("distill_causal_lm", batch=4, seq=2048, vocab=32000, topk=64, temperature=2.0, shift=True),
        # a vocabulary of 50257, whose rows start at any even address, in half precision; the teacher alone
        _distill("distill_odd_vocab", batch=2, seq=1024, vocab=50257, topk=50, dtype="fp16", labels=False),
        # a model trained in single precision
        _distill("distill_fp32", batch=1, seq=2048, vocab=32000, topk=128, dtype="fp32", temperature=1.5),
        # a large multilingual vocabulary
        _distill("distill_long_vocab", batch=2, seq=1024, vocab=131072, topk=256),
        # the teacher's values come from disk in 8-bit codes, one scale per 128
        _distill("distill_stored_8bit", batch=4, seq=1000, vocab=50257, topk=100, temperature=2.0, bits=8),
        # evaluation against a teacher stored in 4-bit codes: the loss of every token, no gradient
        _distill("distill_eval_4bit", batch=4, seq=1024, vocab=32000, topk=64, bits=4, train=False),
        # the last tokens of one sequence: fewer rows than the card has compute units
        _distill("distill_few_rows", batch=1, seq=24, vocab=50257, topk=32, temperature=2.0),
        # a test model's batch, where launches and host work are what a call costs
        _distill("distill_small", batch=1, seq=16, vocab=8192, topk=8),
        # a layer of 256 experts on 65536 tokens, padding masked, with the penalty on large router logits
        _balance("balance_large", tokens=65536, experts=256, picks=8, mask=True, z_weight=0.001),
        # an ordinary layer
        _balance("balance_ordinary", tokens=8192, experts=64, picks=2, dtype="bf16"),
        # balance within each sequence, of odd length, with an expert count that is no power of two
        _balance("balance_sequences", groups=16, tokens=1023, experts=60, picks=4, mask=True),
        # a test model's layer
        _balance("balance_small", tokens=16, experts=8, picks=2, z_weight=0.001),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.6:
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        vocab = _log_int(rng, 1000, 131072)
        if rng.random() < 0.5:
            vocab = max(1, vocab // 64) * 64
        most = 4 * 2047 * 32000 * 2 // (vocab * (4 if dtype == "fp32" else 2))  # no more than distill_causal_lm
        rows = _log_int(rng, 8, min(8192, most))
        batch = rng.choice([b for b in (1, 2, 3, 4) if b * 4 <= rows])
        return _distill(batch=batch, seq=rows // batch, vocab=vocab, topk=_log_int(rng, 1, 256), dtype=dtype,
                        temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), labels=rng.random() < 0.6, shift=rng.random() < 0.4,
                        bits=rng.choice([0, 0, 4, 8]), train=rng.random() < 0.75)
    experts = _log_int(rng, 4, 256)
    tokens = _log_int(rng, 16, 65536)
    groups = rng.choice([0, 0, rng.randint(1, 32)])
    if groups:
        tokens = max(1, tokens // groups)
    return _balance(groups=groups, tokens=tokens, experts=experts, picks=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), mask=rng.random() < 0.5, z_weight=rng.choice([0.0, 0.001]))


# ---- inputs ------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rows(case):
    return case["batch"] * (case["seq"] - 1 if case["shift"] else case["seq"])


def _store(values, bits):
    """Values in the package's stored form: blocks of 128 with the largest magnitude as scale, codes of a linear map."""
    n = values.numel()
    padded = torch.zeros(-(-n // 2048) * 2048, device=values.device)
    padded[:n] = values.reshape(-1)
    blocks = padded.view(-1, GROUP)[: -(-n // GROUP)]
    scale = blocks.abs().amax(dim=1, keepdim=True)
    qmap = torch.linspace(-1, 1, 2 ** bits).to(values.device)
    normal = torch.zeros_like(padded).view(-1, GROUP)
    normal[: blocks.shape[0]] = blocks / scale.clamp(min=1e-30)
    code = ((normal + 1) * (0.5 * (2 ** bits - 1))).round().to(torch.int64).clamp(0, 2 ** bits - 1).view(-1)
    if bits == 4:
        code = code[0::2] + 16 * code[1::2]
    codes = torch.cat([code, code.new_zeros(1)]).to(torch.uint8).view(torch.int8)
    return dict(codes=codes, scale=scale, qmap=qmap)


def _prepare_distill(case, seed):
    g = _generator(seed)
    dtype, vocab, topk, rows = DTYPES[case["dtype"]], case["vocab"], case["topk"], _rows(case)
    seq = case["seq"] - 1 if case["shift"] else case["seq"]
    top = (case["batch"], seq, topk)
    full = torch.randn(case["batch"], case["seq"], vocab, device="cuda", dtype=dtype, generator=g).mul_(2.5)
    # distinct entries anywhere in the vocabulary, the teacher's values from the largest down; a tenth of the rows has fewer
    # entries (a nucleus of the teacher's probabilities), some none (positions the teacher has not seen)
    step = (torch.rand(rows, 1, device="cuda", generator=g) * (vocab // topk)).long().clamp(1, max(1, vocab // topk))
    base = (torch.rand(rows, 1, device="cuda", generator=g) * vocab).long()
    ids = (base + step * torch.arange(topk, device="cuda")) % vocab
    held = (torch.rand(rows, 1, device="cuda", generator=g) * (topk + 1)).long()
    held = torch.where(torch.rand(rows, 1, device="cuda", generator=g) < 0.1, held, topk)
    ids = ids.masked_fill(torch.arange(topk, device="cuda") >= held, -1).view(top)
    values = (torch.randn(rows, topk, device="cuda", generator=g) * 3 + 12).sort(dim=1, descending=True).values.view(top)
    logits = full[:, :-1] if case["shift"] else full
    logits.scatter_add_(2, ids.clamp(min=0), (ids >= 0).to(dtype) * 5)  # the student has learnt some of it
    state = dict(case=case, logits=logits.detach().requires_grad_(case["train"]), labels=None)
    if case["labels"]:
        labels = (torch.rand(case["batch"], seq, device="cuda", generator=g) * vocab).long().clamp(max=vocab - 1)
        state["labels"] = labels.masked_fill(torch.rand(case["batch"], seq, device="cuda", generator=g) < 0.1, IGNORE)
    if case["bits"]:
        state["stored"] = _store(values - values[..., :1], case["bits"])
        state["ids"] = ids.int()
    else:
        state["values"] = values.to(dtype)
        state["ids"] = ids
    return state


def _prepare_balance(case, seed):
    g = _generator(seed)
    lead = (case["groups"], case["tokens"]) if case["groups"] else (case["tokens"],)
    liked = torch.randn(case["experts"], device="cuda", generator=g)  # experts are not liked alike
    logits = (torch.randn(*lead, case["experts"], device="cuda", generator=g) * 1.5 + liked).to(DTYPES[case["dtype"]])
    ids = logits.float().topk(case["picks"], dim=-1).indices
    ids = ids.masked_fill(torch.rand(ids.shape, device="cuda", generator=g) < 0.02, -1)  # dropped: the expert was full
    state = dict(case=case, logits=logits.requires_grad_(True), ids=ids, mask=None)
    if case["mask"]:
        length = (torch.rand(*lead[:-1], 1, device="cuda", generator=g) * 0.5 + 0.5) * case["tokens"]
        state["mask"] = (torch.arange(case["tokens"], device="cuda") < length).view(lead)
    return state


def prepare(case, seed):
    return _prepare_distill(case, seed) if case["op"] == "distill" else _prepare_balance(case, seed)


# ---- the package's calls -----------------------------------------------------------------------
def _package():
    path = os.path.join(os.getcwd(), "low-bit-optimizers_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import lpmm.functional

    return lpmm.functional


def _gradient(loss, s):
    scaled = loss * HALF_SCALE if s["case"]["dtype"] == "fp16" else loss
    return torch.autograd.grad(scaled, s["logits"])[0]


def _own_distill(s):
    case, stored = s["case"], s.get("stored")
    values, quant = s.get("values"), None
    if stored:
        values = stored["codes"]
        quant = dict(b=case["bits"], signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", qmap=stored["qmap"],
                     max1=stored["scale"], scaled_shape=torch.Size((stored["scale"].shape[0], GROUP)), dtype=torch.float32, stride=None)
    loss = _package().distill_loss(s["logits"], values, s["ids"], temperature=case["temperature"], labels=s["labels"], teacher_weight=0.5,
                                   label_weight=0.5 if case["labels"] else 0.0, ignore_index=IGNORE,
                                   reduction="mean" if case["train"] else "none", teacher_quant=quant)
    if not case["train"]:
        return [loss]
    return [loss.detach(), _gradient(loss, s)]


def _own_balance(s):
    loss, counts = _package().balance_loss(s["logits"], s["ids"], mask=s["mask"], weight=0.01, z_weight=s["case"]["z_weight"])
    return [loss.detach(), counts, _gradient(loss, s)]


# ---- the plain forms ---------------------------------------------------------------------------
def _scale(case):
    return HALF_SCALE if case["dtype"] == "fp16" else 1.0


def _teacher(s):
    if "stored" not in s:
        return s["values"].float()
    stored, shape = s["stored"], s["ids"].shape
    code = stored["codes"].view(torch.uint8)[:-1].int()
    if s["case"]["bits"] == 4:
        code = torch.stack([code & 15, code >> 4], dim=1).view(-1)
    code = code[: stored["scale"].numel() * GROUP].view(-1, GROUP)
    return (stored["qmap"][code] * stored["scale"]).view(-1)[: shape.numel()].view(shape)


def _plain_distill(s):
    case, temperature = s["case"], s["case"]["temperature"]
    with torch.no_grad():
        x, ids = s["logits"].float(), s["ids"].long()
        held = ids >= 0
        some = held.any(dim=-1, keepdim=True)
        t = torch.where(held, _teacher(s) / temperature, -math.inf)
        t = torch.where(some, t - t.amax(dim=-1, keepdim=True), -math.inf)
        p = torch.exp(t)
        total = torch.where(some, p.sum(dim=-1, keepdim=True), 1.0)
        p, log_p = p / total, t - torch.log(total)
        x = x - x.amax(dim=-1, keepdim=True)
        z = x / temperature
        q = torch.exp(z)
        norm = q.sum(dim=-1, keepdim=True)
        at = ids.clamp(min=0)
        kd = torch.where(held, p * (log_p - z.gather(-1, at) + torch.log(norm)), 0.0).sum(dim=-1) * temperature ** 2
        loss = 0.5 * kd
        grad = None
        if case["train"]:
            grad = (q / norm * some).scatter_add_(-1, at, -p) * (0.5 * temperature)
        count = ids.shape[0] * ids.shape[1]
        if case["labels"]:
            counts = s["labels"] != IGNORE
            label = s["labels"].clamp(min=0).unsqueeze(-1)
            e = torch.exp(x)
            norm = e.sum(dim=-1, keepdim=True)
            loss = torch.where(counts, loss + 0.5 * (torch.log(norm) - x.gather(-1, label)).squeeze(-1), 0.0)
            count = counts.sum().clamp(min=1)
            if case["train"]:
                grad += 0.5 * (e / norm).scatter_add_(-1, label, torch.full_like(norm, -1.0))
                grad *= counts.unsqueeze(-1)
        if not case["train"]:
            return [loss]
        return [loss.sum() / count, (grad * (_scale(case) / count)).to(s["logits"].dtype)]


def _plain_balance(s):
    case = s["case"]
    with torch.no_grad():
        r, ids, experts, picks = s["logits"].float(), s["ids"], case["experts"], case["picks"]
        if r.dim() == 2:
            r, ids = r.unsqueeze(0), ids.unsqueeze(0)
        groups, tokens = r.shape[:2]
        mask = torch.ones(groups, tokens, dtype=torch.bool, device=r.device) if s["mask"] is None else s["mask"].view(groups, tokens)
        seen = mask.unsqueeze(-1)
        count = mask.sum(dim=1).clamp(min=1).float().view(groups, 1, 1)
        held = (ids >= 0) & seen
        picked = torch.zeros(groups, experts, dtype=torch.int64, device=r.device)
        picked.scatter_add_(1, ids.clamp(min=0).view(groups, -1), held.view(groups, -1).long())
        m = r.amax(dim=-1, keepdim=True)
        e = torch.exp(r - m)
        norm = e.sum(dim=-1, keepdim=True)
        p, lse = e / norm, m + torch.log(norm)
        c = picked.float().unsqueeze(1)
        mean = torch.where(seen, p, 0.0).sum(dim=1, keepdim=True) / count
        loss = 0.01 * experts * (c / (count * picks) * mean).sum(dim=(1, 2))
        loss = loss + case["z_weight"] * (torch.where(seen, lse * lse, 0.0).sum(dim=1, keepdim=True) / count).view(groups)
        grad = 0.01 * experts / (count * count * picks) * p * (c - (c * p).sum(dim=-1, keepdim=True)) + case["z_weight"] * 2 * lse * p / count
        grad = (torch.where(seen, grad, 0.0) * (_scale(case) / groups)).to(s["logits"].dtype)
        return [loss.sum() / groups, picked.view(experts) if s["logits"].dim() == 2 else picked, grad.view(s["logits"].shape)]


def run(state):
    if state["case"]["op"] == "distill":
        return _own_distill(state) if own else _plain_distill(state)
    return _own_balance(state) if own else _plain_balance(state)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    if case["op"] == "distill":
        rows, size = _rows(case), DTYPES[case["dtype"]].itemsize
        values = rows * case["vocab"]
        teacher = rows * case["topk"] * (4 + case["bits"] / 8 + 4 / GROUP if case["bits"] else 8 + size)
        extra = (rows * 8 if case["labels"] else 0) + (4 if case["train"] else rows * 4)
        # a row's largest value, differences, exponentials, sums, then the scaled probabilities
        per_value = (4 if case["temperature"] == 1.0 or not case["labels"] else 7) + (2 if case["train"] else 0)
        return {"bytes": values * size * (2 if case["train"] else 1) + teacher + extra, "flops": values * per_value + rows * case["topk"] * 8}
    rows, size = max(1, case["groups"]) * case["tokens"], DTYPES[case["dtype"]].itemsize
    values = rows * case["experts"]
    return {"bytes": 2 * values * size + rows * case["picks"] * 8 + (rows if case["mask"] else 0) + 8 * max(1, case["groups"]) * case["experts"],
            "flops": values * 10 + rows * case["picks"]}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_teacher(s):
    if "stored" not in s:
        return s["values"].double()
    n, stored = s["ids"].numel(), s["stored"]
    at = torch.arange(n, device="cuda")
    byte = stored["codes"].view(torch.uint8).long()
    code = byte[at] if s["case"]["bits"] == 8 else (byte[at // 2] >> (4 * (at % 2))) & 15
    return (stored["qmap"].double()[code] * stored["scale"].double().view(-1)[at // GROUP]).view(s["ids"].shape)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].detach().double().requires_grad_(True)
    if case["op"] == "distill":
        rows, T = _rows(case), case["temperature"]
        ids = s["ids"].long().view(rows, -1)
        t = _exact_teacher(s).view(rows, -1).masked_fill(ids < 0, -1e300)
        p = (torch.softmax(t / T, dim=-1)).masked_fill(ids < 0, 0.0)
        flat = x.view(rows, -1) if x.is_contiguous() else x.reshape(rows, -1)
        log_q = torch.log_softmax(flat / T, dim=-1).gather(1, ids.clamp(min=0))
        each = 0.5 * T * T * (torch.special.xlogy(p, p) - p * log_q).sum(dim=-1)
        count = rows
        if case["labels"]:
            labels = s["labels"].reshape(rows)
            each = each + 0.5 * torch.nn.functional.cross_entropy(flat, labels, ignore_index=IGNORE, reduction="none")
            each = each * (labels != IGNORE)
            count = max(1, int((labels != IGNORE).sum()))
        if not case["train"]:
            return [each.detach().view(case["batch"], -1)]
        loss = each.sum() / count
        return [loss.detach(), torch.autograd.grad(loss * _scale(case), x)[0]]
    groups = max(1, case["groups"])
    r = x.view(groups, case["tokens"], case["experts"])
    seen = torch.ones(groups, case["tokens"], device="cuda", dtype=torch.float64) if s["mask"] is None else s["mask"].view(groups, -1).double()
    ids = s["ids"].view(groups, case["tokens"], -1)
    spare = torch.where((ids >= 0) & (seen > 0).unsqueeze(-1), ids, case["experts"]).view(groups, -1)
    place = spare + torch.arange(groups, device="cuda").unsqueeze(1) * (case["experts"] + 1)
    counts = torch.bincount(place.view(-1), minlength=groups * (case["experts"] + 1)).view(groups, -1)[:, :-1]
    tokens = seen.sum(dim=1).clamp(min=1)
    mean = (torch.softmax(r, dim=-1) * seen.unsqueeze(-1)).sum(dim=1) / tokens.unsqueeze(1)
    share = counts.double() / (tokens * case["picks"]).unsqueeze(1)
    loss = 0.01 * case["experts"] * (share * mean).sum(dim=1)
    loss = loss + case["z_weight"] * (torch.logsumexp(r, dim=-1) ** 2 * seen).sum(dim=1) / tokens
    loss = loss.mean()
    return [loss.detach(), counts.view(-1) if s["logits"].dim() == 2 else counts, torch.autograd.grad(loss * _scale(case), x)[0]]
