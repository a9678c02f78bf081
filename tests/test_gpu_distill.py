"""distill_loss on the GPU against its definition in 64 bits: types, sizes, masks, strides, gradients, and the ways in which a training
program calls it."""
import math

import pytest
import torch

import lpmm
import lpmm.functional as F
import losses_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(rows, vocab, topk, dtype, seed=0, labels=True, ignored=0.2):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 7919 + vocab * 31 + topk)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    t = torch.randn(rows, topk, generator=g) * 3 + 5
    step = max(1, vocab // max(1, topk))
    ids = (torch.randint(0, vocab, (rows, 1), generator=g) + step * torch.arange(topk)) % vocab
    ids = ids.masked_fill(torch.rand(rows, topk, generator=g) < 0.1, -1)
    y = None
    if labels:
        y = torch.randint(0, vocab, (rows,), generator=g)
        y = y.masked_fill(torch.rand(rows, generator=g) < ignored, -100)
    return x, t, ids, y


def _cuda(t):
    return None if t is None else t.cuda()


def _check(x, t, ids, y, grad_loss=None, what="", move=_cuda, **kw):
    """Loss and gradient of one call against the definition; x etc. on the CPU.  Returns what the GPU gave."""
    leaf = move(x).detach().requires_grad_(True)
    loss = F.distill_loss(leaf, _cuda(t), _cuda(ids), labels=_cuda(y), **kw)
    assert loss.dtype == torch.float32
    loss.backward(gradient=None if grad_loss is None else grad_loss.cuda())
    names = dict(temperature="temperature", teacher_weight="wt", label_weight="wl", ignore_index="ignore", reduction="reduction")
    reduction = kw.get("reduction", "mean")
    if reduction == "none" and grad_loss is None:
        raise AssertionError("the losses of rows need their gradients")
    want, bound, grad, gbound = ref.distill(x, t, ids, labels=y, grad_loss=grad_loss, **{names[k]: v for k, v in kw.items()})
    ref.assert_within(loss, want, bound, what + " loss")
    ref.assert_within(leaf.grad, grad, gbound, what + " gradient")
    plain = F.distill_loss(move(x), _cuda(t), _cuda(ids), labels=_cuda(y), **kw)
    ref.assert_within(plain, want, bound, what + " loss without a gradient")
    return loss.detach(), leaf.grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 64, 65, 255, 511, 1000, 1025, 2047, 4096, 4099, 8192, 16385, 32000, 33001, 50257, 65536, 65543, 131072, 150001])
def test_vocabularies(vocab, dtype):
    x, t, ids, y = _inputs(3, vocab, min(vocab, 20), dtype)
    for temperature, wl in ((1.0, 0.0), (1.0, 0.5), (2.0, 0.5), (1.5, 0.25), (4.0, 0.5)):
        print(dtype, vocab, temperature, wl, flush=True)
        _check(x, t, ids, y if wl else None, temperature=temperature, label_weight=wl, what=f"{vocab} {dtype} T={temperature} wl={wl}")


@pytest.mark.parametrize("topk", [0, 1, 2, 63, 64, 65, 255, 256, 257, 512, 700, 1024])
def test_numbers_of_entries(topk):
    for vocab in (700, 5003):
        for dtype in (torch.bfloat16, torch.float32):
            x, t, ids, y = _inputs(3, vocab, topk, dtype)
            _check(x, t, ids, None, what=f"{topk} of {vocab}")
            _check(x, t, ids.int(), y, temperature=3.0, label_weight=1.0, what=f"{topk} of {vocab} with labels")


@pytest.mark.parametrize("rows", [0, 1, 2, 5, 64, 255, 256, 257, 300, 2500])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_and_reductions(rows, reduction):
    for dtype in (torch.bfloat16, torch.float16):
        x, t, ids, y = _inputs(rows, 67, 6, dtype)
        grad_loss = torch.randn(rows) if reduction == "none" else None
        _check(x, t, ids, y, grad_loss, temperature=2.0, label_weight=0.5, teacher_weight=0.75, reduction=reduction, what=f"{rows} {reduction}")
        _check(x, t, ids, None, grad_loss, reduction=reduction, what=f"{rows} {reduction} without labels")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("teacher", TYPES)
def test_types_of_the_teacher(dtype, teacher):
    x, t, ids, y = _inputs(4, 501, 12, dtype)
    _check(x, t.to(teacher), ids, y, temperature=2.0, label_weight=0.5)


@pytest.mark.parametrize("temperature", [1.0 / 1024, 0.1, 0.5, 1.0, 1.7, 3.0, 8.0, 1024.0])
@pytest.mark.parametrize("wl", [0.0, 0.5])
def test_temperatures(temperature, wl):
    for dtype in TYPES:
        x, t, ids, y = _inputs(4, 301, 9, dtype, seed=5)
        _check(x, t, ids, y, temperature=temperature, label_weight=wl, what=f"{dtype}")


@pytest.mark.parametrize("wt,wl", [(1.0, 0.0), (0.0, 1.0), (0.0, 0.0), (-0.5, 2.0), (1e-3, 1e3)])
def test_weights(wt, wl):
    x, t, ids, y = _inputs(5, 1003, 9, torch.bfloat16, seed=6)
    _check(x, t, ids, y, temperature=2.0, teacher_weight=wt, label_weight=wl)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_gradient_other_than_one(reduction, dtype):
    x, t, ids, y = _inputs(6, 999, 9, dtype, seed=7)
    for scale in (0.25, 1.0, -3.7, 0.0):
        grad_loss = torch.full((6,), scale) if reduction == "none" else torch.tensor(scale)
        _check(x, t, ids, y, grad_loss, temperature=2.0, label_weight=0.5, reduction=reduction, what=f"{scale}")


def test_rows_that_take_no_part_may_hold_anything():
    for dtype in TYPES:
        x, t, ids, y = _inputs(6, 203, 5, dtype, seed=8, ignored=0.0)
        y[1] = y[4] = -100
        x[1], t[1], ids[1] = math.nan, math.nan, 1 << 40
        x[4], t[4] = math.inf, -math.inf
        _check(x, t, ids, y, temperature=2.0, label_weight=0.5)
        _check(x, t, ids, y)  # labels without a weight still say which rows count
        y[:] = -100
        loss, grad = _check(x, t, ids, y, label_weight=0.5)
        assert float(loss) == 0.0 and not grad.any()
        y[:] = 7
        _check(_inputs(6, 203, 5, dtype)[0], t.nan_to_num(1.0, 1.0, 1.0), ids.clamp(max=202), y.masked_fill(y == 7, 300), ignore_index=300)


def test_rows_without_entries():
    for dtype in TYPES:
        x, t, ids, y = _inputs(5, 203, 5, dtype, seed=9, ignored=0.0)
        ids[1] = -1
        t[2] = -math.inf
        ids[3, :3], t[3, 3:] = -1, -math.inf
        t[0, 1] = -math.inf  # one entry of probability 0
        t[0, 2], ids[0, 2] = math.nan, -5  # an empty entry's value is not looked at
        _check(x, t, ids, y, temperature=2.0, label_weight=0.5)
        x[1], x[2] = math.nan, math.inf  # nothing to say of these rows: without labels they may hold anything
        loss, grad = _check(x, t, ids, None, temperature=2.0)
        assert not grad[1].any() and not grad[2].any()


def test_ids_that_occur_several_times():
    for dtype in TYPES:
        for topk in (3, 64, 200, 1000):
            x, t, ids, y = _inputs(4, 1201, topk, dtype, seed=10)
            ids[0] = 17
            ids[1] = ids[1] % 5
            ids[2, topk // 2:] = ids[2, :topk - topk // 2].clone()
            y[0], y[1], y[2] = 17, 3, ids[2].clamp(min=0)[-1]
            got = [_check(x, t, ids, y, temperature=2.0, label_weight=0.5, what=f"{topk}") for _ in range(2)]
            assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][0], got[1][0])


def test_any_negative_id_is_an_empty_entry():
    """Also one whose low 32 bits are the id of an entry behind it, or the label."""
    for dtype in TYPES:
        x, t, ids, y = _inputs(4, 203, 6, dtype, seed=51, ignored=0.0)
        ids[0], y[0] = torch.tensor([-(1 << 32), 0, 9, -1, 4, 2]), 1
        ids[1], y[1] = torch.tensor([-(1 << 32) + 5, -(1 << 40) + 7, 1, 2, 5, 3]), 7
        ids[2] = -(1 << 63)
        _check(x, t, ids, y, temperature=2.0, label_weight=0.5)


def test_what_is_wrong_makes_its_row_nan_and_no_other():
    x, t, ids, y = _inputs(7, 203, 5, torch.bfloat16, seed=11, ignored=0.0)
    good = (x.clone(), t.clone(), ids.clone(), y.clone())
    ids[0, 2] = 203
    ids[1, 0] = (1 << 32) + 3
    t[2, 1], ids[2, 1] = math.nan, 4
    t[3, 1], ids[3, 1] = math.inf, 4
    y[4], y[5] = 203, -1
    leaf = x.cuda().requires_grad_(True)
    loss = F.distill_loss(leaf, t.cuda(), ids.cuda(), labels=y.cuda(), label_weight=0.5, reduction="none")
    loss.backward(torch.ones(7, device="cuda"))
    assert loss[:6].isnan().all() and leaf.grad[:6].isnan().all()
    want, bound, grad, gbound = ref.distill(*(a[6:] for a in good[:3]), labels=good[3][6:], wl=0.5, reduction="none")
    ref.assert_within(loss[6:], want, bound, "the good row")
    ref.assert_within(leaf.grad[6:], grad, gbound, "its gradient")
    leaf.grad = None
    F.distill_loss(leaf, t.cuda(), ids.cuda(), labels=y.cuda(), label_weight=0.5).backward()
    assert leaf.grad[:6].isnan().all() and not leaf.grad[6].isnan().any()
    low = ids.int()
    low[1] = -1
    assert F.distill_loss(x.cuda(), t.cuda(), low.cuda(), reduction="none")[0].isnan()


def test_logits_of_no_softmax_are_nan():
    x, t, ids, y = _inputs(5, 203, 5, torch.float32, seed=12, ignored=0.0)
    ids.clamp_(min=0)
    x[0, 9], x[1], x[2, 7] = math.nan, -math.inf, math.inf
    x[3] = math.nan
    for kw in (dict(), dict(labels=y.cuda(), label_weight=0.5, temperature=2.0)):
        leaf = x.cuda().requires_grad_(True)
        loss = F.distill_loss(leaf, t.cuda(), ids.cuda(), reduction="none", **kw)
        loss.backward(torch.ones(5, device="cuda"))
        assert loss[:4].isnan().all() and leaf.grad[:4].isnan().all() and loss[4].isfinite() and leaf.grad[4].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_vocabulary(dtype):
    """Logits of -infinity and of the type's lowest value have no probability; a row of lowest values is even."""
    lowest = torch.finfo(dtype).min
    x, t, ids, y = _inputs(5, 203, 5, dtype, seed=13, ignored=0.0)
    x[0, 50:] = -math.inf
    x[1, 50:] = lowest
    x[2] = lowest
    x[3] = torch.finfo(dtype).max
    ids[:2] = ids[:2].clamp(min=0) % 50
    y[:2] = y[:2] % 50
    for temperature in (0.25, 1.0, 2.0):
        _check(x, t, ids, y, temperature=temperature, label_weight=0.5)
    t[4] = torch.finfo(torch.float32).min
    t[0, 2:] = torch.finfo(torch.float32).min
    _check(x, t, ids, y, temperature=0.5, label_weight=0.5)
    # the teacher wants what the student cannot give: an infinite loss, a finite gradient
    y[0] = 2
    ids[0, 0] = 60
    loss, grad = _check(x, t, ids, y, torch.ones(5), temperature=2.0, label_weight=0.5, reduction="none")
    assert loss[0] == math.inf and grad[0].isfinite().all()


def test_large_and_close_logits():
    x, t, ids, y = _inputs(4, 1003, 7, torch.float32, seed=14, ignored=0.0)
    x[0] *= 1000
    x[1] = 1e4 + x[1]
    x[2] = 1e-30
    x[3, 5] = 3e38
    _check(x, t, ids, y, torch.ones(4), label_weight=0.5, reduction="none")


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows(dtype):
    x, t, ids, y = _inputs(24, 517, 6, dtype, seed=15)
    full, t, ids, y = x.view(4, 6, 517), t.view(4, 6, 6), ids.view(4, 6, 6), y.view(4, 6)
    kw = dict(temperature=2.0, label_weight=0.5)
    on = full.cuda()
    for name, view in (("shift", lambda a: a[:, :-1]), ("tail", lambda a: a[:, 1:]), ("one", lambda a: a[:, 2]), ("swapped", lambda a: a.transpose(0, 1)),
                       ("row", lambda a: a[3, 4]), ("every second", lambda a: a[:, ::2]), ("whole", lambda a: a)):
        cut = [view(a) for a in (full, t, ids, y)]
        _check(*cut, move=lambda _: view(on), what=name, **kw)
    columns = torch.randn(4, 5, 600, device="cuda").to(dtype)[..., 3:520]
    _check(columns.cpu(), t[:, :5], ids[:, :5], y[:, :5], move=lambda _: columns, what="columns of a wider tensor", **kw)
    turned = full.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    assert turned.stride(-1) != 1
    _check(full, t, ids, y, move=lambda _: turned, what="values apart", **kw)
    four = full.view(2, 2, 6, 517).cuda().permute(1, 2, 0, 3)
    _check(four.cpu(), *(a.view(2, 2, 6, -1).permute(1, 2, 0, 3) for a in (t, ids)), y.view(2, 2, 6).permute(1, 2, 0), move=lambda _: four, what="copied", **kw)


def test_gradient_of_a_broadcast_and_of_a_view():
    x, t, ids, y = _inputs(12, 301, 6, torch.float32, seed=16)
    base = x[:1].cuda().requires_grad_(True)
    F.distill_loss(base.expand(12, 301), t.cuda(), ids.cuda(), labels=y.cuda(), label_weight=0.5, temperature=2.0).backward()
    _, _, grad, gbound = ref.distill(x[:1].expand(12, 301), t, ids, 2.0, y, 1.0, 0.5)
    ref.assert_within(base.grad, grad.sum(0, keepdim=True), gbound.sum(0, keepdim=True) + 12 * ref.U * grad.abs().sum(0, keepdim=True), "broadcast")
    whole = torch.randn(3, 4, 301, device="cuda", requires_grad=True)
    F.distill_loss(whole[:, :-1], t[:9].view(3, 3, 6).cuda(), ids[:9].view(3, 3, 6).cuda()).backward()
    _, _, grad, gbound = ref.distill(whole.detach().cpu()[:, :-1], t[:9].view(3, 3, 6), ids[:9].view(3, 3, 6))
    ref.assert_within(whole.grad[:, :-1], grad, gbound, "view")
    assert not whole.grad[:, -1].any()


@pytest.mark.parametrize("shift", range(1, 8))
def test_rows_at_any_address(shift):
    for dtype in (torch.bfloat16, torch.float32):
        x, t, ids, y = _inputs(5, 1031, 6, dtype, seed=17)
        room = torch.zeros(5 * 1031 + 8, dtype=dtype, device="cuda")
        at = room[shift: shift + 5 * 1031].view(5, 1031)
        at.copy_(x)
        _check(x, t, ids, y, move=lambda _: at, temperature=2.0, label_weight=0.5)


@pytest.mark.parametrize("bits,gp_sz", [(4, 128), (5, 128), (6, 2048), (7, 256), (8, 128), (8, 4096)])
@pytest.mark.parametrize("rows,topk", [(1, 1), (7, 33), (40, 64)])
def test_stored_teacher(bits, gp_sz, rows, topk):
    """A teacher stored by vectorwise_quant gives what its values read back give."""
    x, t, ids, y = _inputs(rows, 801, topk, torch.bfloat16, seed=18)
    kw = dict(b=bits, signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", gp_sz=gp_sz,
              qmap=F.create_general_qmap("power-1", bits, True).cuda())
    codes, md = F.vectorwise_quant((t - 8).cuda(), **kw)
    quant = dict(kw, **md)
    back = F.vectorwise_dequant(codes, shape=torch.Size((rows, topk)), **quant)
    want, wgrad = _check(x, back.cpu(), ids, y, temperature=2.0, label_weight=0.5)
    for held in (ids, ids.int()):
        leaf = x.cuda().requires_grad_(True)
        loss = F.distill_loss(leaf, codes, held.cuda(), labels=y.cuda(), temperature=2.0, label_weight=0.5, teacher_quant=quant)
        loss.backward()
        assert torch.equal(loss, want) and torch.equal(leaf.grad, wgrad)
    by_name = dict(quant, qmap={(bits, True): {"power-1": kw["qmap"]}})
    assert torch.equal(F.distill_loss(x.cuda(), codes, ids.cuda(), labels=y.cuda(), temperature=2.0, label_weight=0.5, teacher_quant=by_name), want)


def test_gradient_against_differences():
    """float32 differences of the loss itself: h = 2^-4, third derivatives of at most the weights, loss errors of the stated bounds."""
    x, t, ids, y = _inputs(2, 23, 5, torch.float32, seed=19, ignored=0.0)
    _, bound, grad, gbound = ref.distill(x, t, ids, 2.0, y, 1.0, 0.5, reduction="sum")
    leaf = x.cuda().requires_grad_(True)
    args = (t.cuda(), ids.cuda())
    kw = dict(temperature=2.0, labels=y.cuda(), label_weight=0.5, reduction="sum")
    F.distill_loss(leaf, *args, **kw).backward()
    h = 2.0 ** -4
    # third derivative of log sum exp: at most 1/4 in size; of T^2 kd: T^2 / T^3 of it
    tolerance = h * h / 6 * (0.25 * (1.0 / 2 + 0.5)) + float(bound) / h + float(gbound.max())
    for n in range(2):
        for v in range(23):
            d = torch.zeros(2, 23)
            d[n, v] = h
            up, down = ((x + s * d) for s in (1, -1))
            slope = (float(F.distill_loss(up.cuda(), *args, **kw)) - float(F.distill_loss(down.cuda(), *args, **kw))) / float((up - down)[n, v])
            assert abs(slope - float(leaf.grad[n, v])) <= tolerance + 2 * h * ref.U * 8


def test_several_passes_over_one_graph():
    x, t, ids, y = _inputs(5, 301, 6, torch.bfloat16, seed=20)
    leaf = x.cuda().requires_grad_(True)
    loss = F.distill_loss(leaf, t.cuda(), ids.cuda(), labels=y.cuda(), label_weight=0.5, temperature=2.0)
    first = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
    kept = first.clone()
    first.zero_()  # a caller's own from here on
    assert torch.equal(torch.autograd.grad(loss, leaf, retain_graph=True)[0], kept)
    half = torch.autograd.grad(loss, leaf, torch.tensor(0.5, device="cuda"))[0]
    assert torch.equal(half, kept * 0.5)  # a power of two
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, leaf)
    loss = F.distill_loss(leaf, t.cuda(), ids.cuda())
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g = torch.autograd.grad(loss, leaf, create_graph=True)[0]
        torch.autograd.grad(g.float().sum(), leaf)
    with torch.no_grad():
        assert not F.distill_loss(leaf, t.cuda(), ids.cuda()).requires_grad
    loss = F.distill_loss(leaf, t.cuda(), ids.cuda())
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_a_loss_that_is_kept_does_not_keep_the_logits():
    head = torch.zeros(64, 1 << 16, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    head.grad = torch.zeros_like(head)
    t, ids = torch.zeros(64, 4, device="cuda"), torch.arange(4, device="cuda").expand(64, 4).contiguous()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    kept = []
    for _ in range(3):
        loss = F.distill_loss(head * 2, t, ids)
        loss.backward()
        kept.append(loss)
    assert torch.cuda.memory_allocated() - before < head.numel()


def test_another_stream_and_two_calls_at_once():
    sets = [_inputs(40, 5003, 16, torch.bfloat16, seed=21 + i) for i in range(2)]
    on = [[_cuda(a) for a in s] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for (x, t, ids, y), stream in zip(on, streams):
        with torch.cuda.stream(stream):
            leaf = x.requires_grad_(True)
            loss = F.distill_loss(leaf, t, ids, labels=y, label_weight=0.5, temperature=2.0)
            out.append((loss, torch.autograd.grad(loss, leaf)[0]))
    torch.cuda.synchronize()
    for (loss, grad), (x, t, ids, y) in zip(out, sets):
        want, bound, wgrad, gbound = ref.distill(x, t, ids, 2.0, y, 1.0, 0.5)
        ref.assert_within(loss, want, bound, "loss")
        ref.assert_within(grad, wgrad, gbound, "gradient")


@pytest.mark.parametrize("dtype,scale", [(torch.bfloat16, 1.0), (torch.bfloat16, 4.0), (torch.float16, 512.0)])
def test_captured_and_replayed(dtype, scale):
    """Two graphs of the loss and its gradient, replayed in turn with eager calls between, on new contents of the same tensors."""
    rows, vocab, topk = 20, 3001, 12
    held = [[_cuda(a) for a in _inputs(rows, vocab, topk, dtype, seed=30)] for _ in range(2)]
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def step(x, t, ids, y):
        leaf = x.detach().requires_grad_(True)
        loss = F.distill_loss(leaf, t, ids, labels=y, label_weight=0.5, temperature=2.0)
        return loss, torch.autograd.grad(loss if scale == 1.0 else loss * scale, leaf)[0]

    with torch.cuda.stream(stream):
        for s in held:
            step(*s)
    torch.cuda.current_stream().wait_stream(stream)
    for s in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    for turn in range(3):
        for k in range(2):
            new = _inputs(rows, vocab, topk, dtype, seed=31 + 2 * turn + k)
            for a, b in zip(held[k], new):
                a.copy_(b)
            graphs[k].replay()
            eager = step(*[_cuda(a) for a in new])
            torch.cuda.synchronize()
            assert torch.equal(outs[k][0], eager[0]) and torch.equal(outs[k][1], eager[1]), f"turn {turn}, graph {k}"


def test_a_recorded_backward_pass_of_an_eager_loss_writes_its_gradient_at_every_replay():
    stream = torch.cuda.Stream()
    sets = [_cuda(a) for a in _inputs(20, 3001, 12, torch.bfloat16, seed=56)]
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        leaf = sets[0].clone().requires_grad_(True)
        loss = F.distill_loss(leaf, sets[1], sets[2], labels=sets[3], label_weight=0.5, temperature=2.0)
        factor = torch.ones((), device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        grad = torch.autograd.grad(loss, leaf, factor, retain_graph=True)[0]
    torch.cuda.synchronize()
    want = torch.autograd.grad(loss, leaf)[0]
    torch.cuda.synchronize()
    for value in (1.0, 0.5, 1.0):
        factor.fill_(value)
        grad.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want * value)  # powers of two


def test_nothing_is_written_past_the_rows():
    from lpmm import _native

    x, t, ids, y = _inputs(3, 1003, 6, torch.bfloat16, seed=40, ignored=0.0)
    x, t, ids, y = x.cuda(), t.cuda(), ids.cuda(), y.cuda()
    pad = 64
    room = [torch.full((n + 2 * pad,), 7.0, dtype=d, device="cuda") for n, d in ((3 * 1003, torch.bfloat16), (3, torch.float32), (12, torch.float32),
                                                                                (1, torch.float32), (1, torch.float32))]
    grad, row_loss, stats, loss, share = (r[pad:].data_ptr() for r in room)
    record = ref.DISTILL_CALL.pack(x.data_ptr(), t.data_ptr(), 0, 0, ids.data_ptr(), y.data_ptr(), row_loss, stats, loss, share, grad, 3, 1003, 6,
                                       3, 0, 1003, 1, -100, 2.0, 1.0, 0.5, ref.TYPE_BF16, ref.TYPE_F32, 64, ref.REDUCE_MEAN, 8)
    lib = _native.lib()
    assert lib.lpmm_distill_loss(record, _native.current_stream(0)) == 0
    one = torch.tensor(3.0, device="cuda")
    assert lib.lpmm_distill_loss_grad(record, one.data_ptr(), 0, 1, _native.current_stream(0)) == 0
    torch.cuda.synchronize()
    for r in room:
        assert (r[:pad] == 7).all() and (r[-pad:] == 7).all()
    _, _, want, gbound = ref.distill(x.cpu(), t.cpu(), ids.cpu(), 2.0, y.cpu(), 1.0, 0.5, grad_loss=torch.tensor(3.0))
    ref.assert_within(room[0][pad:-pad].view(3, 1003), want, gbound, "gradient")


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last rows are what a call on them alone gives."""
    rows, vocab = 66000, 33000
    x = torch.randn(64, vocab, device="cuda").to(torch.bfloat16).repeat(rows // 64 + 1, 1)[:rows].requires_grad_(True)
    assert x.numel() > 2 ** 31
    t = torch.randn(rows, 5, device="cuda")
    ids = torch.randint(0, vocab, (rows, 5), device="cuda")
    y = torch.randint(0, vocab, (rows,), device="cuda")
    loss = F.distill_loss(x, t, ids, labels=y, label_weight=0.5, temperature=2.0, reduction="sum")
    grad = torch.autograd.grad(loss, x)[0]
    for cut in (slice(rows - 3, rows), slice(2 ** 31 // vocab - 1, 2 ** 31 // vocab + 2)):
        part = x.detach()[cut].clone().requires_grad_(True)
        alone = F.distill_loss(part, t[cut], ids[cut], labels=y[cut], label_weight=0.5, temperature=2.0, reduction="sum")
        assert torch.equal(torch.autograd.grad(alone, part)[0], grad[cut])
    assert loss.isfinite()


def test_more_rows_than_a_launch_has():
    """Short rows, so many that their threads do not fit 32 bits: the rows at the ends of the launches."""
    rows, vocab = (1 << 24) + 5, 3
    x = torch.randn(rows, vocab, device="cuda").requires_grad_(True)
    t, ids = torch.randn(rows, 2, device="cuda"), torch.randint(-1, vocab, (rows, 2), device="cuda", dtype=torch.int32)
    weight = torch.rand(rows, device="cuda")
    loss = F.distill_loss(x, t, ids, temperature=2.0, reduction="none")
    grad = torch.autograd.grad(loss, x, weight)[0]
    whole = F.distill_loss(x.detach(), t, ids, temperature=2.0, reduction="sum")
    for cut in (slice(rows - 7, rows), slice((1 << 21) - 2, (1 << 21) + 2)):
        want, bound, wgrad, gbound = ref.distill(x.detach()[cut].cpu(), t[cut].cpu(), ids[cut].cpu(), 2.0, reduction="none", grad_loss=weight[cut].cpu())
        ref.assert_within(loss[cut], want, bound, "loss")
        ref.assert_within(grad[cut], wgrad, gbound, "gradient")
    total = float(loss.detach().double().sum())  # the sum is in 64 bits, and rounded once
    assert abs(float(whole) - total) <= 2 * ref.U * abs(total)


def test_a_training_step_with_a_stored_teacher():
    """As it is used: the teacher's top logits stored in 8 bits, the student's loss with the balance of its router, 4-bit optimizer steps."""
    torch.manual_seed(50)
    width, vocab, experts, tokens = 64, 503, 8, 96
    h = torch.randn(tokens, width, device="cuda")
    teacher = torch.randn(tokens, vocab, device="cuda") * 3
    top = teacher.topk(16, dim=-1)
    kw = dict(b=8, signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", gp_sz=128,
              qmap=F.create_general_qmap("power-1", 8, True).cuda())
    codes, md = F.vectorwise_quant(top.values - top.values[:, :1], **kw)
    head = torch.nn.Parameter(torch.randn(vocab, width, device="cuda") * 0.05)
    router = torch.nn.Parameter(torch.randn(experts, width, device="cuda") * 0.05)
    opt = lpmm.optim.AdamW([head, router], lr=1e-3, fused=True)
    labels = teacher.argmax(-1).masked_fill(torch.rand(tokens, device="cuda") < 0.2, -100)
    for _ in range(3):
        logits, routed = h @ head.t(), h @ router.t()
        logits.retain_grad()
        routed.retain_grad()
        picks = routed.topk(2, dim=-1).indices
        aux, counts = F.balance_loss(routed, picks, mask=labels != -100, weight=0.01, z_weight=0.001)
        loss = F.distill_loss(logits, codes, top.indices, labels=labels, label_weight=0.5, teacher_weight=0.5, temperature=2.0,
                              teacher_quant=dict(kw, **md)) + aux
        opt.zero_grad()
        loss.backward()
        values = F.vectorwise_dequant(codes, shape=top.values.shape, **dict(kw, **md)).cpu()
        want, bound, grad, gbound = ref.distill(logits.detach().cpu(), values, top.indices.cpu(), 2.0, labels.cpu(), 0.5, 0.5)
        ref.assert_within(logits.grad, grad, gbound, "the student's gradient")
        bwant, bbound, bcounts, bgrad, bgbound = ref.balance(routed.detach().cpu(), picks.cpu(), (labels != -100).cpu(), 0.01, 0.001)
        ref.assert_within(routed.grad, bgrad, bgbound, "the router's gradient")
        assert torch.equal(counts.cpu(), bcounts)
        ref.assert_within(loss, want + bwant, bound + bbound + 2 * ref.U * (want + bwant).abs(), "the loss")
        before = head.detach().clone()
        opt.step()
        assert not torch.equal(before, head)


@pytest.mark.parametrize("dtype", TYPES)
def test_saved_tensors_that_come_back_elsewhere(dtype):
    """Hooks that keep saved tensors on the host, with other strides when they come back; what was on the device is overwritten by then."""
    x, t, ids, y = _inputs(6, 517, 6, dtype, seed=52)
    whole = torch.randn(6, 600, device="cuda").to(dtype)
    whole[:, 30:547] = x.cuda()
    args = [_cuda(a) for a in (t, ids, y)]
    view, router = whole.detach()[:, 30:547].requires_grad_(True), whole.detach()[:, 30:47].requires_grad_(True)
    picks = torch.randint(0, 17, (6, 2))
    mask = torch.tensor([True, False, True, True, True, False], device="cuda")
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), lambda v: v.cuda().contiguous()):
        loss = F.distill_loss(view, args[0], args[1], labels=args[2], temperature=2.0, label_weight=0.5)
        aux, _ = F.balance_loss(router, picks.cuda(), mask=mask, weight=0.5, z_weight=0.1)
    for a in (whole, *args, mask):
        a.zero_()
    grads = torch.autograd.grad(loss, view)[0], torch.autograd.grad(aux, router)[0]
    want, bound, grad, gbound = ref.distill(x, t, ids, 2.0, y, 1.0, 0.5)
    ref.assert_within(loss, want, bound, "loss")
    ref.assert_within(grads[0], grad, gbound, "gradient")
    want, bound, _, grad, gbound = ref.balance(x[:, :17], picks, torch.tensor([True, False, True, True, True, False]), 0.5, 0.1)
    ref.assert_within(aux, want, bound, "balance")
    ref.assert_within(grads[1], grad, gbound, "gradient of the balance")


def test_saved_tensors_that_come_back_as_others_are_refused():
    x, t, ids, y = _inputs(6, 517, 6, torch.float32, seed=53)
    for unpack in (lambda v: v, lambda v: v.cuda()[:1], lambda v: v.cuda().double()):
        leaf = x.cuda().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda v: v.cpu(), unpack):
            loss = F.distill_loss(leaf, t.cuda(), ids.cuda())
            aux, _ = F.balance_loss(leaf, ids.cuda())
        for out in (loss, aux):
            with pytest.raises(RuntimeError, match="came back from its hooks"):
                out.backward()


@pytest.mark.parametrize("reentrant", [False, True])
def test_inside_a_checkpoint(reentrant):
    """The head and its loss by chunks of rows, made again in the backward pass; no logits are kept between."""
    from torch.utils.checkpoint import checkpoint

    rows, vocab, width = 64, 5003, 16
    g = torch.Generator().manual_seed(54)
    h = torch.randn(rows, width, generator=g).cuda().requires_grad_(True)
    head = (torch.randn(vocab, width, generator=g) * 0.3).cuda().requires_grad_(True)
    _, t, ids, y = (_cuda(a) for a in _inputs(rows, vocab, 8, torch.float32, seed=55))

    def part(h, cut):
        return F.distill_loss(h @ head.t(), t[cut], ids[cut], labels=y[cut], label_weight=0.5, temperature=2.0, reduction="sum")

    whole = torch.autograd.grad(sum(part(h[n:n + 16], slice(n, n + 16)) for n in range(0, rows, 16)), (h, head))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = sum(checkpoint(part, h[n:n + 16], slice(n, n + 16), use_reentrant=reentrant) for n in range(0, rows, 16))
    assert torch.cuda.memory_allocated() - before < 16 * vocab * 4
    loss.backward()
    for got, want in zip((h.grad, head.grad), whole):
        assert torch.allclose(got, want, rtol=1e-4, atol=1e-4 * float(want.abs().max()))


def _awkward(x, vocab):
    """Rows that the sums relative to a thread's first values do not fit: the first half or all but one value masked, a late value far above the rest,
    values that grow along the row, magnitudes past one step."""
    x[0, :vocab // 2] = -math.inf
    x[1, :] = -math.inf
    x[1, vocab - 3] = 2.0
    x[2, vocab - 5] = 90.0
    x[3] = torch.linspace(-60, 60, vocab).to(x.dtype)
    x[4] = x[4] + 30000.0
    x[5, ::7] = -math.inf
    x[6, : vocab // 3] = torch.finfo(x.dtype).min
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,topk", [(100, 300), (4097, 5), (8191, 257), (9000, 600), (16384, 20), (16389, 20), (20001, 513), (32761, 9), (40000, 1024), (60001, 9), (70000, 9), (140001, 9)])
def test_many_rows_of_every_length(vocab, topk, dtype):
    """As many rows as the shapes for many rows ask for; what is checked is a part of them, with rows that need their largest value first."""
    x, t, ids, y = _inputs(10, vocab, topk, dtype, seed=57)
    x, rows = _awkward(x, vocab), 260
    t[1], ids[1] = 1.0, vocab - 3  # what the one value left can give
    ids[0], ids[6] = ids[0].clamp(min=vocab // 2), ids[6].clamp(min=vocab // 2)
    ids[5] = ids[5].masked_fill(ids[5] % 7 == 0, -1)
    y[:7] = torch.tensor([vocab - 1, vocab - 3, vocab - 5, vocab - 1, 3, 1, vocab - 2])
    many = lambda a: a.repeat((rows // 10,) + (1,) * (a.dim() - 1)).cuda()
    for temperature, wl in ((1.0, 0.5), (2.0, 0.5), (1.5, 0.25)):
        want, bound, grad, gbound = ref.distill(x, t, ids, temperature, y, 1.0, wl, reduction="none")
        leaf = many(x).requires_grad_(True)
        loss = F.distill_loss(leaf, many(t), many(ids), labels=many(y), temperature=temperature, label_weight=wl, reduction="none")
        loss.backward(torch.ones(rows, device="cuda"))
        for cut in (slice(0, 10), slice(rows - 10, rows)):
            ref.assert_within(loss[cut], want, bound, f"T={temperature} loss")
            ref.assert_within(leaf.grad[cut], grad, gbound, f"T={temperature} gradient")
        if dtype != torch.float16:  # the gradient that is made along with the loss
            made = leaf.detach().requires_grad_(True)
            F.distill_loss(made, many(t), many(ids), labels=many(y), temperature=temperature, label_weight=wl, reduction="sum").backward()
            ref.assert_within(made.grad[:10], grad, gbound, f"T={temperature} gradient made with the loss")
