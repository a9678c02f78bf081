"""Ways of calling the training-loss terms in which the call itself, not a row, is what can go wrong."""
import pytest
import torch

import lpmm.functional as F

pytestmark = pytest.mark.gpu


def _distill():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 300, generator=g).cuda().requires_grad_(True)
    t, ids, y = torch.randn(6, 5, generator=g).cuda(), torch.randint(0, 300, (6, 5), generator=g).cuda(), torch.randint(0, 300, (6,), generator=g).cuda()
    return x, lambda: F.distill_loss(x, t, ids, temperature=2.0, labels=y, label_weight=0.5)


def _balance():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 12, generator=g).cuda().requires_grad_(True)
    ids = torch.randint(0, 12, (40, 2), generator=g).cuda()
    return x, lambda: F.balance_loss(x, ids, z_weight=0.1)[0]


BOTH = [_distill, _balance]


@pytest.mark.parametrize("make", BOTH)
def test_a_backward_pass_that_is_traced_or_dual_is_refused(make):
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x, loss = make()
    value = loss()
    want = torch.autograd.grad(value, x, retain_graph=True)[0].clone()
    one = torch.ones((), device="cuda")

    def backward(g):
        return torch.autograd.grad(value, x, g, retain_graph=True)[0]

    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(backward)(one)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="gradient of the loss has a forward-mode gradient"):
        backward(forward_ad.make_dual(one, torch.ones_like(one)))
    assert torch.equal(backward(one), want)


@pytest.mark.parametrize("make", BOTH)
def test_transforms_raise(make):
    x, loss = make()
    with pytest.raises(RuntimeError):  # several gradients in one backward pass
        torch.autograd.grad(loss(), x, torch.ones(3, device="cuda"), is_grads_batched=True)


@pytest.mark.parametrize("make", BOTH)
def test_modes_that_look_on_change_nothing(make):
    from torch.utils._python_dispatch import TorchDispatchMode
    from torch.utils.flop_counter import FlopCounterMode

    class Names(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    x, loss = make()

    def step():
        value = loss()
        return value.detach(), torch.autograd.grad(value, x)[0]

    want = step()
    for mode in (Names(), FlopCounterMode(display=False)):
        with mode:
            got = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("make", BOTH)
def test_a_compiled_step_runs_the_call_as_it_is(make):
    x, loss = make()

    def step(scale):
        return (loss() * scale).sin()

    want = step(torch.full((), 0.5, device="cuda"))
    got = torch.compile(step, backend="eager")(torch.full((), 0.5, device="cuda"))
    assert torch.equal(got.detach(), want.detach())
    a, b = torch.autograd.grad(got, x)[0], torch.autograd.grad(want, x)[0]
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("with_label", [True, False])
def test_labels_that_leave_the_last_position_out(dtype, with_label):
    """Whole logits with shifted labels are the loss of the slice, in 64 bits and as the package computes the slice."""
    import losses_ref as ref

    g = torch.Generator().manual_seed(3)
    x = (torch.randn(3, 9, 67, generator=g) * 3).to(dtype)
    t, ids = torch.randn(3, 9, 6, generator=g) * 3, torch.randint(-1, 67, (3, 9, 6), generator=g)
    tokens = torch.randint(0, 67, (3, 9), generator=g)
    shifted = torch.nn.functional.pad(tokens[:, 1:], (0, 1), value=-100)
    kw = dict(temperature=2.0, teacher_weight=0.75, label_weight=0.5 if with_label else 0.0)
    leaf, view = x.cuda().requires_grad_(True), x.cuda().requires_grad_(True)
    F.distill_loss(leaf, t.cuda(), ids.cuda(), labels=shifted.cuda(), **kw).backward()
    loss = F.distill_loss(leaf, t.cuda(), ids.cuda(), labels=shifted.cuda(), **kw)
    sliced = F.distill_loss(view[:, :-1], t[:, :-1].cuda(), ids[:, :-1].cuda(), labels=tokens[:, 1:].cuda() if with_label else None, **kw)
    sliced.backward()
    want, bound, grad, gbound = ref.distill(x[:, :-1], t[:, :-1], ids[:, :-1], 2.0, tokens[:, 1:] if with_label else None, 0.75, kw["label_weight"])
    ref.assert_within(loss, want, bound, "whole")
    ref.assert_within(sliced, want, bound, "slice")
    ref.assert_within(leaf.grad[:, :-1], grad, gbound, "whole gradient")
    ref.assert_within(view.grad[:, :-1], grad, gbound, "slice gradient")
    assert not leaf.grad[:, -1].any() and not view.grad[:, -1].any()


def test_the_documented_step():
    """Teacher stored offline, whole logits, labels that leave the last position out, the balance beside it, one backward pass."""
    import losses_ref as ref

    g = torch.Generator().manual_seed(4)
    teacher, tokens = (torch.randn(2, 33, 301, generator=g) * 3).cuda(), torch.randint(0, 301, (2, 33), generator=g)
    top = teacher.topk(16, dim=-1)
    kw = dict(b=8, signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", gp_sz=128,
              qmap=F.create_general_qmap("power-1", 8, True).cuda())
    codes, md = F.vectorwise_quant((top.values - top.values[..., :1]).float(), **kw)
    back = F.vectorwise_dequant(codes, shape=top.values.shape, **kw, **md).cpu()
    shifted = torch.nn.functional.pad(tokens[:, 1:], (0, 1), value=-100)
    x, r = torch.randn(2, 33, 301, generator=g) * 2, torch.randn(66, 12, generator=g)
    picks = r.topk(2, dim=-1).indices
    logits, router = x.cuda().requires_grad_(True), r.cuda().requires_grad_(True)
    loss = F.distill_loss(logits, codes, top.indices, temperature=2.0, labels=shifted.cuda(), teacher_weight=0.5, label_weight=0.5,
                          teacher_quant=dict(kw, **md))
    aux, counts = F.balance_loss(router, picks.cuda(), weight=0.01, z_weight=0.001)
    (loss + aux).backward()
    want, bound, grad, gbound = ref.distill(x, back, top.indices.cpu(), 2.0, shifted, 0.5, 0.5)
    ref.assert_within(loss, want, bound, "loss")
    ref.assert_within(logits.grad, grad, gbound, "gradient")
    want, bound, wcounts, grad, gbound = ref.balance(r, picks, None, 0.01, 0.001)
    ref.assert_within(aux, want, bound, "balance")
    ref.assert_within(router.grad, grad, gbound, "its gradient")
    assert torch.equal(counts.cpu(), wcounts)


@pytest.mark.parametrize("make", BOTH)
def test_a_gradient_that_is_negated_where_it_is_read(make):
    """What complex arithmetic behind the loss sends back may be the imaginary part of a conjugate, whose memory has the other sign."""
    x, loss = make()
    plain = torch.autograd.grad(loss(), x)[0]
    seen = []
    value = loss()
    value.register_hook(lambda g: seen.append(g.is_neg()))
    grad = torch.autograd.grad((torch.complex(torch.ones((), device="cuda"), value).conj() * (2 + 3j)).imag, x)[0]
    assert seen == [True]
    assert ((grad + 2 * plain).abs() <= 4 * 2.0 ** -24 * grad.abs() + 2.0 ** -126).all()  # two roundings of a product on either side


def test_inputs_that_are_negated_where_they_are_read():
    x, _ = _distill()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 300, (6, 5), generator=g).cuda()
    t = torch.randn(6, 5, generator=g).cuda()
    for neg in (lambda a: torch._neg_view(-a), lambda a: torch.complex(a, -a).conj().imag):
        other = neg(x.detach())
        assert other.is_neg()
        want, got = (F.distill_loss(a, b, ids, temperature=2.0) for a, b in ((x.detach(), t), (other, neg(t))))
        assert torch.equal(want, got)
        leaf = neg(x.detach()).requires_grad_(True)
        grads = [torch.autograd.grad(F.distill_loss(a, t, ids), a)[0] for a in (x, leaf)]
        assert torch.equal(*grads)
    router, picks = torch.randn(40, 12, generator=g).cuda(), torch.randint(0, 12, (40, 2), generator=g).cuda()
    leaves = [router.clone().requires_grad_(True), torch._neg_view(-router).requires_grad_(True)]
    both = [F.balance_loss(a, picks, z_weight=0.1)[0] for a in leaves]
    assert torch.equal(both[0].detach(), both[1].detach())
    assert torch.equal(*[torch.autograd.grad(b, a)[0] for b, a in zip(both, leaves)])


class _Wraps(torch.Tensor):
    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device, strides=inner.stride())

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} of a wrapper")


@pytest.mark.parametrize("make,wrapped", [(_distill, torch.int64), (_balance, torch.bool)])
def test_saved_tensors_that_come_back_without_memory_are_refused(make, wrapped):
    """Labels and masks above all: an address of NULL means that there are none."""
    if make is _balance:
        x = torch.randn(40, 12, device="cuda", requires_grad=True)
        ids, mask = torch.randint(0, 12, (40, 2), device="cuda"), torch.rand(40, device="cuda") < 0.5

        def loss():
            return F.balance_loss(x, ids, mask=mask)[0]
    else:
        x, loss = make()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: _Wraps(t) if t.dtype == wrapped else t):
        value = loss()
    with pytest.raises(RuntimeError, match="came back from its hooks as another"):
        value.backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.25, 1.0, 1.25, 2.0])
def test_entries_and_labels_at_masked_logits_of_the_lowest_value(dtype, temperature):
    """Their losses are large and not infinite: a logit of -3.4e38 has an exponent of 2 that float32 has not."""
    import losses_ref as ref

    g = torch.Generator().manual_seed(5)
    least, most = torch.finfo(dtype).min, torch.finfo(dtype).max
    for vocab in (203, 9001):
        x = (torch.randn(6, vocab, generator=g) * 2).to(dtype)
        t, y = torch.randn(6, 5, generator=g), torch.randint(100, 200, (6,), generator=g)
        ids = torch.arange(5).expand(6, 5) * 17 + 3
        x[0, 20] = least  # an entry
        x[1, y[1]] = least  # the label
        x[2, 20], x[2, y[2]] = least, least
        x[3, 1] = most  # all but one
        x[4, 1], x[4, 20], x[4, y[4]] = most, least, least
        for wt, wl in ((0.125, 0.125), (0.125, 0.0), (0.0, 0.125)):
            kw = dict(temperature=temperature, teacher_weight=wt, label_weight=wl, reduction="none")
            leaf = x.cuda().requires_grad_(True)
            loss = F.distill_loss(leaf, t.cuda(), ids.cuda(), labels=y.cuda(), **kw)
            up = 1024.0 if dtype == torch.float16 else 1.0
            grad = torch.autograd.grad(loss, leaf, torch.full((6,), up, device="cuda"))[0]
            want, bound, wgrad, gbound = ref.distill(x, t, ids, temperature, y, wt, wl, reduction="none", grad_loss=torch.full((6,), up))
            assert want.lt(torch.finfo(torch.float32).max).all()
            ref.assert_within(loss, want, bound, f"{vocab} {wt} {wl} loss")
            ref.assert_within(grad, wgrad, gbound, f"{vocab} {wt} {wl} gradient")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_entries_of_little_probability_at_masked_logits(dtype):
    """Whatever the teacher gives to a logit of -infinity, the smallest numbers that float32 has among it, the loss is infinite and not NaN."""
    for weight, temperature in ((1.0, 1.0), (1e-3, 1.0), (0.25, 0.25), (-0.5, 2.0)):
        x = torch.zeros(4, 40, dtype=dtype)
        x[:, 7] = -float("inf")
        t = torch.zeros(4, 3)
        t[:, 1] = torch.tensor([-1.0, -60.0, -92.0, -100.0]) * temperature  # e^-100: 4e-44, which a weight takes to 0
        ids, y = torch.tensor([3, 7, 5]).expand(4, 3), torch.tensor([0, 1, 7, 2])
        loss = F.distill_loss(x.cuda(), t.cuda(), ids.cuda(), temperature=temperature, teacher_weight=weight, reduction="none")
        assert loss.isinf().all() and (loss * weight > 0).all()
        loss = F.distill_loss(x.cuda(), t.cuda(), ids.cuda(), labels=y.cuda(), teacher_weight=0.0, label_weight=abs(weight), reduction="none")
        assert loss.isinf().tolist() == [False, False, True, False] and loss[2] > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts", [8, 17, 200])
def test_router_logits_of_the_largest_and_lowest_values(experts, dtype):
    """The gradient of logsumexp^2 there is large, where it is not 0; experts without probability have none of it."""
    import losses_ref as ref

    least, most = torch.finfo(dtype).min, torch.finfo(dtype).max
    for fill, at in ((least, None), (least, 0.0), (0.0, least), (0.0, most), (least, most), (0.0, most / 4)):
        for tokens in (1, 2):
            r = torch.full((tokens, experts), fill, dtype=dtype)
            if at is not None:
                r[0, 3] = at
            ids = torch.arange(tokens).view(tokens, 1)
            for up in (0.125, 1e-3):
                leaf = r.cuda().requires_grad_(True)
                loss, _ = F.balance_loss(leaf, ids.cuda(), weight=0.5, z_weight=1.0)
                loss.backward(torch.full((), up, device="cuda"))
                want, bound, _, grad, gbound = ref.balance(r, ids, None, 0.5, 1.0, float(torch.tensor(up)))
                what = f"{tokens} x {experts} of {fill} with {at}, factor {up}"
                ref.assert_within(loss, want, bound, what)
                ref.assert_within(leaf.grad, grad, gbound, what)


@pytest.mark.parametrize("make", BOTH)
def test_threads_with_graphs_of_their_own_and_with_one(make):
    import threading

    x, loss = make()
    shared = loss()
    want = torch.autograd.grad(shared, x, retain_graph=True)[0].clone()
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    for value in (loss(), shared):
                        grad = torch.autograd.grad(value, x, retain_graph=value is shared)[0]
                        torch.cuda.synchronize()
                        if not torch.equal(grad, want):
                            wrong.append("gradient")
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
