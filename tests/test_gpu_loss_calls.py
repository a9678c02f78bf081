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
