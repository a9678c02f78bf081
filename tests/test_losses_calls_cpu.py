"""Calls of the training-loss terms that are refused before anything runs, and the versions of their two libraries; without a GPU."""
import pytest
import torch

import lpmm.functional as F
from lpmm import _native


def _stored(**change):
    quant = dict(b=8, signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", qmap=torch.linspace(-1, 1, 256),
                 max1=torch.ones(1, 1), scaled_shape=torch.Size((1, 128)), dtype=torch.float32, stride=None)
    quant.update(change)
    return quant


@pytest.mark.parametrize("name,change,values", [
    ("qmap", dict(qmap={(8, True): {"power-1": None}}), torch.zeros(2049, dtype=torch.int8)),
    ("max1", dict(max1=None), torch.zeros(2049, dtype=torch.int8)),
    ("max1", dict(max1=None), torch.randn(3, 4)),  # plain values: the codes' keywords would be passed over
    ("max1", dict(max1=[1.0]), torch.zeros(2049, dtype=torch.int8)),
])
def test_a_stored_teacher_needs_its_map_and_scales(name, change, values):
    with pytest.raises(TypeError, match=f"{name} must be a tensor"):
        F.distill_loss(torch.randn(3, 20), values, torch.randint(0, 20, (3, 4)), teacher_quant=_stored(**change))


@pytest.mark.parametrize("scale,qmap", [(None, torch.linspace(-1, 1, 256)), (torch.ones(1, 1), None)])
def test_the_host_side_takes_map_and_scales_together(scale, qmap):
    with pytest.raises(RuntimeError, match="both max1 and qmap"):
        _native.losses().distill_loss(torch.randn(3, 20), torch.zeros(2049, dtype=torch.int8), torch.randint(0, 20, (3, 4)), 1.0, None, 1.0, 0.0,
                                      -100, 2, scale, qmap, 128, 8)


def _distill(x):
    return F.distill_loss(x, torch.zeros(3, 4), torch.arange(12).view(3, 4))


def _balance(x):
    return F.balance_loss(x, torch.zeros(3, 2, dtype=torch.int64))[0]


LOSSES = [(_distill, "logits"), (_balance, "router_logits")]


@pytest.mark.parametrize("loss,name", LOSSES)
def test_a_forward_mode_derivative_is_refused(loss, name):
    """It would come out as zero; the values with which it comes are on the device in earnest, where the same check runs first."""
    import torch.autograd.forward_ad as forward_ad

    x = torch.randn(3, 20)
    with forward_ad.dual_level():
        for dual in (forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(torch.randn(6, 20), torch.ones(6, 20))[::2]):
            with pytest.raises(RuntimeError, match=f"^{name} has a forward-mode gradient"):
                loss(dual)
        with pytest.raises(RuntimeError, match="CUDA"):
            loss(x)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(loss, (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("loss,name", LOSSES)
def test_tracers_are_refused(loss, name):
    """They would record the outputs' allocation alone, and give back memory that nothing wrote."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(3, 20)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(loss, (x,))
    for kw in (dict(tracing_mode="real"), dict(tracing_mode="fake"), dict(tracing_mode="symbolic"), dict(pre_dispatch=True)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(loss, **kw)(x)
    with FakeTensorMode() as mode, pytest.raises(RuntimeError, match="cannot be traced"):
        loss(mode.from_tensor(x))
    with pytest.raises(RuntimeError, match="CUDA"):  # nothing of it stays behind
        loss(x)


class _Wraps(torch.Tensor):
    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device="cuda", strides=inner.stride())

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} of a wrapper")


@pytest.mark.parametrize("loss,name", LOSSES)
def test_tensors_without_memory_are_refused(loss, name):
    with pytest.raises(RuntimeError, match=f"{name} has no memory of its own"):
        loss(_Wraps(torch.randn(3, 20)))


def _header():
    import os

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "lpmm_hip.h")) as f:
        return f.read()


def test_versions_and_records_are_those_of_the_header():
    import re

    import losses_ref as ref

    assert int(re.search(r"#define LPMM_HIP_ABI_VERSION (\d+)", _header()).group(1)) == _native.ABI_VERSION
    assert _native.lib().lpmm_abi_version() == _native.ABI_VERSION
    assert _native.losses().record_bytes == (ref.DISTILL_CALL.size, ref.BALANCE_CALL.size)


def test_a_host_side_of_another_version_is_an_error(monkeypatch):
    import sys
    import types

    import lpmm

    _native.losses()
    stale = types.ModuleType("lpmm._losses")
    stale.abi_version = _native.ABI_VERSION - 1
    monkeypatch.setattr(_native, "_losses", None)
    monkeypatch.setattr(lpmm, "_losses", stale)
    monkeypatch.setitem(sys.modules, "lpmm._losses", stale)
    for _ in range(2):
        with pytest.raises(RuntimeError, match=f"built for ABI version {_native.ABI_VERSION - 1}, expected {_native.ABI_VERSION}; rebuild it"):
            F.balance_loss(torch.randn(3, 20), torch.zeros(3, 2, dtype=torch.int64))


def test_a_library_of_another_version_is_named_before_its_functions_are_looked_up(monkeypatch):
    class Old:
        @staticmethod
        def lpmm_abi_version():
            return 2

        def __getattr__(self, name):
            raise AttributeError(f"undefined symbol: {name}")

    monkeypatch.setattr(_native, "_lib", None)
    monkeypatch.setattr(_native.ctypes, "CDLL", lambda path: Old())
    with pytest.raises(RuntimeError, match="ABI version 2, expected .*; rebuild it"):
        _native.lib()


@pytest.mark.parametrize("tokens,picks", [(2 ** 28, 8), (2 ** 21, 1024)])
def test_more_picks_than_31_bits_count_are_refused_by_name(tokens, picks):
    r = torch.zeros(1, 1).expand(tokens, picks)
    ids = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match=f"fewer than 2\\^31 picks in a group are supported, got {tokens} tokens of {picks}"):
        F.balance_loss(r, ids.expand(tokens, picks))
    with pytest.raises(RuntimeError, match="CUDA"):
        F.balance_loss(r, ids.expand(tokens, picks - 1))


def test_more_rows_than_31_bits_count_are_refused_by_name():
    def call(rows):
        x, ids = torch.zeros(1, 1).expand(rows, 1), torch.zeros(1, 0, dtype=torch.int64).expand(rows, 0)
        return F.distill_loss(x, torch.zeros(1, 0).expand(rows, 0), ids)

    with pytest.raises(RuntimeError, match="fewer than 2\\^31 rows, got 2147483648"):
        call(2 ** 31)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(2 ** 31 - 1)
