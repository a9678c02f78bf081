"""The training-loss terms without a GPU: what their calls refuse, the library's argument checks, and that the tests' own definitions
agree with differences and with torch's losses."""
import ctypes
import math

import pytest
import torch

import lpmm.functional as F
import losses_ref as ref

NULL, ALIGN, SIZE, ARG = 1, 2, 3, 5


def _distill_inputs(rows=3, vocab=20, topk=4, **over):
    t = dict(logits=torch.randn(rows, vocab), teacher_logits=torch.randn(rows, topk), teacher_ids=torch.randint(0, vocab, (rows, topk)))
    t.update(over)
    return t


@pytest.mark.parametrize("error,text,change", [
    (RuntimeError, "CUDA", {}),
    (TypeError, "logits must be a tensor", dict(logits=[1.0])),
    (TypeError, "labels must be a tensor", dict(labels=[1, 2, 3])),
    (RuntimeError, "float32, float16 or bfloat16", dict(logits=torch.randn(3, 20).double())),
    (RuntimeError, "teacher_logits is not float32", dict(teacher_logits=torch.zeros(3, 4, dtype=torch.int32))),
    (RuntimeError, "do not belong to logits", dict(logits=torch.randn(4, 20))),
    (RuntimeError, "do not belong to logits", dict(logits=torch.randn(3, 1, 20))),
    (RuntimeError, "do not belong to teacher_ids", dict(teacher_logits=torch.randn(3, 5))),
    (RuntimeError, "teacher_ids must be int32 or int64", dict(teacher_ids=torch.zeros(3, 4))),
    (RuntimeError, "at least one dimension", dict(logits=torch.tensor(1.0))),
    (RuntimeError, "1 to 2\\^31 - 1 values", dict(logits=torch.randn(3, 0))),
    (RuntimeError, "at most 1024 teacher entries", dict(teacher_logits=torch.randn(3, 1025), teacher_ids=torch.zeros(3, 1025, dtype=torch.int64))),
    (RuntimeError, "labels must be int64", dict(labels=torch.zeros(3, dtype=torch.int32))),
    (RuntimeError, "labels of shape", dict(labels=torch.zeros(4, dtype=torch.int64))),
    (ValueError, "label_weight needs labels", dict(label_weight=1.0)),
    (ValueError, "teacher_weight must be finite", dict(teacher_weight=math.nan)),
    (ValueError, "label_weight must be finite", dict(label_weight=math.inf, labels=torch.zeros(3, dtype=torch.int64))),
    (ValueError, "temperature", dict(temperature=0.0)),
    (ValueError, "temperature", dict(temperature=-1.0)),
    (ValueError, "temperature", dict(temperature=math.nan)),
    (ValueError, "temperature", dict(temperature=2048.0)),
    (ValueError, "reduction", dict(reduction="batchmean")),
])
def test_distill_refuses(error, text, change):
    with pytest.raises(error, match=text):
        F.distill_loss(**_distill_inputs(**change))


def _stored(**over):
    quant = dict(b=8, signed=True, quant_type="power-1", round_type="real-nearest", scale_type="group", qmap=torch.linspace(-1, 1, 256),
                 max1=torch.ones(1, 1), scaled_shape=torch.Size((1, 128)), dtype=torch.float32, stride=None)
    quant.update(over)
    return quant


@pytest.mark.parametrize("error,text,change,codes", [
    (RuntimeError, "CUDA", {}, None),
    (NotImplementedError, "by 'group'", dict(scale_type="rank1"), None),
    (NotImplementedError, "4 to 8 bits", dict(b=2), None),
    (ValueError, "Not support", dict(quant_type="linear"), None),
    (ValueError, "group size", dict(scaled_shape=torch.Size((1, 0))), None),
    (RuntimeError, "maps must have 256", dict(qmap=torch.linspace(-1, 1, 16)), None),
    (RuntimeError, "contiguous float32", dict(qmap=torch.linspace(-1, 1, 256).double()), None),
    (RuntimeError, "contiguous float32", dict(max1=torch.ones(1, 1, dtype=torch.float16)), None),
    (RuntimeError, "fewer than the 12 values", dict(max1=torch.ones(0, 1)), None),
    (RuntimeError, "fewer than the 12 values", {}, torch.zeros(11, dtype=torch.int8)),
    (RuntimeError, "1-D int8", {}, torch.zeros(2049)),
    (RuntimeError, "1-D int8", {}, torch.zeros(3, 683, dtype=torch.int8)),
    (TypeError, "qmap must be a tensor|indices|subscriptable", dict(qmap=None), None),
])
def test_stored_teacher_refuses(error, text, change, codes):
    codes = torch.zeros(2049, dtype=torch.int8) if codes is None else codes
    with pytest.raises(error, match=text):
        F.distill_loss(**_distill_inputs(teacher_logits=codes, teacher_quant=_stored(**change)))


@pytest.mark.parametrize("error,text,change", [
    (RuntimeError, "CUDA", {}),
    (TypeError, "mask must be a tensor", dict(mask=[True])),
    (RuntimeError, "float32, float16 or bfloat16", dict(router_logits=torch.randn(5, 8).double())),
    (RuntimeError, "must be \\(tokens, experts\\)", dict(router_logits=torch.randn(8))),
    (RuntimeError, "must be \\(tokens, experts\\)", dict(router_logits=torch.randn(1, 1, 5, 8))),
    (RuntimeError, "do not belong to router_logits", dict(router_logits=torch.randn(6, 8))),
    (RuntimeError, "do not belong to router_logits", dict(router_logits=torch.randn(1, 5, 8))),
    (RuntimeError, "expert_ids must be int32 or int64", dict(expert_ids=torch.zeros(5, 2))),
    (RuntimeError, "experts are supported", dict(router_logits=torch.randn(5, 1025))),
    (RuntimeError, "experts are supported", dict(router_logits=torch.randn(5, 0))),
    (RuntimeError, "3 picks of 2", dict(router_logits=torch.randn(5, 2), expert_ids=torch.zeros(5, 3, dtype=torch.int64))),
    (RuntimeError, "at most 65535 groups", dict(router_logits=torch.zeros(1, 1, 1).expand(65536, 1, 1), expert_ids=torch.zeros(65536, 1, 1, dtype=torch.int32))),
    (RuntimeError, "tokens in all", dict(router_logits=torch.zeros(1, 1, 1).expand(2, 2 ** 27 + 1, 1),
                                         expert_ids=torch.zeros(1, 1, 0, dtype=torch.int32).expand(2, 2 ** 27 + 1, 0))),
    (RuntimeError, "mask must be a bool tensor", dict(mask=torch.ones(5))),
    (RuntimeError, "mask must be a bool tensor", dict(mask=torch.ones(5, 1, dtype=torch.bool))),
    (ValueError, "weight must be finite", dict(weight=math.nan)),
    (ValueError, "z_weight must be finite", dict(z_weight=math.inf)),
])
def test_balance_refuses(error, text, change):
    t = dict(router_logits=torch.randn(5, 8), expert_ids=torch.zeros(5, 2, dtype=torch.int64))
    t.update(change)
    with pytest.raises(error, match=text):
        F.balance_loss(**t)


def _address():
    keep = ctypes.create_string_buffer(256)
    return keep, (ctypes.addressof(keep) + 63) // 64 * 64


DISTILL = ("logits teacher scale map ids labels row_loss stats loss share grad rows vocab topk inner outer inner_stride group ignore temperature "
           "wt wl type teacher_type id_bits reduction bits").split()


def _distill_record(**change):
    from lpmm import _native

    keep, at = _address()
    v = dict(logits=at, teacher=at, scale=0, map=0, ids=at, labels=at, row_loss=at, stats=at, loss=at, share=at, grad=at, rows=2, vocab=8,
             topk=2, inner=2, outer=0, inner_stride=8, group=1, ignore=-100, temperature=1.0, wt=1.0, wl=1.0, type=0, teacher_type=0,
             id_bits=64, reduction=2, bits=8)
    assert list(v) == DISTILL
    for k, to in change.items():
        v[k] = at + to if isinstance(to, int) and k in DISTILL[:11] and to else to
    return keep, ref.DISTILL_CALL.pack(*v.values())


@pytest.mark.parametrize("status,change", [
    (NULL, dict(logits=0)), (NULL, dict(teacher=0)), (NULL, dict(ids=0)), (NULL, dict(row_loss=0)), (NULL, dict(loss=0)), (NULL, dict(share=0)),
    (ALIGN, dict(logits=2)), (ALIGN, dict(ids=4)), (ALIGN, dict(labels=4)), (ALIGN, dict(stats=8)), (ALIGN, dict(grad=2)),
    (ALIGN, dict(teacher=1, teacher_type=2)), (ALIGN, dict(row_loss=2)),
    (SIZE, dict(rows=-1)), (SIZE, dict(vocab=0)), (SIZE, dict(vocab=2 ** 31)), (SIZE, dict(topk=1025)), (SIZE, dict(topk=-1)),
    (SIZE, dict(inner=0)), (SIZE, dict(outer=-8)), (SIZE, dict(inner_stride=-8)), (SIZE, dict(rows=2 ** 41)),
    (ARG, dict(type=3)), (ARG, dict(type=-1)), (ARG, dict(teacher_type=4)), (ARG, dict(id_bits=16)), (ARG, dict(reduction=3)),
    (ARG, dict(reduction=0)),  # with a gradient
    (ARG, dict(temperature=0.0)), (ARG, dict(temperature=math.nan)), (ARG, dict(temperature=1e4)), (ARG, dict(wt=math.inf)), (ARG, dict(wl=math.nan)),
    (NULL, dict(teacher_type=3)), (NULL, dict(teacher_type=3, scale=4)),
    (SIZE, dict(teacher_type=3, scale=4, map=4, group=0)), (SIZE, dict(teacher_type=3, scale=4, map=4, bits=3)),
    (SIZE, dict(teacher_type=3, scale=4, map=4, bits=9)),
])
def test_distill_argument_errors_without_gpu(status, change):
    from lpmm import _native

    keep, record = _distill_record(**change)
    assert _native.lib().lpmm_distill_loss(record, None) == status


@pytest.mark.parametrize("status,change,grad_loss,stride,made", [
    (NULL, {}, 0, 0, 0), (ALIGN, {}, 2, 0, 0), (SIZE, {}, 4, -1, 0), (NULL, dict(grad=0), 4, 0, 0), (NULL, dict(stats=0), 4, 0, 0),
    (ARG, dict(reduction=0), 4, 0, 1), (SIZE, dict(vocab=-1), 4, 0, 0), (0, dict(rows=0), 0, 0, 0),
])
def test_distill_gradient_argument_errors_without_gpu(status, change, grad_loss, stride, made):
    from lpmm import _native

    keep, record = _distill_record(**change)
    at = _address()
    assert _native.lib().lpmm_distill_loss_grad(record, at[1] + grad_loss if grad_loss else None, stride, made, None) == status


BALANCE = "logits ids mask loss counts factors work grad groups tokens experts picks outer inner weight z_weight type id_bits".split()


def _balance_record(**change):
    from lpmm import _native

    keep, at = _address()
    v = dict(logits=at, ids=at, mask=0, loss=at, counts=at, factors=at, work=at, grad=at, groups=1, tokens=4, experts=8, picks=2, outer=0,
             inner=8, weight=1.0, z_weight=0.0, type=0, id_bits=64)
    assert list(v) == BALANCE
    for k, to in change.items():
        v[k] = at + to if k in BALANCE[:8] and to else to
    return keep, ref.BALANCE_CALL.pack(*v.values())


@pytest.mark.parametrize("status,change,grad", [
    (NULL, dict(logits=0), False), (NULL, dict(ids=0), False), (NULL, dict(loss=0), False), (NULL, dict(counts=0), False),
    (NULL, dict(factors=0), False), (NULL, dict(work=0), False), (NULL, dict(grad=0), True), (NULL, dict(factors=0), True),
    (ALIGN, dict(logits=2), False), (ALIGN, dict(ids=4), False), (ALIGN, dict(counts=4), False), (ALIGN, dict(work=4), False),
    (ALIGN, dict(loss=2), False), (ALIGN, dict(grad=2), True), (ALIGN, dict(factors=2), True),
    (SIZE, dict(experts=0), False), (SIZE, dict(experts=1025), False), (SIZE, dict(picks=9), False), (SIZE, dict(picks=-1), False),
    (SIZE, dict(groups=-1), False), (SIZE, dict(tokens=-1), False), (SIZE, dict(tokens=2 ** 30), False), (SIZE, dict(inner=-8), True),
    (SIZE, dict(groups=65536), False), (SIZE, dict(groups=65536, tokens=0), True), (SIZE, dict(tokens=2 ** 28 + 1), True),
    (SIZE, dict(groups=3, tokens=2 ** 27), False),
    (ARG, dict(type=3), False), (ARG, dict(id_bits=8), False), (ARG, dict(weight=math.nan), False), (ARG, dict(z_weight=math.inf), True),
    (0, dict(groups=0), True), (0, dict(tokens=0), True),
])
def test_balance_argument_errors_without_gpu(status, change, grad):
    from lpmm import _native

    keep, record = _balance_record(**change)
    at = _address()
    if grad:
        assert _native.lib().lpmm_balance_loss_grad(record, at[1], None) == status
    else:
        assert _native.lib().lpmm_balance_loss(record, None) == status


def test_records_match_the_header():
    from lpmm import _native

    assert _native.losses().abi_version == _native.ABI_VERSION
    assert ref.DISTILL_CALL.size == 184 and ref.BALANCE_CALL.size == 128
    assert _native.lib().lpmm_distill_loss(None, None) == NULL and _native.lib().lpmm_balance_loss(None, None) == NULL
    assert _native.lib().lpmm_balance_work_bytes(0, 5, 8) == 0 and _native.lib().lpmm_balance_work_bytes(3, 5, 8) > 0


def test_views_of_rows_keep_their_strides():
    from lpmm import _native

    row_strides = _native.losses().row_strides
    t = torch.zeros(4, 6, 8)
    for view, want in [(t, (24, 0, 8)), (t[:, :-1], (5, 48, 8)), (t[:, 1:, :5], (5, 48, 8)), (t[:, 0], (4, 0, 48)), (t[0, 0], (1, 0, 0)),
                       (t.transpose(0, 1), (4, 8, 48)), (t[1:2, :3], (3, 0, 8)), (t[:1].expand(3, 6, 8), (6, 0, 8))]:
        inner, outer, step = got = row_strides(view)
        assert got == want
        index = torch.arange(t.numel()).view(t.shape).as_strided(view.shape, view.stride(), view.storage_offset())
        rows = index[..., 0].reshape(-1)
        assert [view.storage_offset() + n // inner * outer + n % inner * step for n in range(rows.numel())] == rows.tolist()
    assert row_strides(torch.zeros(3, 0, 8)) == (1, 0, 0) and row_strides(torch.zeros(5, 1)) == (5, 0, 1)
    for copied in (torch.zeros(2, 3, 4, 8).permute(2, 1, 0, 3), torch.zeros(8, 4).t()):
        assert row_strides(copied) is None


@pytest.mark.parametrize("temperature,wt,wl", [(1.0, 1.0, 0.0), (2.0, 0.5, 0.5), (0.5, 0.0, 1.0)])
def test_definition_of_the_distillation(temperature, wt, wl):
    """Gradient against differences; the two terms against torch's losses on rows where they say the same."""
    torch.manual_seed(3)
    x, t = torch.randn(4, 11).double() * 2, torch.randn(4, 5).double() * 2
    ids = torch.stack([torch.randperm(11)[:5] for _ in range(4)])
    ids[1, 3:] = -1
    ids[2, 1] = ids[2, 0]
    labels = torch.tensor([3, -100, 0, 10])

    def loss(x):
        return ref.distill(x, t, ids, temperature, labels, wt, wl)[0]

    _, _, grad, _ = ref.distill(x, t, ids, temperature, labels, wt, wl)
    h = 1e-5
    for n in range(4):
        for v in range(11):
            e = torch.zeros_like(x)
            e[n, v] = h
            assert abs((loss(x + e) - loss(x - e)) / (2 * h) - grad[n, v]) < 1e-8
    full = torch.randn(4, 11).double()
    every = torch.arange(11).expand(4, 11)
    got = ref.distill(x, full, every, temperature, labels, wt, wl, reduction="none")[0]
    kd = torch.nn.functional.kl_div(torch.log_softmax(x / temperature, -1), torch.softmax(full / temperature, -1), reduction="none").sum(-1)
    ce = torch.nn.functional.cross_entropy(x, labels, reduction="none")
    want = torch.where(labels == -100, 0.0, wt * temperature ** 2 * kd + wl * ce)
    assert torch.allclose(got, want, atol=1e-12)


def test_definition_of_the_balance():
    torch.manual_seed(4)
    r = torch.randn(2, 7, 5).double()
    ids = torch.randint(-1, 5, (2, 7, 2))
    mask = torch.rand(2, 7) < 0.7
    _, _, counts, grad, _ = ref.balance(r, ids, mask, 0.3, 0.1)
    assert int(counts.sum()) == int(((ids >= 0) & mask.unsqueeze(-1)).sum())
    h = 1e-5
    for g in range(2):
        for n in range(7):
            for e in range(5):
                d = torch.zeros_like(r)
                d[g, n, e] = h
                want = (ref.balance(r + d, ids, mask, 0.3, 0.1)[0] - ref.balance(r - d, ids, mask, 0.3, 0.1)[0]) / (2 * h)
                assert abs(want - grad[g, n, e]) < 1e-8
    even = torch.zeros(8, 4)
    assert abs(ref.balance(even, torch.arange(8).view(8, 1) % 4)[0] - 1.0) < 1e-12


def test_a_missing_host_side_is_an_error(monkeypatch):
    import sys

    import lpmm
    from lpmm import _native

    _native.losses()
    monkeypatch.setattr(_native, "_losses", None)
    monkeypatch.delattr(lpmm, "_losses")
    monkeypatch.setitem(sys.modules, "lpmm._losses", None)
    with pytest.raises(RuntimeError, match="does not load"):
        F.distill_loss(**_distill_inputs())
    with pytest.raises(RuntimeError, match="does not load"):
        F.balance_loss(torch.randn(5, 8), torch.zeros(5, 2, dtype=torch.int64))
