"""balance_loss on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

import lpmm.functional as F
import losses_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(shape, experts, picks, dtype=torch.float32, seed=0, mask=True):
    g = torch.Generator().manual_seed(seed * 1000003 + experts * 31 + sum(shape))
    r = (torch.randn(*shape, experts, generator=g) * 2).to(dtype)
    ids = torch.rand(*shape, experts, generator=g).argsort(dim=-1)[..., :picks]
    ids = ids.masked_fill(torch.rand(*shape, picks, generator=g) < 0.1, -1)
    return r, ids, (torch.rand(*shape, generator=g) < 0.8) if mask else None


def _check(r, ids, mask=None, weight=0.5, z_weight=0.0, scale=None, move=lambda t: t.cuda(), what=""):
    leaf = move(r).detach().requires_grad_(True)
    on = None if mask is None else mask.cuda()
    loss, counts = F.balance_loss(leaf, ids.cuda(), mask=on, weight=weight, z_weight=z_weight)
    assert loss.dtype == torch.float32 and counts.dtype == torch.int64 and not counts.requires_grad
    (loss if scale is None else loss * scale).backward()
    want, bound, wcounts, grad, gbound = ref.balance(r, ids, mask, weight, z_weight, 1.0 if scale is None else scale)
    assert torch.equal(counts.cpu(), wcounts), what
    ref.assert_within(loss, want, bound, what + " loss")
    ref.assert_within(leaf.grad, grad, gbound, what + " gradient")
    with torch.no_grad():
        again, c = F.balance_loss(leaf, ids.cuda(), mask=on, weight=weight, z_weight=z_weight)
    assert torch.equal(again, loss.detach()) and torch.equal(c, counts) and not again.requires_grad
    return loss.detach(), counts, leaf.grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("experts", [1, 2, 3, 4, 5, 7, 8, 16, 17, 31, 60, 64, 65, 127, 128, 160, 255, 256, 257, 384, 500, 512, 513, 1000, 1023, 1024])
def test_numbers_of_experts(experts, dtype):
    scale = 1024.0 if dtype == torch.float16 else None
    for tokens in (1, 3, 70):
        r, ids, mask = _inputs((tokens,), experts, min(experts, 4), dtype)
        print(dtype, experts, tokens, flush=True)
        _check(r, ids, what=f"{tokens} x {experts}", scale=scale)
        _check(r, ids, mask, 0.01, 0.001, scale=scale, what=f"{tokens} x {experts} masked")


@pytest.mark.parametrize("tokens", [0, 1, 2, 63, 64, 65, 127, 129, 255, 257, 1023, 4097, 20000])
def test_numbers_of_tokens(tokens):
    r, ids, mask = _inputs((tokens,), 24, 3)
    _check(r, ids, z_weight=0.1)
    _check(r, ids.int(), mask, z_weight=0.1)


@pytest.mark.parametrize("groups,tokens", [(0, 5), (1, 77), (3, 0), (2, 1), (3, 130), (16, 257), (255, 5), (256, 5), (700, 3), (5, 3000)])
def test_groups(groups, tokens):
    r, ids, mask = _inputs((groups, tokens), 12, 2)
    _check(r, ids, mask, z_weight=0.1)
    if groups > 1 and tokens:
        mask[1] = False  # a group without tokens
        _, counts, grad = _check(r, ids, mask, z_weight=0.1)
        assert not counts[1].any() and not grad[1].any()


@pytest.mark.parametrize("picks", [0, 1, 5, 8, 32])
def test_numbers_of_picks(picks):
    r, ids, mask = _inputs((301,), 32, picks)
    _check(r, ids, mask, z_weight=0.1)


@pytest.mark.parametrize("weight,z_weight", [(0.0, 0.0), (1.0, 0.0), (0.0, 1.0), (-2.0, 0.5), (1e-4, 1e3)])
def test_weights_and_gradients(weight, z_weight):
    r, ids, mask = _inputs((3, 100), 20, 2)
    for scale in (None, 0.0, -2.5):
        _check(r, ids, mask, weight, z_weight, scale)


def test_the_same_pick_twice_and_none_at_all():
    r, ids, mask = _inputs((90,), 12, 3)
    ids[:, 1] = ids[:, 0]
    _check(r, ids, mask)
    ids[:] = -7
    loss, counts, grad = _check(r, ids, mask)
    assert float(loss) == 0.0 and not counts.any() and not grad.any()
    _check(r, torch.zeros_like(ids), mask, z_weight=0.1)
    loss, counts, grad = _check(r, ids, torch.zeros_like(mask), z_weight=0.1)
    assert float(loss) == 0.0 and not grad.any()


def test_masked_tokens_may_hold_anything():
    for dtype in TYPES:
        r, ids, mask = _inputs((200,), 24, 3, dtype)
        out = (~mask).nonzero().view(-1)
        r[out[0]], r[out[1]], r[out[2]] = math.nan, math.inf, -math.inf
        ids[out[0]], ids[out[1]] = 24, 1 << 40
        _check(r, ids, mask, z_weight=0.1, scale=1024.0)


def test_masked_experts():
    for dtype in TYPES:
        r, ids, mask = _inputs((100,), 24, 2, dtype)
        r[:, 5] = -math.inf
        r[3, 1:] = -math.inf
        r[4] = torch.finfo(dtype).min
        r[5, 3:] = torch.finfo(dtype).min
        _check(r, ids, mask, scale=1024.0)


def test_what_is_wrong_is_nan():
    r, ids, mask = _inputs((3, 100), 24, 2)
    mask[1, 7], ids[1, 7, 0] = True, 24
    leaf = r.cuda().requires_grad_(True)
    loss, counts = F.balance_loss(leaf, ids.cuda(), mask=mask.cuda())
    loss.backward()
    assert loss.isnan() and leaf.grad[1][mask[1].cuda()].isnan().all() and not leaf.grad[0].isnan().any() and not leaf.grad[2].isnan().any()
    assert not leaf.grad[1][~mask[1].cuda()].any()
    ids[1, 7, 0] = 0
    assert torch.equal(counts.cpu(), ref.balance(r, ids, mask)[2] - torch.nn.functional.one_hot(torch.tensor([[24], [0], [24]]), 25)[:, 0, :24])
    for bad in (math.nan, math.inf):
        r[2, 3, 1], mask[2, 3] = bad, True
        leaf = r.cuda().requires_grad_(True)
        loss, _ = F.balance_loss(leaf, ids.cuda(), mask=mask.cuda())
        loss.backward()
        assert loss.isnan() and leaf.grad[2, 3].isnan().all()
        assert not leaf.grad[0].isnan().any()


def test_strided_logits():
    r, ids, mask = _inputs((6, 50), 24, 2)
    on = r.cuda()
    for name, view in (("shift", lambda a: a[:, :-1]), ("swapped", lambda a: a.transpose(0, 1)), ("one", lambda a: a[2]), ("step", lambda a: a[:, ::3])):
        _check(view(r), view(ids), view(mask), z_weight=0.1, move=lambda _: view(on), what=name)
    wide = torch.randn(6, 50, 40, device="cuda")[..., 5:29]
    _check(wide.cpu(), ids, mask, z_weight=0.1, move=lambda _: wide, what="columns")
    turned = on.transpose(1, 2).contiguous().transpose(1, 2)
    _check(r, ids, mask, z_weight=0.1, move=lambda _: turned, what="values apart")
    half = torch.zeros(6 * 50 * 24 + 3, dtype=torch.bfloat16, device="cuda")
    at = half[3:].view(6, 50, 24)
    at.copy_(on)
    _check(at.cpu(), ids, mask, move=lambda _: at, what="odd address")
    base = r[:, :1].cuda().requires_grad_(True)
    F.balance_loss(base.expand(6, 50, 24), ids.cuda(), mask=mask.cuda(), z_weight=0.1)[0].backward()
    _, _, _, grad, gbound = ref.balance(r[:, :1].expand(6, 50, 24), ids, mask, 1.0, 0.1)
    ref.assert_within(base.grad, grad.sum(1, keepdim=True), gbound.sum(1, keepdim=True) + 50 * ref.U * grad.abs().sum(1, keepdim=True), "broadcast")


def test_same_results_every_time():
    r, ids, mask = _inputs((30000,), 96, 4)
    first = _check(r, ids, mask, z_weight=0.01)
    for _ in range(3):
        again = _check(r, ids, mask, z_weight=0.01)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_several_passes_and_losses_that_nobody_wants():
    r, ids, mask = _inputs((100,), 24, 2)
    leaf = r.cuda().requires_grad_(True)
    loss, counts = F.balance_loss(leaf, ids.cuda(), mask=mask.cuda())
    one = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
    kept = one.clone()
    one.zero_()
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], kept)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(F.balance_loss(leaf, ids.cuda())[1].float().sum(), leaf)
    loss, _ = F.balance_loss(leaf, ids.cuda())
    with torch.no_grad():
        leaf.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_captured_and_replayed_on_two_streams():
    held = [[a.cuda() for a in _inputs((5, 300), 40, 4, seed=3)] for _ in range(2)]

    def step(r, ids, mask):
        leaf = r.detach().requires_grad_(True)
        loss, counts = F.balance_loss(leaf, ids, mask=mask, weight=0.1, z_weight=0.01)
        return loss, counts, torch.autograd.grad(loss, leaf)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for s in held:
            step(*s)
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [], []
    for s in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*s))
        graphs.append(g)
    others = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        new = [_inputs((5, 300), 40, 4, seed=4 + 2 * turn + k) for k in range(2)]
        for k in range(2):
            for a, b in zip(held[k], new[k]):
                a.copy_(b)
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(others[k]):
                graphs[k].replay()
        eager = [step(*[a.cuda() for a in new[k]]) for k in range(2)]
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], eager[k])), f"turn {turn}, graph {k}"


def test_nothing_is_written_past_the_tokens():
    from lpmm import _native

    r, ids, mask = (a.cuda() for a in _inputs((3, 67), 13, 2, torch.bfloat16))
    lib = _native.lib()
    pad = 64
    sizes = ((1, torch.float32), (39, torch.int64), (45, torch.float32), (lib.lpmm_balance_work_bytes(3, 67, 13), torch.uint8), (3 * 67 * 13, torch.bfloat16))
    room = [torch.full((n + 2 * pad,), 7, dtype=d, device="cuda") for n, d in sizes]
    loss, counts, factors, work, grad = (a[pad:].data_ptr() for a in room)
    record = ref.BALANCE_CALL.pack(r.data_ptr(), ids.data_ptr(), mask.data_ptr(), loss, counts, factors, work, grad, 3, 67, 13, 2, 67 * 13, 13,
                                       0.5, 0.1, ref.TYPE_BF16, 64)
    one = torch.ones(1, device="cuda")
    assert lib.lpmm_balance_loss(record, _native.current_stream(0)) == 0
    assert lib.lpmm_balance_loss_grad(record, one.data_ptr(), _native.current_stream(0)) == 0
    torch.cuda.synchronize()
    for a in room:
        assert (a[:pad] == 7).all() and (a[-pad:] == 7).all()
    _, _, wcounts, wgrad, gbound = ref.balance(r.cpu(), ids.cpu(), mask.cpu(), 0.5, 0.1)
    assert torch.equal(room[1][pad:-pad].view(3, 13).cpu(), wcounts)
    ref.assert_within(room[4][pad:-pad].view(3, 67, 13), wgrad, gbound, "gradient")


@pytest.mark.parametrize("shape,experts", [((65535, 1), 5), ((65535, 2), 1024), ((1 << 22,), 2)])
def test_the_most_groups_and_many_tokens(shape, experts):
    """Each group by itself is what a call on some of them gives, up to the division by their number."""
    r = torch.randn(*shape, experts, device="cuda").to(torch.bfloat16).requires_grad_(True)
    ids = torch.randint(0, experts, (*shape, 1), device="cuda")
    loss, counts = F.balance_loss(r, ids, weight=0.5, z_weight=0.1)
    grad = torch.autograd.grad(loss, r)[0]
    assert int(counts.sum()) == ids.numel() and loss.isfinite() and not grad.isnan().any()
    if len(shape) == 2:
        some = slice(shape[0] - 8, shape[0])
        want, bound, wcounts, wgrad, gbound = ref.balance(r.detach()[some].cpu(), ids[some].cpu(), None, 0.5, 0.1, 8.0 / shape[0])
        assert torch.equal(counts[some].cpu(), wcounts)
        ref.assert_within(grad[some], wgrad, gbound, "gradient")
    else:
        want, bound, wcounts, wgrad, gbound = ref.balance(r.detach().cpu(), ids.cpu(), None, 0.5, 0.1)
        assert torch.equal(counts.cpu(), wcounts)
        ref.assert_within(loss, want, bound, "loss")
        ref.assert_within(grad, wgrad, gbound, "gradient")
