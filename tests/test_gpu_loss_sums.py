"""How far the sums in the training-loss terms may be off: bounds of the longest chains of additions that the kernels have, and inputs
whose sums are whole numbers, where one value left out or taken twice shows."""
import pytest
import torch

import lpmm.functional as F
import losses_ref as ref

pytestmark = pytest.mark.gpu

U = ref.U
TURNS = 128  # tokens at most whose probabilities a thread adds in 32 bits


def _softmax_bound(r):
    """Relative error of a probability: three roundings of |d| and two half steps in its exponential; the sum's terms as much, with 16 of them in
    a lane and 6 exchanges; reciprocal and product."""
    d = r - r.amax(dim=-1, keepdim=True)
    p = torch.softmax(r, dim=-1)
    return U * (3 * d.abs() + 2 + 3 * (p * d.abs()).sum(dim=-1, keepdim=True) + 2 + 22 + 3)


@pytest.mark.parametrize("dtype,experts", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float32, 1000)])
def test_long_groups_of_identical_tokens(dtype, experts):
    """2^18 tokens, 16 of them a turn: where one workgroup takes a group, as it does with more than 512 of them unless they are cut for this, a
    thread adds 16384 values, and in 32 bits that drifts by 1e-4."""
    groups, tokens = 513, 16 * 16384
    g = torch.Generator().manual_seed(experts)
    one = (torch.randn(experts, generator=g) * 0.7).to(dtype)
    r = one.cuda().expand(groups, tokens, experts)
    ids = torch.zeros(1, 1, 1, dtype=torch.int32, device="cuda").expand(groups, tokens, 1)
    loss, counts = F.balance_loss(r, ids)
    assert counts[:, 0].eq(tokens).all() and not counts[:, 1:].any()
    x = one.double()
    want = experts * torch.softmax(x, dim=-1)[0]
    # in a thread, over two exchanges of lanes, over 4 waves; workgroups in 64 bits; the loss in 32
    bound = want * (_softmax_bound(x)[0] + U * (TURNS + 2 + 3 + 1))
    ref.assert_within(loss, want, bound, "loss")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sums_over_tokens_of_any_number(dtype):
    """A thread's chain, the exchanges of its lanes (6 at most) and the 4 waves are all that 32 bits add up, however many tokens there are."""
    for groups, tokens, experts, picks in [(1, 5, 24, 2), (1, 300, 8, 2), (1, 9001, 96, 4), (1, 140000, 24, 2), (3, 70001, 60, 4), (1, 1 << 20, 33, 1),
                                           (700, 4099, 16, 2)]:
        g = torch.Generator(device="cuda").manual_seed(tokens + experts)
        r = (torch.randn(groups, tokens, experts, device="cuda", generator=g) * 2).to(dtype)
        ids = torch.randint(0, experts, (groups, tokens, picks), device="cuda", generator=g)
        loss, counts = F.balance_loss(r, ids)
        want = bound = 0.0
        for n in range(groups):
            x = r[n].double()
            c = torch.bincount(ids[n].view(-1), minlength=experts)
            assert torch.equal(counts[n], c)
            p = torch.softmax(x, dim=-1)
            share = experts * c.double() / (tokens * tokens * picks) / groups
            want += float((share * p.sum(dim=0)).sum())
            bound += float((share * (p * (_softmax_bound(x) + U * (min(tokens, TURNS) + 6 + 3 + 1))).sum(dim=0)).sum())
        ref.assert_within(loss, torch.tensor(want).double(), torch.tensor(bound).double(), f"{groups} x {tokens} x {experts} {dtype}")


def _exact_balance(shape, experts, picks, dtype, mask):
    """Tokens that are sure of one expert: a probability of 1 and the others 0, logsumexp a small whole number.  Sums are whole numbers, and the only
    rounding is that of the loss."""
    g = torch.Generator().manual_seed(experts * 7 + sum(shape))
    groups, tokens = (shape if len(shape) == 2 else (1, *shape))
    sure = torch.randint(0, experts, (groups, tokens), generator=g).cuda()
    level = torch.randint(0, 4, (groups, tokens), generator=g).cuda()
    ids = torch.randint(-1, experts, (groups, tokens, picks), generator=g).cuda()
    seen = (torch.rand(groups, tokens, generator=g) < 0.9).cuda() if mask else torch.ones(groups, tokens, dtype=torch.bool, device="cuda")
    r = torch.full((groups, tokens, experts), -200.0, device="cuda", dtype=dtype)
    r.scatter_(2, sure.unsqueeze(-1), 0.0)
    r += level.unsqueeze(-1).to(dtype)
    loss, counts = F.balance_loss(r.view(*shape, experts), ids.view(*shape, picks), mask=seen.view(shape) if mask else None, weight=1.0, z_weight=0.5)
    want = 0.0
    for n in range(groups):
        on = seen[n]
        T = int(on.sum())
        c = torch.bincount(ids[n][on].view(-1) + 1, minlength=experts + 1)[1:]
        assert torch.equal(counts.view(groups, experts)[n], c)
        sums = torch.bincount(sure[n][on], minlength=experts)
        if T:
            want += experts * int((c * sums).sum()) / (T * T * picks) + 0.5 * int((level[n][on] ** 2).sum()) / T
    want = torch.tensor(want / groups, dtype=torch.float64)
    ref.assert_within(loss, want, 1.001 * U * want, f"loss of {shape} x {experts}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("mask", [False, True])
def test_every_token_is_counted_once(dtype, mask):
    """Groups of one workgroup and of many; 140000 tokens: 137 to each of 1022 workgroups, and none to the last two of the 1024."""
    for shape, experts, picks in [((1,), 3, 1), ((128,), 17, 2), ((129,), 60, 3), ((20000,), 256, 8), ((65537,), 64, 2), ((140000,), 24, 2),
                                  ((140001,), 130, 4), ((300007,), 8, 2), ((3, 70001), 33, 2), ((600, 2051), 40, 2), ((1025, 130), 5, 1)]:
        print(dtype, mask, shape, experts, flush=True)
        _exact_balance(shape, experts, picks, dtype, mask)


def test_every_token_of_four_million_is_counted_once():
    """More workgroups than the join has threads: 2^22 + 77 tokens are cut into 2049 of 2048."""
    _exact_balance(((1 << 22) + 77,), 64, 1, torch.bfloat16, True)


def _exact_distill(rows, vocab, dtype, share, temperature, wt, wl):
    """Logits of 0 or so low that they count nothing, a teacher with one entry, and a label: the sum of a row's exponentials is the number of its zeros,
    the loss its logarithm, the gradient its reciprocal."""
    g = torch.Generator(device="cuda").manual_seed(vocab * 13 + rows)
    live = torch.rand(rows, vocab, device="cuda", generator=g) < share
    label = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    entry = torch.randint(0, vocab, (rows, 1), device="cuda", generator=g)
    live.scatter_(1, label.unsqueeze(1), True).scatter_(1, entry, True)
    x = torch.where(live, 0.0, -400.0).to(dtype).requires_grad_(True)
    up = 4096.0 if dtype == torch.float16 else 1.0  # whose smallest numbers would be lost
    loss = F.distill_loss(x, torch.zeros(rows, 1, device="cuda"), entry, temperature=temperature, labels=label, teacher_weight=wt, label_weight=wl,
                          reduction="none")
    grad = torch.autograd.grad(loss, x, torch.full((rows,), up, device="cuda"))[0]
    n = live.sum(dim=1).double()
    what = f"{rows} x {vocab} {dtype} {share} T={temperature}"
    # a logarithm is off by one step, then four products or sums; one value more or less in n moves it by 1 / n
    want = ((wt * temperature ** 2 + wl) * n.log()).cpu()
    ref.assert_within(loss, want, 8 * U * want, what + " loss")
    each = (wt * temperature + wl) * up
    # the reciprocals, their products with weights and factor, the sums with what entry and label take off
    smooth = each / n.unsqueeze(1)
    wrong = torch.where(live, (grad - smooth).abs() - (8 * U + ref.step(dtype)) * smooth - ref.SMALLEST[dtype], grad.abs())
    off = torch.zeros(rows, vocab, dtype=torch.bool, device="cuda").scatter_(1, label.unsqueeze(1), True).scatter_(1, entry, True)
    assert not (wrong.masked_fill(off, 0.0) > 0).any(), what
    for ids, weight in ((entry, wt * temperature), (label.unsqueeze(1), wl)):
        both = entry == label.unsqueeze(1)
        want = smooth - torch.where(both, each, weight * up)
        got = grad.gather(1, ids).double()
        assert ((got - want).abs() <= 8 * U * each + ref.step(dtype) * want.abs()).all(), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [3, 257])
def test_every_value_of_a_row_is_counted_once(rows, dtype):
    """At the ends of what each kind of workgroup holds, and past all of them."""
    run = 4 if dtype == torch.float32 else 8
    for held in (1, 256 * 4, 256 * 8, 512 * 8, 1024 * 7, 1024 * 8, 1024 * 16):
        for vocab in sorted({held * run - 1, held * run, held * run + run, held * run + run + 3}):
            print(dtype, rows, vocab, flush=True)
            _exact_distill(rows, vocab, dtype, 1.0, 1.0, 0.5, 0.5)
            _exact_distill(rows, vocab, dtype, 0.8, 2.0, 0.25, 0.5)
    for vocab in (777, 9001, 50257, 137 * run * 1024 // 8 + 5):
        _exact_distill(rows, vocab, dtype, 0.5, 1.5, 0.5, 0.25)
        _exact_distill(rows, vocab, dtype, 0.001, 1.0, 1.0, 0.5)  # most first runs say nothing of the rest


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 1.5])
def test_rows_of_millions_of_values(dtype, temperature):
    """2^24 values that are alike but for every thread's first: 16384 to a thread, in which one chain of 32-bit additions drifts by 1e-4."""
    vocab, low = (1 << 24) + 5, -4.28125
    x = torch.full((1, vocab), low, device="cuda", dtype=dtype)
    x[:, : 1024 * 8 + 16] = 0.0
    x[:, -9:] = 0.0
    x.requires_grad_(True)
    label = torch.tensor([vocab // 2], device="cuda")
    entry = torch.tensor([[5]], device="cuda")
    loss = F.distill_loss(x, torch.zeros(1, 1, device="cuda"), entry, temperature=temperature, labels=label, teacher_weight=1.0, label_weight=0.5)
    grad = torch.autograd.grad(loss, x)[0]
    n = 1024 * 8 + 16 + 9
    some = torch.tensor([0.0, low], dtype=torch.float64)
    sums = [(n + (vocab - n) * torch.exp(some[1] / t)) for t in (temperature, 1.0)]
    want = temperature ** 2 * sums[0].log() + 0.5 * (sums[1].log() - low)
    # a term of the sum: three roundings of its exponent and two half steps; 128 additions in a thread, 6 and 10 to join
    off = U * (3 * -low / min(temperature, 1.0) + 2 + 128 + 16)
    ref.assert_within(loss, want, (temperature ** 2 + 0.5) * off + 8 * U * want, "loss")
    for at, v in ((vocab // 3, low), (100, 0.0)):
        q = temperature * torch.exp(torch.tensor(v / temperature).double()) / sums[0] + 0.5 * torch.exp(torch.tensor(v).double()) / sums[1]
        ref.assert_within(grad[0, at], q, q * (off + U * (3 * -low / min(temperature, 1.0) + 10)), f"gradient of {v}")


def test_router_logits_past_32_bits():
    """The last of 9 million tokens of 256 experts lie past 2^31 values; alone they are what they are behind masked ones."""
    tokens, experts, last = 9_000_000, 256, 1000
    r = torch.empty(tokens, experts, device="cuda", dtype=torch.bfloat16).normal_().requires_grad_(True)
    ids = torch.randint(0, experts, (tokens, 2), device="cuda", dtype=torch.int32)
    mask = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    mask[-last:] = True
    loss, counts = F.balance_loss(r, ids, mask=mask, z_weight=0.1)
    grad = torch.autograd.grad(loss, r)[0]
    alone = r.detach()[-last:].clone().requires_grad_(True)
    want, wcounts = F.balance_loss(alone, ids[-last:], z_weight=0.1)
    assert torch.equal(counts, wcounts) and abs(float(loss.detach()) - float(want.detach())) <= 4 * U * float(want.detach())
    assert torch.equal(grad[-last:], torch.autograd.grad(want, alone)[0]) and not grad[:-last].any()
