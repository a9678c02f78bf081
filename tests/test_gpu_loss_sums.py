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
