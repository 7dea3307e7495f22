"""Routing calls of as many tokens as a sort takes: 2^24 pairs, whose rows are
placed, summed and differentiated in one launch each."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import minirun_hip as M

    M.load()
    return M


@pytest.mark.parametrize("tokens,per_token,dim", [(1 << 24, 1, 8), (1 << 24, 1, 3), (1 << 23, 2, 40), ((1 << 22) + 5, 4, 1)])
def test_as_many_tokens_as_a_sort_takes(M, tokens, per_token, dim):
    # whole numbers below 128: every product and sum is exact in bf16
    import torch

    experts = 5
    pairs = tokens * per_token
    pairs = min(pairs, 1 << 24) // per_token * per_token
    tokens = pairs // per_token
    i = torch.arange(pairs, device="cuda", dtype=torch.int32).reshape(tokens, per_token)
    o = M.expert_sort((i * 7 + i // 1000) % (experts + 1), experts)  # a sixth without a row
    n = int(o.offsets[-1])
    x = (torch.arange(tokens, device="cuda")[:, None] * 3 + torch.arange(dim, device="cuda")) % 11
    rows = M.expert_dispatch(x.bfloat16(), o, out=torch.full((pairs, dim), -3.0, device="cuda", dtype=torch.bfloat16))
    pair = o.pair_of_row[:n].long()
    assert torch.equal(rows[:n], x[pair // per_token].bfloat16())
    assert bool((rows[n:] == -3).all())
    has = o.row_of_pair >= 0
    weights = (i % 3).float()
    out = M.expert_combine(rows, o, weights)
    total = torch.where(has, weights, 0.0).sum(1, keepdim=True)
    assert torch.equal(out, (x * total).bfloat16())
    assert torch.equal(M.expert_dispatch_backward(rows, o), (x * has.sum(1, keepdim=True)).bfloat16())
    d_rows, d_weights = M.expert_combine_backward(x.bfloat16(), rows, o, weights)
    assert torch.equal(d_rows[:n], (x[pair // per_token] * weights.reshape(-1)[pair][:, None]).bfloat16())
    assert torch.equal(d_weights, torch.where(has, (x * x).sum(1, keepdim=True).float(), 0.0))
