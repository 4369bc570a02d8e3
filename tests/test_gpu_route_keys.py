"""What the router compares: keys in 64 bits; of equal ones, where there is one group, the larger logit first, and then the lowest index.  A bias that is the same for every
expert changes no choice, however far the scores are saturated."""
import numpy as np
import pytest
import torch

import f8_oracle as orc

pytestmark = pytest.mark.gpu
q = pytest.importorskip("quantised_bayesian_nets_amd")
DEV = "cuda"


def by_logit(l, k):
    """The k largest logits of each row, ties to the lowest index."""
    return (-l.double()).argsort(dim=-1, stable=True)[..., :k].int()


def choose(l, k, score, bias, **kw):
    return q.route_experts(l.to(DEV), k, score=score, bias=None if bias is None else torch.full((l.shape[-1],), bias, device=DEV), **kw)


@pytest.mark.parametrize("bias", [None, 0.0, 0.5, 1e6])
def test_two_saturated_scores(bias):
    assert choose(torch.tensor([[40.0, 41.0]]), 1, "sigmoid", bias).experts.tolist() == [[1]]
    assert choose(torch.tensor([[-800.0, -760.0, -900.0]]), 2, "sigmoid", bias).experts.tolist() == [[1, 0]]
    assert choose(torch.tensor([[0.0, -900.0, -800.0]]), 2, "softmax", bias).experts.tolist() == [[0, 2]]
    assert choose(torch.tensor([[1.0, 1e-20, 3e-20, 2e-20]]), 3, "softmax", bias).experts.tolist() == [[0, 2, 3]]


@pytest.mark.parametrize("E,k", [(5, 3), (16, 8), (60, 4), (256, 8), (1000, 32)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_a_constant_bias_changes_no_choice(dtype, E, k):
    g = torch.Generator().manual_seed(E)
    for score, low, high in (("sigmoid", 20, 60), ("sigmoid", -1000, -700), ("sigmoid", -1000, 60), ("softmax", -2000, 0), ("softmax", -4, 4)):
        l = (low + (high - low) * torch.rand(70, E, generator=g)).to(dtype)
        l[3], l[4, ::2], l[5, 1::3] = l[3, 0], float("-inf"), l[5, 1]
        want = by_logit(l, k)
        for bias in (None, 0.0, 0.5, 1e6):
            r = choose(l, k, score, bias)
            masked = torch.isinf(l.gather(-1, want.long()))
            got = r.experts.cpu()
            assert torch.equal(torch.where(masked, -1, got), torch.where(masked, -1, want)), (score, bias)
            assert (l.gather(-1, got.long())[masked] == float("-inf")).all()
            off, rows = orc.order_of(got.numpy()[None], E)
            assert np.array_equal(r.offsets.cpu().numpy(), off) and np.array_equal(r.rows.cpu().numpy(), rows)


@pytest.mark.parametrize("bias", [None, 0.0, 0.5])
def test_an_infinite_logit_is_chosen_under_a_bias_too(bias):
    l = torch.randn(3, 40, generator=torch.Generator().manual_seed(1))
    l[1, 6] = l[1, 30] = float("inf")
    for score in ("softmax", "sigmoid"):
        r = choose(l, 4, score, bias)
        assert torch.equal(r.experts.cpu(), by_logit(l, 4))
        assert torch.isfinite(r.weights[[0, 2]]).all()
    assert (choose(l, 2, "sigmoid", bias).weights[1] == 1).all() and torch.isnan(choose(l, 4, "softmax", bias).weights[1]).all()


@pytest.mark.parametrize("bias", [False, True])
def test_several_groups_settle_equal_keys_by_the_index(bias):
    """Scores of 1 to the last bit of 64: neither a group nor an expert is preferred for its logit."""
    l = 40 + 20 * torch.rand(20, 32, generator=torch.Generator().manual_seed(2))
    r = choose(l, 5, "sigmoid", 0.25 if bias else None, groups=4, top_groups=2)
    assert torch.equal(r.experts.cpu(), torch.arange(5).int().expand(20, 5))
