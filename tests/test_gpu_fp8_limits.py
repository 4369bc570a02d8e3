"""Calls of the 8-bit float operators at the ends of what the documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
q = pytest.importorskip("quantised_bayesian_nets_amd")
DEV = "cuda"


def rnd(seed, *shape, by=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * by).to(dtype)


def test_forward_mode_derivatives_are_refused():
    """A dual's tangent would be lost without a word."""
    from torch.autograd import forward_ad
    w = q.quantize_fp8(rnd(1, 40, 100).to(DEV), 128)
    x, l = rnd(2, 3, 100).to(DEV), rnd(3, 3, 8).to(DEV)
    with forward_ad.dual_level():
        for call in (lambda: q.quantize_fp8(forward_ad.make_dual(x, x)), lambda: q.linear_fp8(forward_ad.make_dual(x, x), w),
                     lambda: q.linear_fp8(x, w, forward_ad.make_dual(x[0, :40].contiguous(), x[0, :40].contiguous())), lambda: q.route_experts(forward_ad.make_dual(l, l), 2)):
            with pytest.raises(RuntimeError, match="evaluates only"):
                call()
        assert q.linear_fp8(x, w).shape == (3, 40)
