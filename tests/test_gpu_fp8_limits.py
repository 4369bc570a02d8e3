"""Calls of the 8-bit float operators at the ends of what the documentation allows."""
import numpy as np
import pytest
import torch

import f8_oracle as orc

pytestmark = pytest.mark.gpu
q = pytest.importorskip("quantised_bayesian_nets_amd")
DEV = "cuda"


def rnd(seed, *shape, by=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * by).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_more_groups_than_a_grid_axis_holds(dtype):
    """64 samples x 1024 experts, a row each: every sample equals a call of its own to the bit."""
    S, T, E, D, H, N = 64, 1024, 1024, 20, 24, 130
    up, down = q.quantize_fp8(rnd(1, E, H, D).to(DEV), 128), q.quantize_fp8(rnd(2, E, N, H).to(DEV), 128)
    x, l = rnd(3, S, T, D, dtype=dtype).to(DEV), rnd(4, S, T, E).to(DEV)
    r = q.route_experts(l, 1)
    y = q.experts_fp8(x, r, up, down)
    for s in (0, 1, 31, 62, 63):
        assert torch.equal(y[s], q.experts_fp8(x[s], q.route_experts(l[s], 1), up, down))
    assert torch.isfinite(y).all() and (y != 0).any(-1).all()


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
def test_more_samples_than_a_grid_axis_holds(out):
    S = 65541
    w, x = q.quantize_fp8(rnd(1, 40, 100).to(DEV), 128), rnd(2, S, 2, 100).to(DEV)
    y = q.linear_fp8(x, w, out_dtype=out)
    for a in (0, 32767, 65535, S - 1):
        z = q.linear_fp8(x[a], w, out_dtype=out)
        if out == torch.float8_e4m3fn:
            assert torch.equal(y.data[a].view(torch.uint8), z.data.view(torch.uint8)) and torch.equal(y.exponent[a], z.exponent)
        else:
            assert torch.equal(y[a], z)


def test_quantiser_of_more_blocks_than_a_launch_takes():
    """2^24 workgroups of 256 threads are more than one launch's threads: matrices of one row, whose blocks of 128 x 128 are those of 1 x 128."""
    x = torch.randn((1 << 24) + 77, 1, 5, generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    a, b = q.quantize_fp8(x, 128), q.quantize_fp8(x)
    for t in (slice(0, 1000), slice((1 << 23) - 500, (1 << 23) + 500), slice(-1000, None)):
        assert torch.equal(a.data[t].view(torch.uint8), b.data[t].view(torch.uint8)) and torch.equal(a.exponent[t], b.exponent[t])
    assert torch.equal(a.data.view(torch.int32), b.data.view(torch.int32)) and torch.equal(a.exponent, b.exponent)


def check_rows(x, r, up, down, y, at):
    """Rows `at` of a bfloat16 call against the 64-bit form."""
    xv = orc.quantised(x[at].double().cpu().numpy(), 1)[None]
    uv, dv = (w.dequantize(torch.float64).cpu().numpy() for w in (up, down))
    want, bound = orc.experts(xv, r.weights[at].double().cpu().numpy()[None], r.experts[at].cpu().numpy()[None], lambda s, e: uv[e], lambda s, e: dv[e], None, None, "bfloat16")
    assert (np.abs(y[at].double().cpu().numpy() - want[0]) <= bound[0]).all()


@pytest.mark.parametrize("T,k,D,H,N", [(1 << 18, 5, 128, 4096, 128), ((1 << 20) + 200, 2, 4096, 128, 32)], ids=["hidden rows", "gathered rows"])
def test_rows_past_4_gib(T, k, D, H, N):
    """Rows on both sides of the first 4 GiB of the rows that a product reads."""
    g = torch.Generator(DEV).manual_seed(1)
    x = torch.randn(T, D, generator=g, device=DEV, dtype=torch.bfloat16)
    l = torch.randn(T, 8, generator=g, device=DEV)
    up, down = q.quantize_fp8(rnd(2, 8, H, D, by=D ** -0.5).to(DEV), 128), q.quantize_fp8(rnd(3, 8, N, H).to(DEV), 128)
    r = q.route_experts(l, k, renormalize=True)
    y = q.experts_fp8(x, r, up, down)
    for first in (0, T // 2, (1 << 20) - 8 if T > 1 << 20 else T - 40000, T - 16):
        check_rows(x, r, up, down, y, slice(first, first + 16))


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
