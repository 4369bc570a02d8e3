"""Few rows: nothing of a product is cut, whatever the result's type.  Large products that cancel stand beside small ones, which the e4m3 matrix instruction alone would
drop (they lie more than 2^-13 below); every sum is a small integer, so the results are compared to the bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
q = pytest.importorskip("quantised_bayesian_nets_amd")
DEV = "cuda"


def operands(seed, *lead, R, N, K):
    """x [.., R, K] and w [.., N, K]: 448 at even columns of both, of changing sign in w, and integers to +-3 at odd ones."""
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randint(-3, 4, (*lead, R, K), generator=g).float(), torch.randint(-3, 4, (*lead, N, K), generator=g).float()
    x[..., ::2] = 448.0
    w[..., ::4], w[..., 2::4] = 448.0, -448.0
    return x, w


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("S,B,N,K", [(1, 1, 40, 128), (1, 16, 300, 1000), (3, 5, 129, 260), (2, 16, 16, 2048)])
def test_small_products_beside_large_ones(S, B, N, K, out):
    x, w = operands(1, S, R=B, N=N, K=K)
    want = x.double() @ w.double().transpose(1, 2)
    y = q.linear_fp8(x.to(DEV), q.quantize_fp8(w.to(DEV), 128), out_dtype=out)
    if out == torch.float8_e4m3fn:
        t = q.quantize_fp8(want.float().to(DEV))
        assert torch.equal(y.data.view(torch.uint8), t.data.view(torch.uint8)) and torch.equal(y.exponent, t.exponent)
    else:
        assert torch.equal(y.cpu(), want.to(out)) and int((want != 0).sum()) > want.numel() // 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,k,D,H", [(1, 4, 2, 128, 40), (20, 6, 3, 600, 300), (64, 8, 2, 1000, 130)])
def test_experts_hidden_rows(T, E, k, D, H, dtype):
    """The first product's sums; the second product hands the hidden values on."""
    x, w = operands(2, R=T, N=E * H, K=D)
    up, down = w.reshape(E, H, D), torch.eye(H).expand(E, H, H).contiguous()
    r = q.route_experts(torch.randn(T, E, generator=torch.Generator().manual_seed(3)).to(DEV), k)
    r = q.Routing(torch.ones_like(r.weights), r.experts, r.offsets, r.rows, E)
    y = q.experts_fp8(x.to(DEV).to(dtype), r, q.quantize_fp8(up.to(DEV), 128), q.quantize_fp8(down.to(DEV), 128))
    h = torch.relu(x.double() @ w.double().T).reshape(T, E, H).float().to(DEV)
    h = q.quantize_fp8(h).dequantize(torch.float64)
    want = h.gather(1, r.experts.long()[..., None].expand(T, k, H)).sum(1)
    assert torch.equal(y, want.to(dtype))
