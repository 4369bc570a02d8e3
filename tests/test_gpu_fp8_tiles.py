"""Every tile of the 8-bit float products, each shown to be the one that the call takes, on numbers for which nothing is rounded before the result: small integers times
a power of two for each block, whose products and partial sums are integers below 2^24.  Results are compared to the bit.  And the fast form's norm on normal data."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu
q = pytest.importorskip("quantised_bayesian_nets_amd")
from quantised_bayesian_nets_amd import _lib  # noqa: E402

DEV = "cuda"
TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3}
AT = 1 << 20      # an address that nothing reads


def ints(seed, rows, *shape, high=3, scales=3):
    """Integers to +-high times 2^0 .. 2^(scales - 1), one power for each block of `rows` x 128: exact in e4m3 blocks."""
    g = torch.Generator(DEV).manual_seed(seed)
    *lead, R, K = shape
    v = torch.randint(-high, high + 1, shape, generator=g, device=DEV).double()
    s = torch.randint(0, scales, (*lead, -(-R // rows), -(-K // 128)), generator=g, device=DEV)
    s = s.repeat_interleave(rows, -2)[..., :R, :].repeat_interleave(128, -1)[..., :K]
    return v * torch.exp2(s.double())


def dense_tile(S, sx, sw, B, N, K, out):
    kp = -(-K // 128) * 128
    sp = -(-kp // 512) * 4
    v = _lib.lib().qbnn_linear_f8_tile(_lib.F8_LINEAR.pack(0, 0, 0, AT, AT, B * kp if sx > 1 else 0, B * sp if sx > 1 else 0, AT, AT, N * kp if sw > 1 else 0,
                                                         -(-N // 128) * sp if sw > 1 else 0, 0, 0, AT, AT, B, N, K, S, 0, TYPE[out], 0))
    return v >> 16, v & 65535


FAST = [torch.bfloat16, torch.float16, torch.float8_e4m3fn]
BIG = [(16, 16, 16, 769, 1000, 100), (16, 16, 16, 769, 1000, 128), (16, 1, 16, 769, 1000, 129), (16, 16, 1, 769, 1000, 256), (16, 16, 16, 769, 1000, 300), (1, 1, 1, 3329, 3841, 512),
       (1, 1, 1, 3500, 3500, 513), (200, 200, 200, 130, 250, 256), (16, 16, 16, 800, 1024, 2048), (16, 16, 16, 769, 1000, 2176), (1, 1, 1, 4096, 4096, 4100)]
WIDE = [(400, 400, 400, 100, 250, 100), (400, 400, 1, 65, 256, 256), (400, 1, 400, 128, 129, 300), (100, 100, 100, 90, 1000, 2176)]
CASES = ([(out, (256, 256), c) for out in FAST for c in BIG] + [(out, (128, 256), c) for out in FAST + [torch.float32] for c in WIDE] + [(torch.float32, (128, 256), c) for c in BIG]
         + [(out, (128, 128), c) for out in FAST + [torch.float32] for c in [(100, 100, 100, 128, 500, 130), (70, 70, 70, 40, 500, 640), (300, 300, 1, 33, 100, 2176)]]
         + [(out, (64, 128), c) for out in FAST + [torch.float32] for c in [(3, 3, 3, 200, 260, 100), (1, 1, 1, 1000, 700, 2176), (2, 1, 2, 33, 129, 300)]]
         + [(out, (16, 16), c) for out in [torch.bfloat16, torch.float16, torch.float32] for c in [(1, 1, 1, 1, 40, 2176), (3, 1, 3, 16, 129, 100), (2, 2, 2, 5, 500, 300)]]
         + [(out, (32, 64), c) for out in [torch.bfloat16, torch.float16, torch.float32] for c in [(1, 1, 1, 17, 40, 2176), (3, 1, 3, 32, 129, 100)]]
         + [(torch.float8_e4m3fn, t, c) for t, c in [((16, 128), (1, 1, 1, 1, 40, 2176)), ((16, 128), (3, 1, 3, 16, 300, 100)), ((32, 128), (2, 2, 2, 17, 129, 300)), ((32, 128), (1, 1, 1, 32, 1000, 640))]])


@pytest.mark.parametrize("out,tile,size", CASES, ids=lambda v: str(v).replace("torch.", ""))
def test_dense(out, tile, size):
    S, sx, sw, B, N, K = size
    assert dense_tile(*size, out) == tile
    x, w = ints(1, 1, sx, B, K), ints(2, 128, sw, N, K)
    bias = torch.randint(-50, 50, (N,), generator=torch.Generator(DEV).manual_seed(3), device=DEV).float()
    wq, xf = q.quantize_fp8(w.float(), 128), x.float()
    assert torch.equal(wq.dequantize(torch.float64), w)
    want = torch.stack([x[s if sx > 1 else 0] @ w[s if sw > 1 else 0].T for s in range(S)])
    assert float(want.abs().max()) < 1 << 24
    for b, relu in ((None, False), (bias, True)):
        y = q.linear_fp8(xf, wq, b, relu=relu, out_dtype=out)
        v = want if b is None else (want + b.double()).clamp(min=0)
        if out == torch.float8_e4m3fn:
            t = q.quantize_fp8(v.float())
            assert torch.equal(y.data.view(torch.uint8), t.data.view(torch.uint8)) and torch.equal(y.exponent, t.exponent)
        else:
            assert torch.equal(y, v.to(out))


def experts_tiles(S, T, E, k, D, H, N, out):
    tiles = (C.c_int32 * 2)()
    exact = 0 if out == torch.bfloat16 else 1 if out == torch.float16 else 3
    _lib.check(_lib.lib().qbnn_experts_f8_tiles(_lib.F8_EXPERTS.pack(*[0] * 3, AT, AT, *[AT] * 3, AT, AT, 1024, 4, 0, 0, AT, AT, 1024, 4, 0, 0, AT, AT, AT, AT,
                                                                   S, T, E, k, S * T, D, H, N, E, E, exact, 0, TYPE[out]), tiles))
    return [(t >> 16, t & 65535) for t in tiles]


def routing(seed, S, T, E, k):
    """Rows spread unevenly: expert 1 gets none, expert 2 the first row alone, later ones fewer and fewer; weights 1/2, -1/4, 1, ..., and some 0."""
    g = torch.Generator(DEV).manual_seed(seed)
    l = torch.randn(S, T, E, generator=g, device=DEV) - torch.arange(E, device=DEV) * (2.0 / E)
    if E > k + 2:
        l[..., 1] = -100.0
        l[..., 2] = -100.0
        l[:, 0, 2] = 100.0
    r = q.route_experts(l, k)
    w = torch.tensor([0.5, -0.25, 1.0, 0.0], device=DEV)[torch.randint(0, 4, (S, T, k), generator=g, device=DEV)]
    return q.Routing(w, r.experts, r.offsets, r.rows, E)


def expected(x, r, up, down, bu, bd, E):
    """x [S T, D], up / down [sets, ..]: the plain form, its hidden rows cast by the quantiser (its own tests hold it to the bit)."""
    S, T, k = r.experts.shape
    y = torch.zeros(S * T, down.shape[-2], dtype=torch.float64, device=DEV)
    for s in range(S):
        for e in range(E):
            i = s * E + e
            rows = r.rows[r.offsets[i]:r.offsets[i + 1]].long()
            if rows.numel():
                h = (x[rows // k] @ up[i % len(up)].T + bu[i % len(up)]).clamp(min=0)
                h = q.quantize_fp8(h.float()).dequantize(torch.float64)
                o = h @ down[i % len(down)].T + bd[i % len(down)]
                y.index_add_(0, rows // k, o * r.weights.reshape(-1)[rows].double()[:, None])
    return y.reshape(S, T, -1)


def select(seed, n, R, K, high):
    """[n, R, K] with one entry a row, row r's in column r modulo K (so that a block of rows takes from one block of columns): +-high at most, nothing is summed."""
    g = torch.Generator(DEV).manual_seed(seed)
    w = torch.zeros(n, R, K, dtype=torch.float64, device=DEV)
    r = torch.arange(R, device=DEV)
    w[:, r, r % K] = torch.randint(1, high + 1, (n, R), generator=g, device=DEV).double()
    return w


# (S, T, E, k): sizes of which both products take the tile, by the result's type (for float16 the second is not exact and takes the largest)
GROUPED = [(torch.bfloat16, (256, 256), (1, 8192, 8, 2), 700, 700), (torch.bfloat16, (256, 256), (2, 5000, 7, 3), 600, 520), (torch.bfloat16, (128, 256), (1, 1600, 64, 4), 1200, 1200),
           (torch.bfloat16, (128, 128), (5, 300, 12, 3), 600, 600), (torch.bfloat16, (64, 128), (1, 300, 5, 2), 300, 300), (torch.bfloat16, (32, None), (1, 100, 12, 3), 300, 300),
           (torch.bfloat16, (16, None), (2, 9, 12, 3), 300, 300), (torch.float16, (128, 256), (1, 8192, 8, 2), 700, 700), (torch.float32, (128, 256), (1, 8192, 8, 2), 700, 700),
           (torch.float32, (128, 256), (1, 1600, 64, 4), 1200, 1200), (torch.float32, (128, 128), (5, 300, 12, 3), 600, 600), (torch.float16, (64, 128), (1, 300, 5, 2), 300, 300),
           (torch.float32, (32, None), (1, 100, 12, 3), 300, 300), (torch.float16, (16, None), (2, 9, 12, 3), 300, 300)]


@pytest.mark.parametrize("first", [True, False], ids=["first product", "second product"])
@pytest.mark.parametrize("D", [100, 256, 600])
@pytest.mark.parametrize("out,tile,size,H,N", GROUPED, ids=lambda v: str(v).replace("torch.", ""))
def test_groups(out, tile, size, H, N, D, first):
    """One product sums, the other selects: so the cast between them rounds, and nothing else does before the result."""
    S, T, E, k = size
    for i, t in enumerate(experts_tiles(S, T, E, k, D, H, N, out)):
        assert t == ((tile[0], (128, 64)[i]) if tile[1] is None else (256, 256) if out == torch.float16 and T == 8192 and i else tile)
    r = routing(5, S, T, E, k)
    sets = S * E if S > 1 else E
    if first:
        x, up, down, most = ints(1, 1, S * T, D), ints(2, 128, sets, H, D), select(3, sets, N, H, 1), 40
    else:      # sums below 2048: exact where they wait in 11 bits
        x, up, down, most = ints(1, 1, S * T, D, high=1, scales=1), select(2, sets, H, D, 1), ints(3, 128, sets, N, H, high=1, scales=1), 1
    g = torch.Generator(DEV).manual_seed(4)
    bu, bd = (torch.randint(0, top + 1, (sets, n), generator=g, device=DEV).double() for n, top in ((H, most), (N, 0 if first else 1)))
    want = expected(x, r, up, down, bu, bd, E)
    lead = (S, E) if S > 1 else (E,)
    y = q.experts_fp8(x.float().reshape(S, T, D), r, *(q.quantize_fp8(w.float(), 128).reshape(*lead) for w in (up, down)), bu.float().reshape(*lead, H), bd.float().reshape(*lead, N), out_dtype=out)
    assert torch.equal(y, want.to(out))


@pytest.mark.parametrize("T,tile", [(8192, (256, 256)), (200, (64, 128)), (60, (32, 64)), (20, (16, 64))])
@pytest.mark.parametrize("H", [128, 1000, 2048])
def test_the_fast_form_holds_its_stated_norm(H, T, tile):
    """The e4m3 instruction's cut, stated as 1.3e-5 of the result's norm on normal data, seen in a float32 result of the fast form (the C entry alone gives one): the
    first product selects, so that the hidden rows are the inputs'; 5e-5 allowed."""
    E, N = (8, 7500) if T == 8192 else (2, 300)
    g = torch.Generator(DEV).manual_seed(H)
    x = q.quantize_fp8(torch.randn(T, H, generator=g, device=DEV).abs())
    down = q.quantize_fp8(torch.randn(E, N, H, generator=g, device=DEV), 128)
    up = q.quantize_fp8(select(1, E, H, H, 1).float(), 128)
    r = q.route_experts(torch.randn(T, E, generator=g, device=DEV), 1)
    hp = x.data.shape[-1]
    room = torch.empty(T * (hp + hp // 32 + 16 + 4 * N) + 4096, dtype=torch.uint8, device=DEV)
    h = (room.data_ptr() + 255) & ~255
    he = (h + T * hp + 255) & ~255
    o = (he + T * x.exponent.shape[-1] + 255) & ~255
    assert o + T * N * 4 <= room.data_ptr() + room.numel()
    y, ones = torch.empty(T, N, device=DEV), torch.ones(T, device=DEV)
    kb, sp = -(-H // 128), x.exponent.shape[-1]
    call = _lib.F8_EXPERTS.pack(*[0] * 3, x.data.data_ptr(), x.exponent.data_ptr(), r.offsets.data_ptr(), r.rows.data_ptr(), ones.data_ptr(),
                                up.data.data_ptr(), up.exponent.data_ptr(), H * hp, kb * sp, 0, 0, down.data.data_ptr(), down.exponent.data_ptr(), N * hp, -(-N // 128) * sp, 0, 0,
                                h, he, o, y.data_ptr(), 1, T, E, 1, T, H, H, N, E, E, 0, 0, 0)
    tiles = (C.c_int32 * 2)()
    _lib.check(_lib.lib().qbnn_experts_f8_tiles(call, tiles))
    assert (tiles[1] >> 16, tiles[1] & 65535) == tile
    _lib.check(_lib.lib().qbnn_experts_f8(call, _lib.current_stream()))
    xv, dv = x.dequantize(torch.float64), down.dequantize(torch.float64)
    want = torch.zeros(T, N, dtype=torch.float64, device=DEV)
    for e in range(E):
        t = (r.experts[:, 0] == e).nonzero()[:, 0]
        want[t] = xv[t] @ dv[e].T
    assert float((y.double() - want).norm() / want.norm()) <= 5e-5
