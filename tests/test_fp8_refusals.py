"""What the 8-bit float operators and the router refuse, and the format's plain form against torch's own cast: no GPU."""
import numpy as np
import pytest
import torch

import f8_oracle as orc
import quantised_bayesian_nets_amd as q
from quantised_bayesian_nets_amd import _lib


def held(lead, R, K, rows=128):
    kp = -(-K // 128) * 128
    return q.F8Tensor(torch.zeros(*lead, R, kp, dtype=torch.float8_e4m3fn), torch.full((*lead, -(-R // rows), -(-kp // 512) * 4), 127, dtype=torch.uint8), K, rows)


def test_oracle_rounds_as_e4m3():
    v = torch.cat([torch.linspace(-448, 448, 20011), torch.randn(20000) * 0.01, torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 440.0])]).float()
    assert np.array_equal(orc.e4m3(v.double().numpy()), v.to(torch.float8_e4m3fn).double().numpy())


def test_tensor_checks():
    t = held((2,), 5, 130)
    assert t.shape == (2, 5, 130) and t.data.shape == (2, 5, 256) and t.exponent.shape == (2, 1, 4)
    assert t.dequantize().shape == (2, 5, 130) and t.reshape(1, 2).shape == (1, 2, 5, 130)
    for data, exponent, columns, rows, error in (
            (t.data, t.exponent, 130, 64, ValueError), (t.data, t.exponent, 100, 128, ValueError), (t.data, t.exponent, 0, 128, ValueError), (t.data, t.exponent, 130, 1, ValueError),
            (t.data.float(), t.exponent, 130, 128, TypeError), (t.data, t.exponent.int(), 130, 128, TypeError), (t.data, t.exponent[..., :2], 130, 128, ValueError),
            (t.data.transpose(0, 1).contiguous().transpose(0, 1), t.exponent, 130, 128, ValueError), (t.data[0, 0], t.exponent[0, 0], 130, 128, ValueError)):
        with pytest.raises(error):
            q.F8Tensor(data, exponent, columns, rows)


def test_quantiser_refuses():
    for x, rows, error in ((torch.zeros(3, 4, dtype=torch.float64), 1, TypeError), (torch.zeros(4), 1, ValueError), (torch.zeros(3, 0), 1, ValueError), (torch.zeros(3, 4), 64, ValueError),
                           ([1.0], 1, TypeError), (torch.zeros(3, 4), 1, RuntimeError)):      # (the last: not on the GPU)
        with pytest.raises(error):
            q.quantize_fp8(x, rows)


def test_linear_refuses():
    x, w = torch.zeros(3, 200), held((), 5, 200)
    for a, b, kw, error in ((x, x, {}, TypeError), (x, held((), 5, 200, 1), {}, TypeError), (w, w, {}, TypeError), (x, held((), 5, 201), {}, ValueError), (x[0], w, {}, ValueError),
                            (torch.zeros(2, 3, 200), held((3,), 5, 200), {}, ValueError), (x, held((), 0, 200), {}, ValueError), (x, held((1, 1), 5, 200), {}, ValueError),
                            (x, w, dict(out_dtype=torch.float64), TypeError), (x, w, dict(bias=torch.zeros(6)), ValueError), (x, w, dict(bias=torch.zeros(5).double()), ValueError),
                            (x.double(), w, {}, TypeError), (x, w, {}, RuntimeError)):
        with pytest.raises(error):
            q.linear_fp8(a, b, **kw)


def test_router_refuses():
    l = torch.zeros(4, 12)
    for a, k, kw, error in ((l.long(), 2, {}, TypeError), (l[0], 2, {}, ValueError), (torch.zeros(4, 0), 1, {}, ValueError), (torch.zeros(4, 1025), 1, {}, ValueError), (l, 0, {}, ValueError),
                            (l, 13, {}, ValueError), (torch.zeros(4, 64), 33, {}, ValueError), (l, 2, dict(score="relu"), ValueError), (l, 2, dict(groups=5), ValueError),
                            (l, 2, dict(groups=0), ValueError), (l, 2, dict(groups=4, top_groups=5), ValueError), (l, 4, dict(groups=4, top_groups=1), ValueError),
                            (l, 2, dict(bias=torch.zeros(11)), ValueError), (l, 2, dict(bias=torch.zeros(12).double()), ValueError), (l, 2, {}, RuntimeError)):
        with pytest.raises(error):
            q.route_experts(a, k, **kw)


def test_experts_refuse():
    S, T, E, k, D, H, N = 2, 5, 4, 2, 130, 140, 60
    z = torch.zeros(S, T, k)
    good = (z, z.int(), torch.zeros(S * E + 1).int(), torch.zeros(S * T * k).int(), E)
    for i, bad, error in ((0, z.double(), TypeError), (1, z.long(), TypeError), (2, good[2].long(), TypeError), (3, good[3].long(), TypeError), (1, z[:1].int(), ValueError), (2, good[2][1:], ValueError),
                          (3, good[3][1:], ValueError), (4, 5, ValueError), (0, torch.zeros(T, S, k).transpose(0, 1), ValueError)):
        with pytest.raises(error):
            q.Routing(*good[:i], bad, *good[i + 1:])
    r = q.Routing(z, z.int(), torch.zeros(S * E + 1).int(), torch.zeros(S * T * k).int(), E)
    x, up, down = torch.zeros(S, T, D), held((E,), H, D), held((E,), N, H)
    for args, kw, error in (((x, None, up, down), {}, TypeError), ((x, r, x, down), {}, TypeError), ((x, r, held((E,), H, D, 1), down), {}, TypeError), ((x, r, held((), H, D), down), {}, TypeError),
                            ((x[:, :4], r, up, down), {}, ValueError), ((x[..., :100], r, up, down), {}, ValueError), ((torch.zeros(3, T, D), r, up, down), {}, ValueError),
                            ((x, r, up, held((E,), N, 150)), {}, ValueError), ((x, r, held((3,), H, D), down), {}, ValueError), ((x, r, held((3, E), H, D), down), {}, ValueError),
                            ((x, r, up, down, torch.zeros(E, N)), {}, ValueError), ((x, r, up, down, None, torch.zeros(S, E, N)), {}, ValueError),
                            ((x, r, up, down), dict(out_dtype=torch.float8_e4m3fn), TypeError), ((x.double(), r, up, down), {}, TypeError), ((x, r, up, down), {}, RuntimeError)):
        with pytest.raises(error):
            q.experts_fp8(*args, **kw)


def test_c_entries_refuse():
    """Argument errors come back as codes with a text, before any launch."""
    L = _lib.lib()
    assert L.qbnn_quantize_f8(None, 0, 0, 0, 1, 1, 1, 1, None, None, None) == -1
    assert L.qbnn_quantize_f8(None, 5, 0, 0, 0, 1, 1, 1, None, None, None) == -1
    assert L.qbnn_quantize_f8(None, 0, 0, 0, 0, 1, 1, 1, None, None, None) == 0
    linear, experts, route = _lib.F8_LINEAR, _lib.F8_EXPERTS, _lib.ROUTE
    assert L.qbnn_linear_f8_mc(bytes(linear.size), None) == -1 and b"qbnn_linear_f8" in L.qbnn_last_error()
    p = [0, 0, 0, 1032, 1024, 0, 0, 1024, 1024, 0, 0, 0, 0, 1024, 0]
    assert L.qbnn_linear_f8_mc(linear.pack(*p, 1, 1, 1, 1, 0, 0, 0), None) == -1 and b"multiples of 16" in L.qbnn_last_error()
    assert L.qbnn_linear_f8_mc(linear.pack(*p, 1, 1, 1, 1, 0, 4, 0), None) == -1 and b"bad argument" in L.qbnn_last_error()
    assert L.qbnn_linear_f8_mc(linear.pack(*p, 0, 1, 1, 1, 0, 0, 0), None) == 0
    assert L.qbnn_experts_f8(bytes(experts.size), None) == -1
    assert L.qbnn_experts_f8(experts.pack(*[0] * 24, 1, 0, 2, 1, 1, 1, 1, 1, 2, 2, 0, 0, 0), None) == 0          # no rows
    assert L.qbnn_experts_f8(experts.pack(*[0] * 24, 1, 1, 2, 1, 1, 1, 1, 1, 2, 2, 0, 0, 0), None) == -1         # no tensors
    assert L.qbnn_route_experts(bytes(route.size), None) == -1
    assert L.qbnn_route_experts(route.pack(*[1024] * 9, 1, 1, 4, 5, 1, 1, 0, 0, 0, 1.0), None) == -1             # more choices than experts
    assert L.qbnn_route_workspace_ints(0, 5, 5) == 0


def test_descriptors_match_the_header(tmp_path):
    """The packed descriptors are the C structs: sizes (up to the last field) and the offsets of the fields at their ends, by a C compiler."""
    import os
    import shutil
    import subprocess
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text('#include "qbnn.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", offsetof(qbnn_f8_linear, x_type) + 4, offsetof(qbnn_f8_linear, M), '
                   'offsetof(qbnn_f8_experts, y_type) + 4, offsetof(qbnn_f8_experts, S), offsetof(qbnn_route, scale) + 4, offsetof(qbnn_route, S)); return 0; }\n')
    subprocess.check_call(["gcc", "-I", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include"), str(src), "-o", str(exe)])
    linear, experts, route = _lib.F8_LINEAR.size, _lib.F8_EXPERTS.size, _lib.ROUTE.size
    assert [int(v) for v in subprocess.check_output([str(exe)]).split()] == [linear, linear - 28, experts, experts - 52, route, route - 40]
