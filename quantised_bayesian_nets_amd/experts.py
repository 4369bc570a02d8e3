"""Routed layers: a router that sends each row to its top-k experts, and the experts' products over the rows each was sent.

Beside the ensembles here, which evaluate every member on every row: k of E are evaluated, each row by its own choice, and their results are summed
with the router's weights.  Experts are two linear layers with a ReLU between, in 8-bit floating point (fp8.py)."""
import torch

from . import _lib
from .fp8 import BLOCK, FLOAT_TYPES, F8Tensor, _bias, _device, _float, _launch, _room, _rows, padded_columns

MAX_EXPERTS, MAX_CHOICES = 1024, 32      # include/qbnn.h: QBNN_ROUTE_MAX_EXPERTS, QBNN_ROUTE_MAX_CHOICES


class Routing:
    """What the router decided for [S, T] rows: `weights` float32 and `experts` int32 [S, T, top_k] (best first), and the order in which the experts'
    products walk the choices: those of (sample s, expert e) are rows[offsets[s E + e] : offsets[s E + e + 1]], flat indices into [S, T, top_k].  Types and
    shapes are checked; that offsets and rows are such an order is not."""

    __slots__ = ("weights", "experts", "offsets", "rows", "n_experts")

    def __init__(self, weights, experts, offsets, rows, n_experts):
        shape, n = weights.shape, weights.numel()
        if weights.dtype != torch.float32 or experts.dtype != torch.int32 or offsets.dtype != torch.int32 or rows.dtype != torch.int32:
            raise TypeError("a Routing holds float32 weights and int32 experts, offsets and rows")
        if (len(shape) not in (2, 3) or experts.shape != shape or rows.shape != (n,) or offsets.shape != ((shape[0] if len(shape) == 3 else 1) * n_experts + 1,) or
                not (weights.is_contiguous() and experts.is_contiguous() and offsets.is_contiguous() and rows.is_contiguous())):
            raise ValueError("weights and experts are [T, top_k] or [S, T, top_k], offsets [S E + 1], rows [S T top_k], all contiguous")
        self.weights, self.experts, self.offsets, self.rows, self.n_experts = weights, experts, offsets, rows, n_experts


def route_experts(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=False, scale=1.0):
    """logits float [T, E] or [S, T, E] -> Routing.

    score "softmax" or "sigmoid" of the logits; what is compared is score + bias[e] (float32 [E], e.g. for balance) as a 64-bit value, and of equal ones the larger
    logit goes first and then the lowest index: a bias that is the same for all changes no choice.  What the results are weighted with is the score, divided by the
    chosen ones' sum with `renormalize`, times `scale`.  groups > 1: of `groups` equal runs of experts only the `top_groups` with the largest sum of their two
    largest keys take part, and equal keys go by the index alone.  A logit of -inf or of its type's lowest value is masked: behind all others, weight 0.  A NaN, or for
    softmax a logit of +inf, makes its row's weights NaN, the row's experts stay valid."""
    _float(logits, "logits")
    shape = logits.shape
    if len(shape) not in (2, 3):
        raise ValueError("logits is [T, E] or [S, T, E]")
    S, T, E = shape if len(shape) == 3 else (1, *shape)
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError("1 to %d experts" % MAX_EXPERTS)
    if score not in ("softmax", "sigmoid"):
        raise ValueError("score is 'softmax' or 'sigmoid'")
    if not 1 <= groups <= 64 or E % groups or not 1 <= top_groups <= groups:
        raise ValueError("groups divides the experts (at most 64 groups), 1 <= top_groups <= groups")
    if not 1 <= top_k <= min(MAX_CHOICES, E // groups * top_groups):
        raise ValueError("top_k is at most %d and the experts of top_groups groups" % MAX_CHOICES)
    if S * T * top_k >= 1 << 31 or T >= 1 << 29 or S > 65535:
        raise ValueError("too many rows for one call")
    bias = _bias(bias, ((E,),), "[E]")
    dev = _device(logits, bias)
    if logits.stride(-1) != 1 and E > 1:
        logits = logits.contiguous()
    lead = (S, T, top_k) if len(shape) == 3 else (T, top_k)
    weights = torch.empty(lead, dtype=torch.float32, device=dev)
    experts = torch.empty(lead, dtype=torch.int32, device=dev)
    n = S * T * top_k
    if n == 0:
        return Routing(weights, experts, torch.zeros(S * E + 1, dtype=torch.int32, device=dev), torch.empty(0, dtype=torch.int32, device=dev), E)
    L = _lib.lib()
    plan = torch.empty(S * E + 1 + n + L.qbnn_route_workspace_ints(S, T, E), dtype=torch.int32, device=dev)      # offsets, rows, workspace
    offsets, rows = plan.as_strided((S * E + 1,), (1,)), plan.as_strided((n,), (1,), S * E + 1)
    at = plan.data_ptr()
    _launch("route_experts", dev, L.qbnn_route_experts, _lib.ROUTE.pack(
        logits.data_ptr(), logits.stride(0) if len(lead) == 3 else 0, logits.stride(-2), 0 if bias is None else bias.data_ptr(),
        weights.data_ptr(), experts.data_ptr(), at, at + 4 * (S * E + 1), at + 4 * (S * E + 1 + n),
        S, T, E, top_k, groups, top_groups, score == "sigmoid", bool(renormalize), FLOAT_TYPES[logits.dtype], scale))
    r = Routing.__new__(Routing)                                  # (as its checks ask for)
    r.weights, r.experts, r.offsets, r.rows, r.n_experts = weights, experts, offsets, rows, E
    return r


def experts_fp8(x, routing, w_up, w_down, b_up=None, b_down=None, out_dtype=None):
    """y[t] = sum_j weight[t, j] (relu(x[t] w_up[e]^T + b_up[e]) w_down[e]^T + b_down[e]) with e = expert[t, j].

    x: float, or an F8Tensor with block_rows 1, [T, D] or [S or 1, T, D] as the routing's rows; w_up F8Tensor [E, H, D], w_down [E, N, H] (block_rows 128; [S, E, ..]
    gives each sample its own); b_up / b_down float32 [E, H] / [E, N] or [S, E, ..].  The hidden rows are quantised as they leave the first product; the weighted
    results are summed in fp32 and rounded once, to `out_dtype` (x's type; bfloat16 for an F8Tensor; large bfloat16 calls hold the terms as fp16 with a power of two per
    128 columns).  Where the experts get more than 16 rows on average, for a bfloat16 result both products take the fast form of linear_fp8, for float16 the second; they
    are exact otherwise: a hidden value next to a rounding border moves by a whole step.  Inputs of 4 GiB and more
    in e4m3 (2^20 rows of 4096 columns) go through the form for few rows, which is slower."""
    if not isinstance(routing, Routing):
        raise TypeError("routing is a Routing (route_experts)")
    if not isinstance(w_up, F8Tensor) or not isinstance(w_down, F8Tensor) or w_up.block_rows != BLOCK or w_down.block_rows != BLOCK:
        raise TypeError("w_up and w_down are F8Tensors with block_rows 128")
    us, ws = w_up.shape, w_down.shape
    if len(us) not in (3, 4) or len(ws) not in (3, 4):
        raise TypeError("w_up and w_down are [E, rows, columns] or [S, E, rows, columns]")
    if isinstance(x, F8Tensor):
        if x.block_rows != 1:
            raise TypeError("x is a float tensor or an F8Tensor with block_rows 1")
        out_dtype = out_dtype or torch.bfloat16
    else:
        out_dtype = out_dtype or _float(x, "x").dtype
    if out_dtype not in FLOAT_TYPES:
        raise TypeError("out_dtype is float32, bfloat16 or float16")
    (*lead, k), E = routing.experts.shape, routing.n_experts
    S, T = lead if len(lead) == 2 else (1, lead[0])
    xs = x.shape
    *up_sets, H, D = us
    *down_sets, N, Hd = ws
    if len(xs) not in (2, 3) or xs[-2] != T or xs[-1] != D or (len(xs) == 3 and xs[0] not in (1, S)):
        raise ValueError("x is [%d or 1, %d, %d] for this routing and w_up" % (S, T, D))
    if Hd != H or H < 1 or N < 1:
        raise ValueError("w_up [.., H, D] and w_down [.., N, H] do not fit: %s and %s" % (tuple(us), tuple(ws)))
    sets = ([E], [1, E], [S, E])
    if up_sets not in sets or down_sets not in sets:
        raise ValueError("the routing has %d experts and %d samples" % (E, S))
    b_up = _bias(b_up, ((*up_sets, H),), "like w_up without its columns")
    b_down = _bias(b_down, ((*down_sets, N),), "like w_down without its columns")
    held = isinstance(x, F8Tensor)
    dev = _device(x.data if held else x, routing.weights, routing.offsets, routing.rows, w_up.data, w_down.data, b_up, b_down)
    y = torch.empty((*lead, N), dtype=out_dtype, device=dev)
    R = S * T * k
    if R == 0:
        return y
    (dp, ds), (hp, hs) = padded_columns(D), padded_columns(H)
    x_rows = T * (xs[0] if len(xs) == 3 else 1)
    xf = xf_ss = xf_rs = x_type = 0
    if held:
        xq, xe = x.data.data_ptr(), x.exponent.data_ptr()
        room, (h, he, o) = _room(dev, R * hp, R * hs, 4 * R * N)
    else:
        x = _rows(x)
        xf, xf_ss, xf_rs, x_type = x.data_ptr(), (x.stride(0) if len(xs) == 3 else 0), x.stride(-2), FLOAT_TYPES[x.dtype]
        room, (xq, xe, h, he, o) = _room(dev, x_rows * dp, x_rows * ds, R * hp, R * hs, 4 * R * N)
    up, ue, down, de = w_up.data, w_up.exponent, w_down.data, w_down.exponent
    _launch("experts_f8", dev, _lib.lib().qbnn_experts_f8, _lib.F8_EXPERTS.pack(
        xf, xf_ss, xf_rs, xq, xe, routing.offsets.data_ptr(), routing.rows.data_ptr(), routing.weights.data_ptr(),
        up.data_ptr(), ue.data_ptr(), H * dp, -(-H // BLOCK) * ds, 0 if b_up is None else b_up.data_ptr(), H,
        down.data_ptr(), de.data_ptr(), N * hp, -(-N // BLOCK) * hs, 0 if b_down is None else b_down.data_ptr(), N,
        h, he, o, y.data_ptr(), S, T, E, k, x_rows, D, H, N, E if len(us) == 3 else up_sets[0] * E, E if len(ws) == 3 else down_sets[0] * E,
        0 if out_dtype == torch.bfloat16 else 1 if out_dtype == torch.float16 else 3, x_type, FLOAT_TYPES[out_dtype]))
    return y
