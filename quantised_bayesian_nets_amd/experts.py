"""Routed layers: a router that sends each row to its top-k experts, and the experts' products over the rows each was sent.

Beside the ensembles here, which evaluate every member on every row: k of E are evaluated, each row by its own choice, and their results are summed
with the router's weights.  Experts are two linear layers with a ReLU between, in 8-bit floating point (fp8.py)."""
import ctypes as C

import torch

from . import _lib
from .fp8 import BLOCK, FLOAT_TYPES, F8Tensor, _F8, _bias, _evaluates, _float, _on, _operand, padded_columns
from .layers import timed

MAX_EXPERTS, MAX_CHOICES = 1024, 32      # include/qbnn.h: QBNN_ROUTE_MAX_EXPERTS, QBNN_ROUTE_MAX_CHOICES


class Routing:
    """What the router decided for [S, T] rows: `weights` float32 and `experts` int32 [S, T, top_k] (best first), and the order in which the experts'
    products walk the choices: those of (sample s, expert e) are rows[offsets[s E + e] : offsets[s E + e + 1]], flat indices into [S, T, top_k]."""

    __slots__ = ("weights", "experts", "offsets", "rows", "n_experts")

    def __init__(self, weights, experts, offsets, rows, n_experts):
        self.weights, self.experts, self.offsets, self.rows, self.n_experts = weights, experts, offsets, rows, n_experts


def route_experts(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=False, scale=1.0):
    """logits float [T, E] or [S, T, E] -> Routing.

    score "softmax" or "sigmoid" of the logits; what is compared is score + bias[e] (float32 [E], e.g. for balance; compared as 64-bit values, ties to the
    lowest index), what the results are weighted with is the score, divided by the chosen ones' sum with `renormalize`, times `scale`.  groups > 1: of
    `groups` equal runs of experts only the `top_groups` with the largest sum of their two largest keys take part.  A logit of -inf or of its type's lowest
    value is masked: behind all others, weight 0.  A NaN makes its row's weights NaN, the row's experts stay valid."""
    _float(logits, "logits")
    if logits.dim() not in (2, 3):
        raise ValueError("logits is [T, E] or [S, T, E]")
    T, E = logits.shape[-2:]
    S = logits.shape[0] if logits.dim() == 3 else 1
    top_groups = groups if top_groups is None else top_groups
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError("1 to %d experts" % MAX_EXPERTS)
    if score not in ("softmax", "sigmoid"):
        raise ValueError("score is 'softmax' or 'sigmoid'")
    if not 1 <= groups <= 64 or E % groups or not 1 <= top_groups <= groups:
        raise ValueError("groups divides the experts (at most 64 groups), 1 <= top_groups <= groups")
    if not 1 <= top_k <= min(MAX_CHOICES, E // groups * top_groups):
        raise ValueError("top_k is at most %d and the experts of top_groups groups" % MAX_CHOICES)
    if S * T * top_k >= 1 << 31 or S > 65535:
        raise ValueError("too many rows for one call")
    bias = _bias(bias, ((E,),), "[E]")
    dev = _evaluates(logits, bias)
    if logits.stride(-1) != 1 and E > 1:
        logits = logits.contiguous()
    lead = (S, T) if logits.dim() == 3 else (T,)
    weights = torch.empty((*lead, top_k), dtype=torch.float32, device=dev)
    experts = torch.empty((*lead, top_k), dtype=torch.int32, device=dev)
    rows = torch.empty(S * T * top_k, dtype=torch.int32, device=dev)
    if rows.numel() == 0:
        return Routing(weights, experts, torch.zeros(S * E + 1, dtype=torch.int32, device=dev), rows, E)
    offsets = torch.empty(S * E + 1, dtype=torch.int32, device=dev)
    L = _lib.lib()
    ws = torch.empty(int(L.qbnn_route_workspace_ints(S, T, E)), dtype=torch.int32, device=dev)
    d = _lib.Route()
    d.logits, d.logits_ss, d.logits_rs, d.type = logits.data_ptr(), (logits.stride(0) if logits.dim() == 3 else 0), logits.stride(-2), FLOAT_TYPES[logits.dtype]
    d.bias = None if bias is None else bias.data_ptr()
    d.weights, d.experts, d.offsets, d.rows, d.workspace = weights.data_ptr(), experts.data_ptr(), offsets.data_ptr(), rows.data_ptr(), ws.data_ptr()
    d.S, d.T, d.E, d.top_k, d.groups, d.top_groups, d.sigmoid, d.renormalize, d.scale = S, T, E, top_k, groups, top_groups, int(score == "sigmoid"), int(bool(renormalize)), scale
    with _on(dev), timed("route_experts"):
        _lib.check(L.qbnn_route_experts(C.byref(d), _lib.current_stream()))
    return Routing(weights, experts, offsets, rows, E)


def experts_fp8(x, routing, w_up, w_down, b_up=None, b_down=None, out_dtype=None):
    """y[t] = sum_j weight[t, j] (relu(x[t] w_up[e]^T + b_up[e]) w_down[e]^T + b_down[e]) with e = expert[t, j].

    x: float, or an F8Tensor with block_rows 1, [T, D] or [S or 1, T, D] as the routing's rows; w_up F8Tensor [E, H, D], w_down [E, N, H] (block_rows 128; [S, E, ..]
    gives each sample its own); b_up / b_down float32 [E, H] / [E, N] or [S, E, ..].  The hidden rows are quantised as they leave the first product; the weighted
    results stay fp32 and their sum is rounded once, to `out_dtype` (x's type; bfloat16 for an F8Tensor).  For a bfloat16 result both products take the fast form of
    linear_fp8, for float16 the first and for float32 both take the exact one: a hidden value next to a rounding border moves by a whole step."""
    if not isinstance(routing, Routing):
        raise TypeError("routing is a Routing (route_experts)")
    for w in (w_up, w_down):
        if not isinstance(w, F8Tensor) or w.block_rows != BLOCK or len(w.shape) not in (3, 4):
            raise TypeError("w_up and w_down are F8Tensors with block_rows 128, [E, rows, columns] or [S, E, rows, columns]")
    if isinstance(x, F8Tensor):
        if x.block_rows != 1:
            raise TypeError("x is a float tensor or an F8Tensor with block_rows 1")
        out_dtype = out_dtype or torch.bfloat16
    else:
        out_dtype = out_dtype or _float(x, "x").dtype
    if out_dtype not in FLOAT_TYPES:
        raise TypeError("out_dtype is float32, bfloat16 or float16")
    lead, k, E = routing.experts.shape[:-1], routing.experts.shape[-1], routing.n_experts
    S, T = (lead if len(lead) == 2 else (1, lead[0]))
    xs = x.shape
    H, D = w_up.shape[-2:]
    N = w_down.shape[-2]
    if len(xs) not in (2, 3) or xs[-2] != T or xs[-1] != D or (len(xs) == 3 and xs[0] not in (1, S)):
        raise ValueError("x is [%d or 1, %d, %d] for this routing and w_up" % (S, T, D))
    if w_down.shape[-1] != H or H < 1 or N < 1:
        raise ValueError("w_up [.., H, D] and w_down [.., N, H] do not fit: %s and %s" % (w_up.shape, w_down.shape))
    own = []
    for w in (w_up, w_down):
        if tuple(w.shape[:-2]) not in ((E,), (1, E), (S, E)):
            raise ValueError("the routing has %d experts and %d samples" % (E, S))
        own.append(len(w.shape) == 4 and w.shape[0] == S)
    b_up = _bias(b_up, ((*w_up.shape[:-2], H),), "like w_up without its columns")
    b_down = _bias(b_down, ((*w_down.shape[:-2], N),), "like w_down without its columns")
    dev = _evaluates(x.data if isinstance(x, F8Tensor) else x, routing.weights, w_up.data, w_down.data, b_up, b_down)
    y = torch.empty((*lead, N), dtype=out_dtype, device=dev)
    R = S * T * k
    if R == 0:
        return y
    with _on(dev):
        x = _operand(x)
        L, st = _lib.lib(), _lib.current_stream()
        hp, sp = padded_columns(H)
        h = torch.empty((R, hp), dtype=torch.float8_e4m3fn, device=dev)
        he = torch.empty((R, sp), dtype=torch.uint8, device=dev)
        o = torch.empty((R, N), dtype=torch.float32, device=dev)
        for first, w, b, per_sample in ((True, w_up, b_up, own[0]), (False, w_down, b_down, own[1])):
            d, r = _lib.F8Linear(), _lib.F8Routed()
            d.w, d.w_exp, d.w_ss, d.w_exp_ss = w.data.data_ptr(), w.exponent.data_ptr(), w.data.stride(-3), w.exponent.stride(-3)
            if b is not None:
                d.bias, d.bias_ss = b.data_ptr(), b.stride(-2)
            r.offsets, r.groups, r.w_groups = routing.offsets.data_ptr(), S * E, (S * E if per_sample else E)
            d.M, d.n_samples = R, 1
            if first:
                d.x, d.x_exp, d.y, d.y_exp = x.data.data_ptr(), x.exponent.data_ptr(), h.data_ptr(), he.data_ptr()
                d.N, d.K, d.relu, d.y_type, d.exact = H, D, 1, _F8, int(out_dtype != torch.bfloat16)
                r.x_rows, r.topk, r.x_row_count = routing.rows.data_ptr(), k, x.data.shape[:-1].numel()
            else:
                d.x, d.x_exp, d.y = h.data_ptr(), he.data_ptr(), o.data_ptr()
                d.N, d.K, d.relu, d.y_type, d.exact = N, H, 0, 0, int(out_dtype == torch.float32)
                r.y_rows, r.y_weights = routing.rows.data_ptr(), routing.weights.data_ptr()
            with timed("linear_f8_routed"):
                _lib.check(L.qbnn_linear_f8_routed(C.byref(d), C.byref(r), st))
        with timed("combine_routed"):
            _lib.check(L.qbnn_combine_routed(_lib.ptr(o), S * T, k, N, _lib.ptr(y), FLOAT_TYPES[out_dtype], st))
    return y
