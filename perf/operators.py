"""The 8-bit floating-point linear product, the router and the routed experts: cases, plain forms and the framework's calls.

An operand in blocks is held as e4m3 values [..., R, Kp] (Kp: the columns up to a multiple of 128, zeros behind the last) and biased exponents
(uint8, 127 = 2^0) [..., Rb, Sp] (Sp: the blocks of 128 columns up to a multiple of 4), one for each 1 x 128 block of an activation and each
128 x 128 block of a weight."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a single input through one layer: latency alone
        dict(name="linear one row 1024", op="linear", S=1, B=1, N=1024, K=1024, type="bf16", bias=True, relu=False, drawn=False),
        # a few inputs through a wide layer: one pass over the weights
        dict(name="linear 4 rows 8192", op="linear", S=1, B=4, N=8192, K=8192, type="bf16", bias=False, relu=False, drawn=False),
        # LeNet's first linear layer (800 -> 500) at its benchmark's batch and samples, with weights drawn for each sample and so cast in each pass
        dict(name="linear 100 draws of 500x800", op="linear", S=100, B=128, N=500, K=800, type="fp32", bias=True, relu=True, drawn=True),
        # a large batch through a wide layer: bound by the matrix cores
        dict(name="linear 8192^3", op="linear", S=1, B=8192, N=8192, K=8192, type="bf16", bias=True, relu=True, drawn=False),
        # the router for one input
        dict(name="route 1 of 8", op="route", S=1, T=1, E=8, k=2, type="fp32", score="softmax", biased=False, groups=1, kept=1, renorm=True),
        # a batch, every expert in one group
        dict(name="route 4096 of 64", op="route", S=1, T=4096, E=64, k=6, type="bf16", score="softmax", biased=False, groups=1, kept=1, renorm=False),
        # odd sizes, routed for each of three samples on its own
        dict(name="route 3x1001 of 60", op="route", S=3, T=1001, E=60, k=4, type="fp16", score="sigmoid", biased=True, groups=1, kept=1, renorm=True),
        # many inputs and experts, chosen in groups under a balancing bias
        dict(name="route 32768 of 256", op="route", S=1, T=32768, E=256, k=8, type="fp32", score="sigmoid", biased=True, groups=8, kept=4, renorm=True),
        # one input: two experts' weights are read
        dict(name="experts 1 row", op="experts", S=1, T=1, E=8, k=2, D=1024, H=2048, type="bf16", bias=False),
        # a small batch: nearly every expert's weights are read for a few rows each
        dict(name="experts 61 rows of 64", op="experts", S=1, T=61, E=64, k=6, D=2048, H=1024, type="bf16", bias=False),
        # members with weights of their own, odd sizes
        dict(name="experts 5x300 odd", op="experts", S=5, T=300, E=12, k=3, D=777, H=1030, type="fp16", bias=True),
        # a large batch: bound by the matrix cores
        dict(name="experts 8192 rows of 32", op="experts", S=1, T=8192, E=32, k=4, D=4096, H=2048, type="bf16", bias=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "route", "experts"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op == "linear":
        drawn = rng.random() < 0.3
        while True:
            S = _log(rng, 2, 100) if drawn else rng.choice([1, 1, _log(rng, 2, 16)])
            B, N, K = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
            if S * N * K <= 1 << 26 and S * B * max(N, K) <= 1 << 27:
                return dict(op=op, S=S, B=B, N=N, K=K, type=kind, bias=rng.random() < 0.5, relu=rng.random() < 0.5, drawn=drawn)
    if op == "route":
        E = _log(rng, 4, 512)
        groups = rng.choice([1, 1, 2, 4, 8])
        groups = groups if E % groups == 0 and E // groups >= 2 else 1
        kept = rng.randint(1, groups)
        k = _log(rng, 1, min(16, E // groups * kept))
        T = _log(rng, 1, min(32768, 8388608 // E))
        S = rng.choice([1, 1, _log(rng, 2, 8)])
        return dict(op=op, S=S, T=max(1, T // S), E=E, k=k, type=kind, score=rng.choice(["softmax", "sigmoid"]), biased=rng.random() < 0.5,
                    groups=groups, kept=kept, renorm=rng.random() < 0.5)
    kind = rng.choice(["bf16", "fp16"])  # between the two products values are held in 8 bits: sums in another order move a few of them by a step, which 32 bits would show
    while True:
        S, T, E = rng.choice([1, 1, _log(rng, 2, 6)]), _log(rng, 1, 8192), _log(rng, 4, 64)
        k, D, H = _log(rng, 1, min(8, E)), _log(rng, 64, 4096), _log(rng, 64, 4096)
        if S * T * k * D * H <= 1 << 37 and S * E * D * H <= 1 << 28 and S * T * k * max(D, H) <= 1 << 27:
            return dict(op=op, S=S, T=T, E=E, k=k, D=D, H=H, type=kind, bias=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------------- the plain forms
def _blocks(v, rows):
    """[..., R, K] in 32 bits -> (e4m3 values [..., R, Kp], biased exponents [..., Rb, Sp]), one exponent for each rows x 128 block."""
    R, K = v.shape[-2:]
    Rb, Kb = -(-R // rows), -(-K // 128)
    v = torch.nn.functional.pad(v.to(torch.float32), (0, Kb * 128 - K, 0, Rb * rows - R))
    lead = v.shape[:-2]
    v = v.reshape(*lead, Rb, rows, Kb, 128)
    bits = v.abs().amax(dim=(-3, -1)).view(torch.int32)
    e = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(min=-126)
    e = torch.where(bits == 0, 0, e)
    down = ((127 - e) << 23).view(torch.float32)
    q = (v * down[..., :, None, :, None]).to(torch.float8_e4m3fn).reshape(*lead, Rb * rows, Kb * 128)[..., :R, :]
    return q.contiguous(), torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -Kb % 4)).contiguous()


def _values(q, e, rows):
    """What (_blocks) stands for, in 32 bits, with the columns behind the last still there (zeros)."""
    Kb, R = q.shape[-1] // 128, q.shape[-2]
    up = (e[..., :Kb].to(torch.int32) << 23).view(torch.float32)
    up = up.repeat_interleave(rows, dim=-2)[..., :R, :].repeat_interleave(128, dim=-1)
    return q.to(torch.float32) * up


def _linear(st):
    c = st["case"]
    w = _blocks(st["w"], 128) if c["drawn"] else (st["wq"], st["we"])
    y = torch.matmul(_values(*_blocks(st["x"], 1), 1), _values(*w, 128).transpose(-1, -2))
    if c["bias"]:
        y = y + st["b"]
    if c["relu"]:
        y = torch.relu(y)
    return y.to(TYPES[c["type"]])


def _choose(logits, k, score, bias, groups, kept, renorm, scale):
    """(weights [S, T, k] in 64 bits, experts [S, T, k]): the keys are compared in 64 bits."""
    l = logits.to(torch.float64)
    s = torch.softmax(l, dim=-1) if score == "softmax" else torch.sigmoid(l)
    key = s if bias is None else s + bias.to(torch.float64)
    E = key.shape[-1]
    if groups > 1:
        parts = key.reshape(*key.shape[:-1], groups, E // groups)
        best = parts.sort(dim=-1, descending=True)[0][..., :2].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True)[1]
        rank = order.argsort(dim=-1)
        key = torch.where((rank < kept).unsqueeze(-1), parts, float("-inf")).reshape(key.shape)
    experts = key.sort(dim=-1, descending=True, stable=True)[1][..., :k]
    w = s.gather(-1, experts)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    return w * scale, experts


def _plan(experts, E):
    """The rows (sample, input, choice) sorted by (sample, expert), those of one expert in their order: (the groups' ends, the rows, the groups of the rows)."""
    S, T, k = experts.shape
    group = (experts + E * torch.arange(S, device=experts.device)[:, None, None]).reshape(-1)
    group, rows = group.sort(stable=True)
    offsets = torch.searchsorted(group, torch.arange(S * E + 1, device=experts.device))
    return offsets, rows, group


def _route(st):
    c = st["case"]
    w, experts = _choose(st["logits"], c["k"], c["score"], st["bias"], c["groups"], c["kept"], c["renorm"], 2.5)
    offsets, rows, _ = _plan(experts, c["E"])
    return {"weights": w.to(torch.float32), "experts": experts.to(torch.int32), "offsets": offsets.to(torch.int32), "rows": rows.to(torch.int32)}


def _experts(st):
    c = st["case"]
    S, T, k = c["S"], c["T"], c["k"]
    w, experts = _choose(st["logits"], k, "softmax", None, 1, 1, True, 1.0)
    offsets, rows, group = _plan(experts, c["E"])
    at = torch.arange(rows.numel(), device=rows.device) - offsets[group]
    most = int((offsets[1:] - offsets[:-1]).max())
    x = _values(*_blocks(st["x"], 1), 1).reshape(S * T, -1)
    xs = x.new_zeros(S * c["E"], most, x.shape[-1])
    xs[group, at] = x[rows // k]
    h = torch.bmm(xs, _values(st["uq"], st["ue"], 128).flatten(0, 1).transpose(1, 2))
    if c["bias"]:
        h = h + st["ub"].flatten(0, 1).unsqueeze(1)
    h = _values(*_blocks(torch.relu(h), 1), 1)
    o = torch.bmm(h, _values(st["dq"], st["de"], 128).flatten(0, 1).transpose(1, 2))
    if c["bias"]:
        o = o + st["db"].flatten(0, 1).unsqueeze(1)
    y = o.new_empty(rows.numel(), o.shape[-1])
    y[rows] = o[group, at]
    y = (y.reshape(S, T, k, -1) * w.to(torch.float32).unsqueeze(-1)).sum(2)
    return y.to(TYPES[c["type"]])


# ---------------------------------------------------------------------------------------------------------------- the framework's calls
def _own(st):
    import quantised_bayesian_nets_amd as q
    c = st["case"]
    if c["op"] == "linear":
        w = q.quantize_fp8(st["w"], 128) if c["drawn"] else q.F8Tensor(st["wq"], st["we"], c["K"], 128)
        return q.linear_fp8(st["x"], w, st["b"], relu=c["relu"])
    if c["op"] == "route":
        r = q.route_experts(st["logits"], c["k"], score=c["score"], bias=st["bias"], groups=c["groups"], top_groups=c["kept"], renormalize=c["renorm"], scale=2.5)
        return {"weights": r.weights, "experts": r.experts, "offsets": r.offsets, "rows": r.rows}
    r = q.route_experts(st["logits"], c["k"], renormalize=True)
    up, down = q.F8Tensor(st["uq"], st["ue"], c["D"], 128), q.F8Tensor(st["dq"], st["de"], c["H"], 128)
    return q.experts_fp8(st["x"], r, up, down, st["ub"], st["db"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, by=1.0, of=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(by).to(of)

    def weights(S, N, K):
        """Means of a trained layer's size with a few rows far larger, and each sample's deviation from them."""
        w = normal(1, N, K, by=K ** -0.5) * torch.exp2(normal(1, N, 1)) + normal(S, N, K, by=0.1 * K ** -0.5)
        return w

    st = {"case": case}
    if case["op"] == "linear":
        S, B, N, K = case["S"], case["B"], case["N"], case["K"]
        st["x"] = normal(S, B, K, of=t)
        w = weights(S, N, K)
        if case["drawn"]:
            st["w"] = w
        else:
            st["wq"], st["we"] = _blocks(w, 128)
        st["b"] = normal(N, by=0.1) if case["bias"] else None
    elif case["op"] == "route":
        st["logits"] = normal(case["S"], case["T"], case["E"], by=1.5, of=t)
        st["bias"] = normal(case["E"], by=0.05) if case["biased"] else None
    else:
        S, T, E, D, H = case["S"], case["T"], case["E"], case["D"], case["H"]
        st["x"] = normal(S, T, D, of=t)
        st["logits"] = normal(S, T, E)
        st["uq"], st["ue"] = (v.reshape(S, E, *v.shape[-2:]) for v in _blocks(weights(S * E, H, D), 128))
        st["dq"], st["de"] = (v.reshape(S, E, *v.shape[-2:]) for v in _blocks(weights(S * E, D, H), 128))
        st["ub"], st["db"] = (normal(S, E, H, by=0.1), normal(S, E, D, by=0.1)) if case["bias"] else (None, None)
    return st


def run(state):
    if own:
        return _own(state)
    return {"linear": _linear, "route": _route, "experts": _experts}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "linear":
        S, B, N, K, z = case["S"], case["B"], case["N"], case["K"], SIZE[case["type"]]
        return {"bytes": S * B * (K + N) * z + S * N * K * (4 if case["drawn"] else 1) + (4 * N if case["bias"] else 0), "flops": 2 * S * B * N * K}
    S, T, E, k = case["S"], case["T"], case["E"], case["k"]
    if case["op"] == "route":
        return {"bytes": S * T * E * SIZE[case["type"]] + S * T * k * 12 + 4 * (S * E + 1), "flops": 10 * S * T * E}
    D, H, z = case["D"], case["H"], SIZE[case["type"]]
    met = S * E * (1 - (1 - k / E) ** T)  # experts that at least one row is sent to
    return {"bytes": int(met * (2 * D * H + (4 * (D + H) if case["bias"] else 0)) + S * T * (2 * D * z + 4 * E)), "flops": 4 * S * T * k * D * H}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _two(e):
    """2^e in 64 bits: from its bits, since a power function may be off by a unit in the last place."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _near(v, rows):
    """The values that blocks of e4m3 with a power of two hold for v, in 64 bits: each block's scale is the least power that brings it within 448."""
    R, K = v.shape[-2:]
    out = torch.zeros_like(v)
    for k in range(0, K, 128):
        part = v[..., k:k + 128]
        top = torch.nn.functional.pad(part.abs().amax(-1), (0, -R % rows)).unflatten(-1, (-1, rows)).amax(-1)
        m, e = torch.frexp(top / 448.0)  # in [0.5, 1): 2^e is enough, and 2^(e - 1) where m is 0.5
        e = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
        up = _two(e).repeat_interleave(rows, dim=-1)[..., :R].unsqueeze(-1)
        a = part / up
        step = _two(torch.frexp(a)[1].clamp(min=-5) - 4)  # four bits, and the subnormals' 2^-9
        out[..., k:k + 128] = torch.round(a / step) * step * up
    return out


def _held(q, e, K):
    up = _two(e.to(torch.int32) - 127)
    n, k = torch.arange(q.shape[-2], device=q.device) // 128, torch.arange(K, device=q.device) // 128
    return q[..., :K].double() * up[..., n, :][..., k]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        x = _near(st["x"].double(), 1)
        y = torch.stack([x[s] @ (_near(st["w"][s].double(), 128) if case["drawn"] else _held(st["wq"][s], st["we"][s], case["K"])).T for s in range(case["S"])])
        y = y if st["b"] is None else y + st["b"].double()
        return y.clamp(min=0) if case["relu"] else y
    l = st["logits"].double() if case["op"] == "route" else None
    if case["op"] == "route":
        s = torch.exp(l - torch.logsumexp(l, -1, keepdim=True)) if case["score"] == "softmax" else 1 / (1 + torch.exp(-l))
        key = s if st["bias"] is None else s + st["bias"].double()
        if case["groups"] > 1:
            n = case["E"] // case["groups"]
            best = torch.stack([key[..., i * n:(i + 1) * n].topk(2)[0].sum(-1) for i in range(case["groups"])], -1)
            kept = torch.zeros_like(best).scatter_(-1, best.sort(dim=-1, descending=True, stable=True)[1][..., :case["kept"]], 1.0)
            key = key.masked_fill((kept == 0).repeat_interleave(n, -1), -math.inf)
        w = s.gather(-1, key.sort(dim=-1, descending=True, stable=True)[1][..., :case["k"]])
        w = w / w.sum(-1, keepdim=True) if case["renorm"] else w
        return {"weights": 2.5 * w, "experts": None, "offsets": None, "rows": None}
    S, E, k, D, H = (case[n] for n in "SEkDH")
    x = _near(st["x"].double(), 1)
    p = torch.exp(st["logits"].double())
    chosen = p.argsort(dim=-1, descending=True, stable=True)[..., :k]
    y = torch.zeros_like(x)
    for s in range(S):
        for e in range(E):
            t, j = (chosen[s] == e).nonzero(as_tuple=True)
            h = x[s, t] @ _held(st["uq"][s, e], st["ue"][s, e], D).T
            h = h if st["ub"] is None else h + st["ub"][s, e].double()
            o = _near(h.clamp(min=0), 1) @ _held(st["dq"][s, e], st["de"][s, e], H).T
            o = o if st["db"] is None else o + st["db"][s, e].double()
            y[s, t] += o * (p[s, t, e] / p[s, t].gather(-1, chosen[s, t]).sum(-1)).unsqueeze(-1)
    return y
