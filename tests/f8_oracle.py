"""Plain 64-bit forms of the 8-bit float operators, on the CPU and without the package's code: the block quantiser, the product, the router and the
routed experts, and the bounds that their tests hold the kernels to."""
import numpy as np

FP32 = 2.0 ** -24                                            # half a step of fp32, relative
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}      # half a step of the type's subnormals


def block_exponents(v, rows):
    """v [R, K] float64 -> [Rb, Kb] int: the smallest e >= -126 with max finite |v| <= 448 2^e (0 for zeros)."""
    R, K = v.shape
    a = np.where(np.isfinite(v), np.abs(v), 0.0)
    a = np.pad(a, ((0, -R % rows), (0, -K % 128))).reshape(-(-R // rows), rows, -(-K // 128), 128).max(axis=(1, 3))
    m, e = np.frexp(a / 448.0)                               # a = m 2^e, m in [0.5, 1)
    e = np.where(m == 0.5, e - 1, e)
    return np.where(a == 0, 0, np.maximum(e, -126)).astype(np.int64)


def e4m3(v):
    """Nearest e4m3 value, ties to even; NaN for what is not finite.  |v| <= 448."""
    with np.errstate(invalid="ignore"):
        step = np.ldexp(1.0, np.maximum(np.frexp(v)[1], -5) - 4)
        return np.where(np.isfinite(v), np.rint(v / step) * step, np.nan)


def expand(e, rows, R, K):
    return np.repeat(np.repeat(np.ldexp(1.0, e), rows, 0)[:R], 128, 1)[:, :K]


def quantised(v, rows):
    """The values that the block format holds for v [R, K]."""
    s = expand(block_exponents(v, rows), rows, *v.shape)
    return e4m3(v / s) * s


def product(x, w, bias=None, relu=False):
    y = x @ w.T
    if bias is not None:
        y = y + bias
    return np.where(y > 0, y, np.where(np.isnan(y), y, 0.0)) if relu else y


def product_bound(x, w, bias=None, exact=True):
    """Every one of the K additions of an fp32 sum is off by at most half a step (a whole one if the matrix unit cuts off instead of rounding) of a
    partial sum, and no partial sum exceeds the sum of the magnitudes; one more addition for the bias.  exact=False: the e4m3 matrix instruction, which
    cuts each of 8 neighbouring products off 2^-13 below the largest of them before it adds them."""
    x, w = np.abs(x), np.abs(w)
    off = 2 * FP32 * (x.shape[1] + 1) * (x @ w.T + (0 if bias is None else np.abs(bias)))
    if not exact:
        x, w = (np.pad(np.nan_to_num(m), ((0, 0), (0, -m.shape[1] % 8))).astype(np.float32) for m in (x, w))
        cut = np.zeros((x.shape[0], w.shape[0]), np.float32)
        for k in range(0, x.shape[1], 8):
            cut += np.max([np.outer(x[:, k + i], w[:, k + i]) for i in range(8)], axis=0)
        off = off + 8 * 2.0 ** -13 * cut
    return off


def rounding(y, dtype):
    return HALF_STEP[dtype] * np.abs(y) + TINY[dtype]


def route(logits, lowest, k, score="softmax", bias=None, groups=1, top_groups=1, renormalize=False, scale=1.0):
    """logits [T, E] float64 -> (weights [T, k], experts [T, k])."""
    T, E = logits.shape
    W, X = np.zeros((T, k)), np.zeros((T, k), np.int64)
    for t in range(T):
        l = logits[t]
        open_ = l > lowest                                   # (False for NaN)
        p = np.zeros(E)
        if open_.any():
            if score == "softmax":
                z = np.exp(l[open_] - l[open_].max())
                p[open_] = z / z.sum()
            else:
                p[open_] = 1 / (1 + np.exp(-l[open_]))
        key = l.copy() if bias is None and groups == 1 else p + (0 if bias is None else bias)
        key = np.where(open_, key, -np.inf)
        allowed = np.ones(E, bool)
        if groups > 1:
            parts = np.sort(key.reshape(groups, -1), axis=1)[:, ::-1][:, :2]
            best = np.array([q[np.isfinite(q)].sum() if np.isfinite(q).any() else -np.inf for q in parts])
            order = sorted(range(groups), key=lambda g: (-best[g], g))
            allowed = np.repeat(np.isin(np.arange(groups), order[:top_groups]), E // groups)
        order = sorted(np.nonzero(allowed)[0], key=lambda e: (-key[e], e))[:k]
        X[t] = order
        w = p[order]
        if renormalize:
            w = w / w.sum() if w.sum() else np.zeros(k)
        W[t] = np.nan if np.isnan(l).any() else w * scale
    return W, X


def order_of(experts, E):
    """experts [S, T, k] -> (offsets [S E + 1], rows [S T k]): the choices sorted by (sample, expert), stable."""
    S = experts.shape[0]
    group = (experts + E * np.arange(S)[:, None, None]).reshape(-1)
    return np.searchsorted(np.sort(group, kind="stable"), np.arange(S * E + 1)), np.argsort(group, kind="stable")


def experts(x, weights, chosen, up, down, b_up, b_down, dtype):
    """x [S, T, D] (already on the block grid), up(s, e) / down(s, e) -> weight matrices -> (y, bound): the bound allows every hidden value that lies within the first
    product's fp32 bound of a rounding border to fall on either side of it."""
    S, T, k = chosen.shape
    N = down(0, 0).shape[0]
    y, bound, size = (np.zeros((S, T, N)) for _ in range(3))
    for s in range(S):
        for e in np.unique(chosen[s]):
            t, j = np.nonzero(chosen[s] == e)
            u, d = up(s, e), down(s, e)
            bu, bd = (None if b is None else b(s, e) for b in (b_up, b_down))
            h = product(x[s, t], u, bu, relu=True)
            off = product_bound(x[s, t], u, bu, exact=dtype != "bfloat16")
            hq = quantised(h, 1)
            q = expand(block_exponents(h, 1), 1, *h.shape)
            swing = np.maximum(np.abs(e4m3(np.clip((h + off) / q, -448, 448)) * q - hq), np.abs(e4m3(np.maximum(h - off, 0) / q) * q - hq))
            o = product(hq, d, bd)
            w = weights[s, t, j][:, None]
            y[s, t] += np.where(w == 0, 0, o * w)
            size[s, t] += np.abs(o * w)
            part = np.abs(w) * (product_bound(hq, d, bd, exact=dtype == "float32") + swing @ np.abs(d).T)
            bound[s, t] += part + 3 * FP32 * np.abs(o * w)          # the weight's own error and its product
            if dtype == "bfloat16":
                # may be held as halves of v 2^-e, |v 2^-e| <= 448 and 2^e <= the block's largest / 224: half a step of v 2^-e, or of the subnormals (2^-25) below 2^-14
                blocks = np.pad(np.abs(np.nan_to_num(o * w, posinf=0, neginf=0)), ((0, 0), (0, -N % 128))).reshape(len(w), -1, 128).max(2)
                bound[s, t] += HALF_STEP["float16"] * np.abs(o * w) + np.repeat(blocks, 128, 1)[:, :N] * 2.0 ** -25 / 224
    return y, bound * (1 + HALF_STEP[dtype]) + k * 2 * FP32 * size + rounding(y, dtype)
