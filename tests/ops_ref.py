"""Plain implementations in 64 bits of the operators on device buffers (routing, microscaled 4-bit floats, experts)."""
import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])  # between neighbours: a half goes to the even code
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # a rounding's largest relative error


def pad128(n):
    return -(-n // 128) * 128


def mx4_parts(x):
    """(codes, exponents, bad, |x| / 2^exponent) of rows of values, in blocks of 32, rows padded to 128."""
    x = np.asarray(x, np.float64)
    v = np.zeros((x.shape[0], pad128(x.shape[1])))
    v[:, :x.shape[1]] = x
    v = v.reshape(x.shape[0], -1, 32)
    most = np.abs(v).max(-1)
    bad = ~(most < np.inf)  # an infinity, or a NaN (which max passes on)
    m, e = np.frexp(np.where(bad | (most == 0), 1.0, most))
    exp = np.where(most == 0, -127, np.maximum(e - 3, -127))
    a = np.abs(np.where(bad[..., None], 0.0, v)) / np.exp2(exp)[..., None]
    code = np.searchsorted(BORDERS, a, side="left")  # a border itself stays with the lower code
    at = np.searchsorted(BORDERS, a, side="right") > code  # exactly on a border: up if the lower code is odd
    code = code + (at & (code % 2 == 1))
    sign = np.signbit(v) & ~bad[..., None]
    return code | (sign.astype(np.int64) << 3), exp, bad, a


def mx4_quantize(x):
    """codes (rows, C / 2) and scales (rows, C / 32) as bytes."""
    code, exp, bad, _ = mx4_parts(x)
    code = code.reshape(len(code), -1)
    return (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8), np.where(bad, 255, exp + 127).astype(np.uint8)


def mx4_values(codes, scales, cols):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1, 32)
    v = VALUES[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(*codes.shape[:-1], -1)[..., :cols]


def mx4(x):
    return mx4_values(*mx4_quantize(x), np.shape(x)[1])


def route(x, K, sigmoid=False, bias=None, groups=0, kept=0, best=1, renorm=True, scale=1.0):
    """ids, weights and load of logits (T, E); E = 0 rows allowed."""
    x = np.asarray(x, np.float64)
    T, E = x.shape
    known = x > -np.inf
    x = np.where(known, x, -np.inf)
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            s = np.where(known, 1 / (1 + np.exp(-x)), 0.0)
        else:
            top = x.max(-1, keepdims=True)
            p = np.where(known, np.where(x == top, 1.0, np.exp(x - top)), 0.0)
            s = p / np.maximum(p.sum(-1, keepdims=True), 1e-300)
    if bias is not None:
        b = np.asarray(bias, np.float64)
        key = np.where(known & (b > -np.inf), s + b, -np.inf)
    else:
        key = np.where(known, s, -np.inf) if groups > 1 and best > 1 else x
    ids = np.full((T, K), -1, np.int64)
    w = np.zeros((T, K))
    for t in range(T):
        k = key[t].copy()
        if groups > 1:
            g = k.reshape(groups, -1)
            top = -np.sort(-g, axis=1)[:, :best]
            worth = np.where(top[:, 0] == -np.inf, -np.inf, np.where(top == -np.inf, 0.0, top).sum(1))
            stays = np.argsort(-worth, kind="stable")[:kept]
            k = np.where(np.isin(np.arange(E) // (E // groups), stays), k, -np.inf)
        o = np.argsort(-k, kind="stable")[:K]
        o = o[k[o] > -np.inf]
        ids[t, :len(o)] = o
        w[t, :len(o)] = s[t, o]
    if renorm:
        w = w / np.maximum(w.sum(-1, keepdims=True), 1e-20)
    return ids, w * scale, np.bincount(ids[ids >= 0], minlength=E)


def swiglu(g, u, limit):
    if limit:
        g, u = np.where(g > limit, limit, g), np.where(u > limit, limit, np.where(u < -limit, -limit, u))
    return g / (1 + np.exp(-g)) * u


def experts(x, ids, w, gate, up, down, limit=0.0):
    """y and how far it may be off: gate, up (E, F, H) and down (E, H, F) values.

    The bound: the kernel's g and u are off by at most n 2^-23 of their terms' absolute sum (n additions in fp32, the
    exact products of the format), h by those and by 2^-20 of itself (the SiLU's roundings, an exponential good to a few
    of them). Where h is that near a border between two codes the code may be either: one step of the block's scale; where
    a block's largest is that near a power of two, the block may have the other scale: all its values may move by a step
    of the larger. The down sums and the weighted sum are off by n 2^-23 of their terms again."""
    xq = mx4(x)
    T, H = xq.shape
    E, F, _ = gate.shape
    y, off = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for k, e in enumerate(ids[t]):
            if not 0 <= e < E:
                continue
            g, u = gate[e] @ xq[t], up[e] @ xq[t]
            n = (H / 32 + 8) * 2.0 ** -23
            dg, du = n * (np.abs(gate[e]) @ np.abs(xq[t])), n * (np.abs(up[e]) @ np.abs(xq[t]))
            h = swiglu(g, u, limit)
            dh = 1.2 * np.abs(u) * dg + np.abs(g) * du + 2.0 ** -20 * np.abs(h) + 2.0 ** -149
            code, exp, _, a = mx4_parts(h[None])
            hq = mx4(h[None])[0]
            unit = np.repeat(np.exp2(exp[0].astype(float)), 32)[:F]
            r = a.reshape(-1)[:F]
            d = dh / unit
            near = (np.abs(r[:, None] - BORDERS) <= d[:, None]).any(1)
            step = np.where(near, np.where(r < 2, 0.5, np.where(r < 3.9, 1.0, 2.0)), 0.0) * unit
            blocks = np.abs(np.pad(h, (0, -F % 32))).reshape(-1, 32)
            most, at = blocks.max(1), np.pad(dh, (0, -F % 32)).reshape(-1, 32).max(1)
            p = np.exp2(np.round(np.log2(np.maximum(most, 2.0 ** -140))))
            edge = np.repeat(np.where(np.abs(most - p) <= at, 2 * p / 2, 0.0), 32)[:F]  # a step at twice the scale: 2 * 2^(e - 1)
            dq = np.maximum(step, edge)
            o = down[e] @ hq
            m = (F / 32 + 8 + len(ids[t])) * 2.0 ** -23
            y[t] += w[t, k] * o
            off[t] += np.abs(w[t, k]) * (np.abs(down[e]) @ dq + m * (np.abs(down[e]) @ (np.abs(hq) + dq)))
    return y, off
