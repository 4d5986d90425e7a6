"""Plain implementations in 64 bits of the dispatch of routed tokens and of 8-bit integers with a scale a row."""
import numpy as np

from tests.ops_ref import EPS, pad128, swiglu  # noqa: F401


def dispatch(ids, E):
    """order, places and offsets of ids (T, K)."""
    flat = np.asarray(ids).ravel().astype(np.int64)
    counts = (flat >= 0) & (flat < E)
    a = np.nonzero(counts)[0]
    by = a[np.argsort(flat[a], kind="stable")]
    order = np.full(flat.size, -1)
    order[:len(by)] = by
    places = np.full(flat.size, -1)
    places[by] = np.arange(len(by))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[a], minlength=E))])
    return order, places.reshape(np.shape(ids)), offsets


def combine(o, places, w=None):
    """Each token's sum, and the sum of its terms' sizes."""
    T, K = places.shape
    y, size = np.zeros((T, o.shape[1])), np.zeros((T, o.shape[1]))
    for k in range(K):
        t = np.nonzero((places[:, k] >= 0) & (places[:, k] < T * K))[0]
        v = o[places[t, k]] * (1.0 if w is None else w[t, k:k + 1].astype(np.float64))
        y[t] += v
        size[t] += np.abs(v)
    return y, size


def i8_scales(x):
    """Rows' scales (fp32's largest |x| / 127, rounded once) as doubles; NaN for a row that is not finite."""
    most = np.abs(np.asarray(x, np.float64)).max(-1)
    bad = ~(most < np.inf)
    s = np.maximum((np.where(bad, 1.0, most) / 127).astype(np.float32).astype(np.float64), 2.0 ** -100)
    return np.where(bad, np.nan, s)


def i8_quantize(x):
    """Codes (rows, cols) and scales. (Operands of 24 bits: a quotient that is not halfway is 2^-32 of itself or more away from
    it, so the double's rounding does not hide it.)"""
    x, s = np.asarray(x, np.float64), i8_scales(x)
    bad = np.isnan(s)[:, None]
    return np.where(bad, 0, np.rint(np.where(bad, 0.0, x) / np.where(bad, 1.0, s[:, None]))).astype(np.int64), s


def i8_padded(codes):
    out = np.zeros((codes.shape[0], pad128(codes.shape[1])), np.int8)
    out[:, :codes.shape[1]] = codes
    return out


def i8_product(xc, xs, wc, ws):
    """The product's value and the bound of its three roundings in fp32 (the sum's, the two scales')."""
    y = (xc.astype(np.float64) @ wc.astype(np.float64).T) * xs[:, None] * ws  # (sums of at most 2^30: exact)
    return y, 3 * 2.0 ** -24 * np.abs(y) + 2.0 ** -148


def i8_experts(x, ids, w, gate, up, down, limit=0.0):
    """y and how far it may be off; gate, up, down: (codes (E, rows, cols), scales (E, rows)).

    The bound: g and u are off by three roundings, h by those and by 2^-20 of itself (the SiLU's roundings, an exponential good to
    a few of them; the SiLU's slope is at most 1.1). A row's scale moves with its largest |h| and one rounding; a code whose
    quotient lies that near a border between two may be either, the others' values move with the scale. Each value of down is off
    by three roundings, their sum by one a rank."""
    xc, xs = i8_quantize(x)
    T, H = xc.shape
    E = gate[0].shape[0]
    y, off = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for k, e in enumerate(ids[t]):
            if not 0 <= e < E:
                continue
            g, u = ((m[0][e].astype(np.float64) @ xc[t].astype(np.float64)) * xs[t] * m[1][e] for m in (gate, up))
            three = 3.01 * 2.0 ** -24
            h = swiglu(g, u, limit)
            dh = three * (1.2 * np.abs(u * g) + np.abs(g * u)) + 2.0 ** -20 * np.abs(h) + 2.0 ** -140
            s = i8_scales(h[None])[0]
            ds = dh[np.abs(h).argmax()] / 127 + 2.0 ** -23 * s
            at = np.abs(h) >= np.abs(h).max() - 2 * dh.max()  # (whichever is the largest)
            ds = max(ds, dh[at].max() / 127 + 2.0 ** -23 * s)
            r = h / s
            q = np.rint(r)
            near = np.abs(np.abs(r - q) - 0.5) <= dh / s + np.abs(r) * ds / s + 2.0 ** -40
            dq = np.where(near, s, 0.0) + (np.abs(q) + 1) * ds
            dc, dsc = down[0][e].astype(np.float64), down[1][e]
            o = (dc @ q) * s * dsc
            do = (np.abs(dc) @ dq) * dsc + three * np.abs(o)
            y[t] += w[t, k] * o
            off[t] += np.abs(w[t, k]) * (do + (len(ids[t]) + 1) * 2.0 ** -24 * (np.abs(o) + do))
    return y, off * 1.001 + 2.0 ** -140
