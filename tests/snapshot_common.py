"""The served snapshots' definition in plain 64-bit numpy, with the error a 32-bit evaluation may make beside every value."""
import numpy as np

U = 2.0 ** -24                     # half a step of fp32, relative
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def split_flat(flat, dims):
    """flat rows [G x P] -> [(W [G, out, in], b [G, out])]"""
    out, at = [], 0
    for i, o in zip(dims, dims[1:]):
        out.append((flat[:, at:at + i * o].reshape(-1, o, i), flat[:, at + i * o:at + i * o + o]))
        at += i * o + o
    return out


def n_params(dims):
    return sum(i * o + o for i, o in zip(dims, dims[1:]))


def round4(w):
    """what fp32 weights [.., in] stand for in 4 bits (E2M1 with a power of two for 32 inputs); NaN where an output has a
    weight that is not finite or is 2^126 or more"""
    w = np.asarray(w, np.float64)
    out = np.zeros_like(w)
    for b in range(0, w.shape[-1], 32):
        v = w[..., b:b + 32]
        a = np.abs(v).max(-1, keepdims=True)
        live = np.isfinite(a) & (a >= 2.0 ** -118) & (a < 2.0 ** 126)
        e = np.ceil(np.log2(np.where(live, a, 6.0) / 6.0))
        s = 2.0 ** e
        q = np.where(live, v / s, 0.0)
        m = np.abs(q)
        step = np.where(m < 2, 0.5, np.where(m < 4, 1.0, 2.0))
        out[..., b:b + 32] = np.copysign(np.round(m / step) * step, q) * s
    return out


def act(kind, z):
    if kind == 1:
        return np.where(z > 0, z, np.float64(np.float32(0.01)) * z)
    if kind == 2:
        return np.tanh(z)
    if kind == 3:
        return np.where(z > 0, z, 0 * z)
    return z


def forward(layers, x, hidden, last):
    """x [.., n, in] through nets [.., out, in] -> (y, bound): a 32-bit evaluation is within `bound` of y, for any order of the
    sums: with K terms, |error of a sum| <= (K + 1) U sum |w||x| (K products and K additions in 32 bits, the bias's among them);
    what the inputs are off by comes through |w|; leaky, tanh and ReLU do not enlarge it; their own rounding is within 4 U of
    the value (tanhf: 2 units in the last place, each 2 U at most)."""
    h, e = np.asarray(x, np.float64), np.zeros(np.shape(x))
    for i, (w, b) in enumerate(layers):
        wt = np.swapaxes(np.asarray(w, np.float64), -1, -2)
        b = np.asarray(b, np.float64)[..., None, :]
        k = w.shape[-1]
        with np.errstate(all="ignore"):
            z = h @ wt + b
            e = (k + 1) * U * (np.abs(h) @ np.abs(wt) + np.abs(b)) + (1 + (k + 1) * U) * (e @ np.abs(wt))
            h = act(last if i == len(layers) - 1 else hidden, z)
            e = e + 4 * U * np.abs(h)
    return h, e + 1e-37


def stored(layers, bits):
    return [(round4(w) if bits == 4 else w, b) for w, b in layers]


def mixture(layers, x, rw, rb, k, allowed, hidden, last):
    """-> out, its bound, idx, prob, y"""
    n, g = x.shape[0], rw.shape[0]
    with np.errstate(all="ignore"):                              # (summed in the same order for every agent: equal rows give equal logits)
        logits = (x.astype(np.float64)[:, None, :] * rw.astype(np.float64)[None]).sum(-1) + (0 if rb is None else rb.astype(np.float64))
    if allowed is not None:
        logits = np.where(np.broadcast_to(allowed, (n, g)) != 0, logits, -np.inf)
    a = layers[-1][1].shape[-1]
    idx, prob, y, ye = np.full((n, k), -1), np.zeros((n, k)), np.zeros((n, k, a)), np.zeros((n, k, a))
    for t in range(n):
        order = sorted((e for e in range(g) if not logits[t, e] == -np.inf),
                       key=lambda e: (-np.inf if np.isnan(logits[t, e]) else -logits[t, e], not np.isnan(logits[t, e]), e))[:k]
        if not order:
            continue
        l = logits[t, order]
        with np.errstate(all="ignore"):
            p = np.exp(l - l[0])
            prob[t, :len(order)] = p / p.sum()
        idx[t, :len(order)] = order
        for j, e in enumerate(order):
            v, b = forward([(w[e], bb[e]) for w, bb in layers], x[t:t + 1], hidden, last)
            y[t, j], ye[t, j] = v[0], b[0]
    out = (prob[..., None] * y).sum(1)
    # prob: the argument of exp is a 64-bit difference rounded once (|argument| U), expf 2 units in the last place (4 U), a sum of
    # k and a division ((k + 1) U), the sum's terms off alike: (2 * 4 + 2 * 88 + k + 1) U is above all of it where exp(-88) ends
    pe = (8 + 176 + k + 1) * U
    bound = (prob[..., None] * (ye + (pe + (k + 1) * U) * (np.abs(y) + ye))).sum(1) + 1e-37
    return out, bound, idx, prob, y


def mixture_grad(x, idx, prob, y, dout, g):
    """-> dw, db, dy and bounds of dw, db: a place's dot products have A terms, the sum over places k, sums over rows are exact
    to U (64 bits, one rounding)"""
    x, prob, y, dout = (np.asarray(v, np.float64) for v in (x, prob, y, dout))
    n, k, a = y.shape
    ok = (idx >= 0) & (idx < g)
    p = np.where(ok, prob, 0.0)
    score = (y * dout[:, None]).sum(-1)
    dl = p * (score - (p * score).sum(1, keepdims=True))
    mag = (np.abs(y) * np.abs(dout[:, None])).sum(-1)
    dle = (a + k + 4) * U * np.abs(p) * (mag + (np.abs(p) * mag).sum(1, keepdims=True))
    dw, db, dwe, dbe = np.zeros((g, x.shape[1])), np.zeros(g), np.zeros((g, x.shape[1])), np.zeros(g)
    for t, j in zip(*np.nonzero(ok)):
        dw[idx[t, j]] += dl[t, j] * x[t]; db[idx[t, j]] += dl[t, j]
        dwe[idx[t, j]] += dle[t, j] * np.abs(x[t]); dbe[idx[t, j]] += dle[t, j]
    return dw, db, p[..., None] * dout[:, None], dwe + 2 * U * np.abs(dw) + 1e-37, dbe + 2 * U * np.abs(db) + 1e-37
