"""The 8-bit integer path in numpy and 64 bits, from the definitions: what the GPU tests compare with."""
import numpy as np

EPS24 = 2.0 ** -24                                                     # largest relative error of one rounding to f32


def bf16(x):
    """values rounded to bf16, nearest even, as float64"""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = (((b + 0x7FFF + ((b >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, x).astype(np.float64)


def route(logits, topk, sigmoid, bias=None, groups=1, kept=0, rank=1, norm=True, scale=1.0):
    """-> (ids, weights); one token after the other, the largest first, the lowest index of equals"""
    l = np.asarray(logits, np.float64); T, E = l.shape
    kept, size = kept or groups, E // groups
    ids, wts = np.empty((T, topk), np.uint32), np.empty((T, topk))
    for t in range(T):
        nan = np.isnan(l[t])
        if sigmoid:
            with np.errstate(over="ignore"):
                s = 1.0 / (1.0 + np.exp(-l[t]))
        else:
            top = np.max(np.where(nan, -np.inf, l[t]))
            with np.errstate(invalid="ignore"):
                e = np.where(l[t] == top, 1.0, np.exp(l[t] - top))
            e[nan | (l[t] == -np.inf)] = 0.0
            s = e / e.sum() if e.sum() > 0 else e
        s = np.where(nan, 0.0, s).astype(np.float32)
        c = s if bias is None else (s + np.asarray(bias, np.float32)).astype(np.float32)
        c = np.where(nan | np.isnan(c), -np.inf, c); low = nan | np.isnan(s if bias is None else s + bias)
        order = lambda v, worst: sorted(range(len(v)), key=lambda i: (worst[i], -v[i], i))     # noqa: E731
        alive = np.ones(E, bool)
        if kept < groups:
            best = [float(np.sum(np.sort(c[g * size:(g + 1) * size].astype(np.float32))[::-1][:rank], dtype=np.float32)) for g in range(groups)]
            keep = order(best, np.zeros(groups, bool))[:kept]
            alive = np.isin(np.arange(E) // size, keep)
        picks = [e for e in order(c, low) if alive[e]][:topk]
        ids[t] = picks
        w = s[picks].astype(np.float64)
        wts[t] = (w / (w.sum() + 1e-20) if norm else w) * scale
    return ids, wts


def quant(y):
    """-> (y / s unrounded, s) of float64 rows; NaN scale where a row is not finite"""
    fine = np.isfinite(y).all(1)
    top = np.maximum(np.abs(np.where(np.isfinite(y), y, 0)).max(1), 2.0 ** -100)
    s = np.where(fine, top / 127, np.nan)
    return np.where(fine[:, None], y / (top / 127)[:, None], 0.0), s


def codes(y):
    v, s = quant(y)
    return np.clip(np.rint(v), -127, 127), s


def norm(h, w, eps):
    with np.errstate(invalid="ignore", over="ignore"):
        return h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * (1.0 if w is None else np.asarray(w, np.float64))


def gate(gu):
    g, u = np.split(np.asarray(gu, np.float64), 2, axis=1)
    with np.errstate(invalid="ignore", over="ignore"):
        return g / (1 + np.exp(-g)) * u


def gemm(x, xs, w, ws):
    """exact sums: at most 2^29, so float64 holds them"""
    return (x.astype(np.float64) @ w.astype(np.float64).T) * (np.asarray(xs, np.float64)[:, None] * np.asarray(ws, np.float64))


def layer(ids, wts, q, s, gu, gus, dn, dns):
    """codes and scales of the input rows, expert weights int8 [E][2I][H] / [E][H][I] -> f64 [T][H]"""
    T, H = q.shape
    out = np.zeros((T, H))
    for e in range(len(gu)):
        t, slot = np.nonzero(ids == e)
        if not len(t):
            continue
        a, sa = codes(gate(bf16(gemm(q[t], s[t], gu[e], gus[e]))))
        np.add.at(out, t, bf16(gemm(a, sa, dn[e], dns[e])) * wts[t, slot][:, None])
    return out
