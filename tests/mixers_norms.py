"""Attention's results held row by row: the 2-norm of a (row, head)'s error against the size of what the row is made of.

What rounding does to a row.  A kernel whose operands keep a relative error of at most u (2^-22 for the two-part operands of f32 rows, half a step of
f16, 2^-11, for f16 rows) makes errors of about u / sqrt(3) in each product, of either sign.  They reach a score as u / sqrt(3) * scale * sqrt(sum_i (q_i
k_i)^2), which is about u / sqrt(3) * scale * |q| * rms(k), and so a weight as that relative error; the weight, the value and (f16) the result are rounded once
more each.  Errors of different weights are independent: a row is off by those relative errors, added in quadrature, of
    size = max(|want|, |(sqrt(sum_j p_j^2 v_jd^2))_d|).
Four times that is the bound for f16 rows: scores are sums of many roundings and so near a normal distribution, of which one in 16000 is further out, and only
the difference of a row's scores' errors matters.  For f32 rows it is six times: the matrix unit's sums are cut as well (up to four steps of 2^-23 a tile of 32 to 128
products, one-sided).  f32 rows also add their slots in tiles: n / 64 rounded additions of 2^-24."""
import numpy as np

U = {"f32": 2.0 ** -22, "f16": 2.0 ** -11}


def attention(q, k, v, pos, scale):
    """As ref_mixers.attention, for many rows: (out, size) in float64; size [T, heads] as above (0 for a row that sees nothing)."""
    T, nq, hd = q.shape
    G, pos = nq // k.shape[1], np.asarray(pos)
    out, size = np.zeros((T, nq, hd)), np.zeros((T, nq))
    for h in range(nq):
        kk, vv = k[:, h // G], v[:, h // G]
        s = q[:, h].astype(np.float64) @ kk.T * scale
        s[np.arange(len(kk))[None] > pos[:, None]] = -np.inf
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0))
        total = p.sum(1, keepdims=True)
        p /= np.where(total == 0, 1, total)
        out[:, h] = p @ vv
        size[:, h] = np.maximum(np.linalg.norm(out[:, h], axis=1), np.sqrt((p * p) @ (vv * vv).sum(1)))
    return out, size


def allowed(q, k, n, scale, act):
    """The relative error of a row: [T, heads]."""
    u = U[act] / np.sqrt(3)
    G = q.shape[1] // k.shape[1]
    rms = np.sqrt((k * k).mean(axis=(0, 2)))  # per KV head
    score = scale * np.linalg.norm(q.astype(np.float64), axis=2) * np.repeat(rms, G)[None]
    rest = 3.0 if act == "f16" else 2.0
    return (4 if act == "f16" else 6) * u * np.sqrt(rest + score ** 2) + n / 64 * 2.0 ** -24


def violations(got, want, size, q, k, n, scale, act):
    """[T, heads]: rows that are further off than rounding explains (f16 results also round to steps of 2^-24 near 0)."""
    err = np.linalg.norm(np.asarray(got, np.float64) - want, axis=2)
    floor = 2.0 ** -25 * np.sqrt(q.shape[2]) if act == "f16" else 0.0
    return ~(err <= allowed(q, k, n, scale, act) * size + floor)


def hold(got, want, size, q, k, n, scale, act):
    bad = violations(got, want, size, q, k, n, scale, act)
    if bad.any():
        err = np.linalg.norm(np.asarray(got, np.float64) - want, axis=2)
        t, h = np.unravel_index(np.argmax(np.where(bad, err / np.maximum(size, 1e-300), 0)), bad.shape)
        raise AssertionError(f"{bad.sum()} of {bad.size} rows are off; row {t}, head {h}: {err[t, h]:.3g} of {size[t, h]:.3g}, "
                             f"allowed {allowed(q, k, n, scale, act)[t, h]:.3g}")
