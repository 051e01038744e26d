"""Plain 64-bit statements of the token mixers: attention over the KV cache, the gated delta rule, the gated norm."""
import numpy as np

from agention_infer_b200 import AGN_F16, AGN_KV_Q8_0_WORDS, AGN_Q8_0

U32, U16 = 2.0 ** -24, 2.0 ** -11  # half a step of f32 / f16


def cache_values(kv_dtype, raw, width):
    """Cache bytes [slots, bytes_per_token] -> float64 [slots, width]."""
    raw = np.ascontiguousarray(raw)
    with np.errstate(all="ignore"):
        if kv_dtype == AGN_F16:
            return raw.view(np.float16).astype(np.float64)
        size = {AGN_Q8_0: 34, AGN_KV_Q8_0_WORDS: 36}[kv_dtype]
        b = raw.reshape(raw.shape[0], -1, size)
        if kv_dtype == AGN_Q8_0:
            x = b[..., :2].copy().view(np.float16).astype(np.float64) * b[..., 2:].copy().view(np.int8)
        else:
            x = b[..., :4].copy().view(np.float32).astype(np.float64) * (b[..., 4:].astype(np.float64) - 128)
        return x.reshape(raw.shape[0], -1)[:, :width]


def attention(q, k, v, pos, scale):
    """q [T, nq, hd]; k, v: [slots, nkv, hd] float64 of the one sequence the rows share; pos [T] -> (out, weight) in float64.
    weight = sum_j p_j |v_j|: what a relative error of every p_j moves the output by."""
    T, nq, hd = q.shape
    G = nq // k.shape[1]
    out, mag = np.zeros((T, nq, hd)), np.zeros((T, nq, hd))
    for t in range(T):
        n = pos[t] + 1
        if n <= 0:
            continue
        for h in range(nq):
            kk, vv = k[:n, h // G], v[:n, h // G]
            s = kk @ q[t, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h], mag[t, h] = p @ vv, p @ np.abs(vv)
    return out, mag


def attention_bound(q, k, mag, n, scale, operand=0.0):
    """Largest error of the kernels' output.  A score is a sum of hd products, each rounded (at most U32 of it, or `operand` where an
    operand was rounded to fewer bits) and summed in f32: off by (hd + 8) U32 + operand of sum |q k|.  exp turns that into a relative
    error of p, once in the weight and once in the sum; exp itself and the scaling add 8 U32.  The weights and the values may
    be rounded once more (2 operand), and the sum over the slots is taken in tiles of at most 128 in the matrix unit, whose adder
    cuts instead of rounding (2 U32 a step), the tiles then added one after the other."""
    hd = q.shape[-1]
    big = np.abs(q).astype(np.float64).max(axis=-1)[..., None] * np.abs(k).sum(axis=-1).max() * scale  # >= sum |q k| of any slot
    rel = 2 * ((hd + 8) * U32 + operand) * big + 2 * operand + (8 + 2 * 128 + n / 8) * U32
    return mag * rel + 1e-30


def delta_rule(q, k, v, g, beta, S, scale, eps):
    """One sequence: q, k [n, nk, dk]; v [n, nv, dv]; g, beta [n, nv]; S [nv, dk, dv] -> (out, S) in float64, token by token."""
    q, k, v, S = (x.astype(np.float64) for x in (q, k, v, S))
    if eps >= 0:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    rep = v.shape[1] // k.shape[1]
    q, k = (np.repeat(x, rep, axis=1) for x in (q * scale, k))
    out = np.zeros(v.shape)
    for t in range(v.shape[0]):
        S = S * np.exp(g[t].astype(np.float64))[:, None, None]
        d = beta[t].astype(np.float64)[:, None] * (v[t] - np.einsum("hkv,hk->hv", S, k[t]))
        S = S + k[t][:, :, None] * d[:, None, :]
        out[t] = np.einsum("hkv,hk->hv", S, q[t])
    return out, S


def gated_norm(x, gate, w, eps):
    x, z = x.astype(np.float64), gate.astype(np.float64)
    return w.astype(np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * z / (1 + np.exp(-z))
