"""agn_attention_kv_* row by row against 64 bits: every form, layout, head size and share-out, held by the norm of each row's error; rows whose maximum
grows while their slots are worked on; replayed, on a batch with rows that see nothing, and beside other calls."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_F32, AGN_KV_Q8_0_WORDS, AGN_Q8_0
from tests import mixers_norms as norms
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu
KV = {"f16": AGN_F16, "q8_0": AGN_Q8_0, "words": AGN_KV_Q8_0_WORDS}
ACT = {"f32": (AGN_F32, np.float32), "f16": (AGN_F16, np.float16)}


def write(be, kv, k, v, slots):
    """k, v [sequences, n, heads, hd] into caches of `slots` slots; returns the caches and what they hold."""
    m, n, nkv, hd = k.shape
    bpt = be.kv_bytes_per_token(KV[kv], nkv * hd)
    bufs, held = [], []
    for x in (k, v):
        b = be.upload(np.zeros(m * slots * bpt, np.uint8))
        for s in range(m):
            d = be.upload(x[s].reshape(n, -1).astype(np.float32))
            at = b.data_ptr() + s * slots * bpt
            be.kv_write(KV[kv], d, d, at, at, n, nkv * hd, None, slots)
            be.sync()
        bufs.append(b)
        raw = be.read(b, np.uint8, (m, slots, bpt))[:, :n]
        held.append(np.stack([ref.cache_values(KV[kv], r, nkv * hd).reshape(n, nkv, hd) for r in raw]))
    return bufs, held


def prompt(be, kv, act, q, bufs, start, slots, nkv):
    T, nq, hd = q.shape
    out = be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], KV[kv], T, nq, nkv, hd, slots, pos_start=start, act_dtype=ACT[act][0])
    return be.read(out, ACT[act][1], q.shape)


def single(be, kv, act, q, bufs, pos, seq, m, slots, nkv):
    T, nq, hd = q.shape
    out = be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], KV[kv], T, nq, nkv, hd, slots, pos=be.upload(np.asarray(pos, np.int32)),
                                 seq=be.upload(np.asarray(seq, np.int32)), n_seqs=m, act_dtype=ACT[act][0])
    return be.read(out, ACT[act][1], q.shape)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("T,start,nq,nkv,hd", [(1, 0, 4, 2, 64), (8, 0, 28, 4, 128), (13, 500, 8, 8, 64), (16, 4000, 8, 2, 128), (37, 4091, 4, 2, 256), (64, 2936, 4, 1, 256),
                                               (129, 257, 6, 3, 96), (200, 0, 32, 8, 64), (257, 63, 7, 1, 128), (300, 1000, 9, 3, 32), (24, 2000, 4, 1, 64),
                                               (520, 0, 16, 2, 256), (700, 41, 28, 4, 128), (40, 1500, 5, 5, 160), (33, 700, 6, 2, 224)])
def test_prompts(backend, kv, act, T, start, nq, nkv, hd):
    rng, n = np.random.default_rng(T), start + T
    bufs, (k, v) = write(backend, kv, rng.standard_normal((1, n, nkv, hd)), rng.standard_normal((1, n, nkv, hd)), n + 5)
    for size in (1.0, 3.0):
        q = (size * rng.standard_normal((T, nq, hd))).astype(ACT[act][1])
        got = prompt(backend, kv, act, q, bufs, start, n + 5, nkv)
        want, of = norms.attention(q, k[0], v[0], [start + t for t in range(T)], hd ** -0.5)
        norms.hold(got, want, of, q, k[0], n, hd ** -0.5, act)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("nq,nkv,hd", [(28, 4, 128), (8, 8, 64), (16, 2, 256), (12, 3, 96), (32, 8, 128), (20, 1, 64), (9, 9, 32), (4, 2, 192)])
@pytest.mark.parametrize("T,n", [(1, 5000), (5, 900), (40, 300), (600, 70)])
def test_single_rows(backend, kv, act, T, n, nq, nkv, hd):
    rng, m = np.random.default_rng(n + hd), min(T, 3)
    bufs, (k, v) = write(backend, kv, rng.standard_normal((m, n, nkv, hd)), rng.standard_normal((m, n, nkv, hd)), n + 2)
    q = (1.5 * rng.standard_normal((T, nq, hd))).astype(ACT[act][1])
    seq = rng.integers(0, m, T)
    pos = rng.integers(-1, n, T)
    pos[0] = n - 1
    got = single(backend, kv, act, q, bufs, pos, seq, m, n + 2, nkv)
    backend.sync()
    for s in range(m):
        rows = np.flatnonzero(seq == s)
        if len(rows):
            want, of = norms.attention(q[rows], k[s], v[s], pos[rows], hd ** -0.5)
            norms.hold(got[rows], want, of, q[rows], k[s], n, hd ** -0.5, act)
    assert not got[pos < 0].any()


def rising(rng, n, nkv, hd, steps):
    """Keys whose scores against a query along `one` rise (and fall) slot by slot as `steps` says (in nats)."""
    one = np.where(rng.random(hd) < 0.5, -1.0, 1.0)
    return one, (steps / hd ** 0.5)[:, None, None] * one + 0.02 * rng.standard_normal((n, nkv, hd))


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("hd,T,start", [(64, 300, 0), (128, 300, 0), (128, 20, 280), (64, 20, 3000), (256, 150, 0)])
@pytest.mark.parametrize("top", [300, 40])
@pytest.mark.parametrize("shape", ["slowly", "by 10 at every slot", "in jumps of 32 slots", "in jumps of 128", "late in each tile", "falling"])
def test_maxima_that_grow(backend, shape, top, hd, T, start, kv, act):
    """A row's reference maximum is moved when it has been outgrown by 2^8: at the first slots, between pieces of a tile, from tile to tile, again and again."""
    rng, nq, nkv, n = np.random.default_rng(hd + T), 4, 2, start + T
    at = np.arange(n)
    steps = {"slowly": at * 0.25, "by 10 at every slot": at * 10.0, "in jumps of 32 slots": at // 32 * 9.0, "in jumps of 128": at // 128 * 30.0,
             "late in each tile": at // 128 * 20.0 + (at % 128 > 100) * 12.0, "falling": at * -0.25}[shape]
    if shape != "falling":
        steps = steps % (2 * top) - top  # scores of up to 300, over and over
    one, k = rising(rng, n, nkv, hd, steps)
    bufs, (k, v) = write(backend, kv, k[None], rng.standard_normal((1, n, nkv, hd)), n)
    q = (one + 0.02 * rng.standard_normal((T, nq, hd))).astype(ACT[act][1])
    got = prompt(backend, kv, act, q, bufs, start, n, nkv).astype(np.float64)
    want, of = norms.attention(q, k[0], v[0], [start + t for t in range(T)], hd ** -0.5)
    # Scores of hundreds: a score is off by what its products are rounded to (2^-22 of each; f16 keys half a step of f16, 2^-11, and since a slot's keys are all nearly one
    # number here, all of them to the same side: 2^-11 of sum |q k|) and the cuts of their sum (up to 16 of 2^-23 of sum |q k|); that error is a weight's relative one, in
    # the weight and in the sum.
    G = nq // nkv
    qk = [(np.abs(q[:, h].astype(np.float64)) @ np.abs(k[0][:, h // G]).T).max() for h in range(nq)]
    score = hd ** -0.5 * (max(qk) * 9 * 2.0 ** -22 + (max(qk) * 2.0 ** -11 if act == "f16" else 0))
    near = 2 * score + (2.0 ** -9 if act == "f16" else 16 * 2.0 ** -22)
    assert np.all(np.linalg.norm(got - want, axis=2) <= near * of + (2.0 ** -25 * hd ** 0.5 if act == "f16" else 0))


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_same_rows_whatever_the_call_beside_them(backend, act):
    """A prompt's rows, its rows one by one, and two pieces of it agree, each within its own rounding."""
    be, kv, T, nq, nkv, hd = backend, "words", 150, 8, 2, 128
    rng = np.random.default_rng(3)
    bufs, (k, v) = write(be, kv, rng.standard_normal((1, T, nkv, hd)), rng.standard_normal((1, T, nkv, hd)), T)
    q = rng.standard_normal((T, nq, hd)).astype(ACT[act][1])
    want, of = norms.attention(q, k[0], v[0], list(range(T)), hd ** -0.5)
    for got in (prompt(be, kv, act, q, bufs, 0, T, nkv), single(be, kv, act, q, bufs, np.arange(T), np.zeros(T), 1, T, nkv),
                np.concatenate([prompt(be, kv, act, q[:61], bufs, 0, T, nkv), prompt(be, kv, act, q[61:], bufs, 61, T, nkv)])):
        norms.hold(got, want, of, q, k[0], T, hd ** -0.5, act)


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("nq,nkv,hd,T,n,form", [(28, 4, 128, 3, 2000, "rows"), (8, 8, 64, 5, 900, "rows"), (16, 2, 256, 2, 700, "rows"), (6, 3, 96, 1, 5000, "rows"),
                                                (16, 2, 256, 60, 500, "prompt"), (6, 3, 96, 100, 100, "prompt"), (4, 2, 160, 20, 3000, "prompt")])
def test_f16_rows_are_rounded_once(backend, kv, nq, nkv, hd, T, n, form):
    """Single rows, and prompts of head sizes without a form of their own for f16: beside half a step of f16 of each result (2^-11 of it, or of f16's smallest normal
    number), a row is off by what an f32 row may be."""
    rng = np.random.default_rng(n)
    bufs, (k, v) = write(backend, kv, rng.standard_normal((1, n, nkv, hd)), rng.standard_normal((1, n, nkv, hd)), n)
    q = (1.5 * rng.standard_normal((T, nq, hd))).astype(np.float16)
    pos = np.arange(n - T, n)
    got = single(backend, kv, "f16", q, bufs, pos, np.zeros(T), 1, n, nkv) if form == "rows" else prompt(backend, kv, "f16", q, bufs, n - T, n, nkv)
    want, of = norms.attention(q, k[0], v[0], pos, hd ** -0.5)
    off = got.astype(np.float64) - want
    beyond = np.sign(off) * np.maximum(np.abs(off) - 2.0 ** -11 * np.maximum(np.abs(want), 2.0 ** -14), 0)
    norms.hold(want + beyond, want, of, q, k[0], n, hd ** -0.5, "f32")
