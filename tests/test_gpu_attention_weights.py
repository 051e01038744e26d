"""f32 rows in which a slot of little weight has the larger value: small beside the row's largest weight is not small beside the result."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_KV_Q8_0_WORDS, AGN_Q8_0
from tests import mixers_norms as norms
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu
KV = {"f16": AGN_F16, "q8_0": AGN_Q8_0, "words": AGN_KV_Q8_0_WORDS}


def run(be, kv, form, hd, T, weight, v, seed):
    """Attends with scores log(weight) (plus a little) over values v; checks every row."""
    nq, nkv, n = 4, 2, len(weight)
    start = n - T
    rng, scale = np.random.default_rng(seed), hd ** -0.5
    one = np.where(rng.random(hd) < 0.5, -1.0, 1.0)
    k = (np.log(weight) / (scale * hd))[:, None, None] * one + 1e-3 * rng.standard_normal((n, nkv, hd))
    q = (one + 0.01 * rng.standard_normal((T, nq, hd))).astype(np.float32)
    bpt = be.kv_bytes_per_token(KV[kv], nkv * hd)
    bufs = [be.upload(np.zeros(n * bpt, np.uint8)) for _ in range(2)]
    be.kv_write(KV[kv], be.upload(k.reshape(n, -1).astype(np.float32)), be.upload(v.reshape(n, -1).astype(np.float32)), bufs[0], bufs[1], n, nkv * hd, None, n)
    kw = dict(pos_start=start) if form == "prompt" else dict(pos=be.upload(np.arange(start, n, dtype=np.int32)))
    got = be.read(be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], KV[kv], T, nq, nkv, hd, n, **kw), np.float32, q.shape).astype(np.float64)
    be.sync()
    ck, cv = (ref.cache_values(KV[kv], be.read(b, np.uint8, (n, bpt)), nkv * hd).reshape(n, nkv, hd) for b in bufs)
    want, size = norms.attention(q, ck, cv, [start + t for t in range(T)], scale)
    # A product of a score is off by at most 2^-22 of itself, and the matrix unit cuts its sum eight times at 2^-23: 5 * 2^-22 of sum |q k|, which is the relative error
    # of a weight (once in the weight, once in the sum); the output's own products and sums add less than 16 * 2^-22.
    most = scale * np.abs(q).astype(np.float64).max() * np.abs(ck).sum(axis=2).max()
    assert np.all(np.linalg.norm(got - want, axis=2) <= (10 * most + 16) * 2.0 ** -22 * size)


VALUES = [("f16", 1e-4, 3e4), ("f16", 1.0, 3e4), ("q8_0", 1e-3, 1e5), ("q8_0", 1e-2, 0.5), ("words", 1e-6, 1e6), ("words", 1e-2, 0.5), ("words", 1e-15, 1e5)]


@pytest.mark.parametrize("kv,small,large", VALUES)
@pytest.mark.parametrize("bits", [12, 25, 34, 45])
@pytest.mark.parametrize("hd,T,start,at", [(128, 40, 150, (10, 30)), (64, 200, 0, (3, 180)), (96, 16, 4000, (5, 3990)), (256, 30, 60, (60, 20))])
@pytest.mark.parametrize("form", ["prompt", "single rows"])
def test_a_light_slot_of_large_values(backend, form, hd, T, start, at, bits, kv, small, large):
    """Slot at[0] has weight 1 and values of size `small`, slot at[1] a weight of 2^-bits and values of size `large`, the others 2^-60 and 1."""
    rng, n = np.random.default_rng(bits), start + T
    weight, v = np.full(n, 2.0 ** -60), rng.standard_normal((n, 2, hd))
    weight[at[0]], weight[at[1]] = 1, 2.0 ** -bits
    for slot, size in zip(at, (small, large)):
        v[slot] = rng.uniform(-2, 2, (2, hd)) * size  # f16 ends at 65504
    run(backend, kv, form, hd, T, weight, v, bits)


@pytest.mark.parametrize("kv,small,large", VALUES)
@pytest.mark.parametrize("bits", [25, 34, 45])
@pytest.mark.parametrize("hd,T,start", [(128, 40, 200), (256, 30, 200)])
def test_light_slots_of_large_values_throughout(backend, hd, T, start, bits, kv, small, large):
    """The same with every slot but the first hundred light and large: a run of slots of one size."""
    rng, n = np.random.default_rng(bits), start + T
    weight, v = np.full(n, 2.0 ** -bits), rng.uniform(1, 2, (n, 2, hd)) * large
    weight[:100] = 1
    v[:100] = rng.uniform(1, 2, (100, 2, hd)) * small
    run(backend, kv, "prompt", hd, T, weight, v, bits)


@pytest.mark.parametrize("hd,T,start", [(128, 40, 150), (64, 300, 0), (128, 16, 3000), (64, 70, 130)])
@pytest.mark.parametrize("bits", [10, 14, 17, 20])
def test_light_slots_of_f16_prompts(backend, hd, T, start, bits):
    """f16 rows over an f16 cache: a weight of 2^-bits with values that outweigh those of the slot of weight 1 by as much."""
    be, nq, nkv, n = backend, 4, 2, start + T
    rng, scale = np.random.default_rng(bits), hd ** -0.5
    weight, v = np.full(n, 2.0 ** -30), rng.uniform(-2, 2, (n, nkv, hd)) * 1e-3
    weight[2], weight[n // 2] = 1, 2.0 ** -bits
    v[n // 2] *= 2.0 ** bits
    one = np.where(rng.random(hd) < 0.5, -1.0, 1.0)
    k = ((np.log(weight) / (scale * hd))[:, None, None] * one + 1e-3 * rng.standard_normal((n, nkv, hd))).astype(np.float16)
    v = np.ascontiguousarray(v, np.float16)
    q = (one + 0.01 * rng.standard_normal((T, nq, hd))).astype(np.float16)
    bufs = [be.upload(x.reshape(n, -1)) for x in (k, v)]
    got = be.read(be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], AGN_F16, T, nq, nkv, hd, n, pos_start=start, act_dtype=AGN_F16), np.float16, q.shape)
    k, v = k.astype(np.float64), v.astype(np.float64)
    want, size = norms.attention(q, k, v, [start + t for t in range(T)], scale)
    # queries, keys and values are f16 as they are: a weight is rounded once (2^-11) and the result once (2^-11, or 2^-25 for its subnormals); scores as for f32 rows
    most = scale * np.abs(q).astype(np.float64).max() * np.abs(k).sum(axis=2).max()
    assert np.all(np.linalg.norm(got - want, axis=2) <= (2.0 ** -10 + 10 * most * 2.0 ** -22) * size + 2.0 ** -25 * hd ** 0.5)
