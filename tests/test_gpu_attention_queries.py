"""f32 rows whose queries are large in some dims and small in others, with keys the other way round: every dim has its share of the score."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_KV_Q8_0_WORDS, AGN_Q8_0
from tests import mixers_norms as norms
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu
KV = {"f16": AGN_F16, "q8_0": AGN_Q8_0, "words": AGN_KV_Q8_0_WORDS}


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("spread", [1e2, 1e4])
@pytest.mark.parametrize("hd,nq,nkv,T,start", [(64, 8, 2, 16, 100), (128, 4, 2, 40, 2000), (256, 4, 1, 20, 50), (96, 3, 3, 200, 0)])
@pytest.mark.parametrize("form", ["prompt", "single rows"])
def test_small_queries_beside_large_ones(backend, form, hd, nq, nkv, T, start, spread, kv):
    be, n = backend, start + T
    rng, scale = np.random.default_rng(hd), hd ** -0.5
    sizes = np.repeat(spread ** np.linspace(-0.5, 0.5, hd // 32), 32)
    q = (rng.standard_normal((T, nq, hd)) * sizes).astype(np.float32)
    k = rng.standard_normal((n, nkv, hd)) / sizes
    v = rng.standard_normal((n, nkv * hd)).astype(np.float32)
    bpt = be.kv_bytes_per_token(KV[kv], nkv * hd)
    bufs = [be.upload(np.zeros(n * bpt, np.uint8)) for _ in range(2)]
    be.kv_write(KV[kv], be.upload(k.reshape(n, -1).astype(np.float32)), be.upload(v), bufs[0], bufs[1], n, nkv * hd, None, n)
    kw = dict(pos_start=start) if form == "prompt" else dict(pos=be.upload(np.arange(start, n, dtype=np.int32)))
    got = be.read(be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], KV[kv], T, nq, nkv, hd, n, **kw), np.float32, q.shape).astype(np.float64)
    be.sync()
    ck, cv = (ref.cache_values(KV[kv], be.read(b, np.uint8, (n, bpt)), nkv * hd).reshape(n, nkv, hd) for b in bufs)
    want, size = norms.attention(q, ck, cv, [start + t for t in range(T)], scale)
    # the scores' products are off by at most 2^-22 of themselves and cut at 2^-23 of their sum up to 16 times: 9 * 2^-22 of sum |q k| in a weight, twice
    G = nq // nkv
    most = scale * max((np.abs(q[:, h].astype(np.float64)) @ np.abs(ck[:, h // G]).T).max() for h in range(nq))
    assert np.all(np.linalg.norm(got - want, axis=2) <= (18 * most + 16) * 2.0 ** -22 * size)


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("size,scale", [(3.4025e38, 2e-38), (3.4e38, 2e-38), (1e30, 1e-30), (1e-30, 1e30), (1e-36, 1e36)])
@pytest.mark.parametrize("form", ["prompt", "single rows"])
def test_queries_at_the_ends_of_f32s_range(backend, form, size, scale, kv):
    be, hd, nq, nkv, T, n = backend, 64, 4, 2, 20, 90
    rng = np.random.default_rng(5)
    scale = float(np.float32(scale))
    q = (np.where(rng.random((T, nq, hd)) < 0.5, -1, 1) * size * (np.arange(hd) == 3) + 0.1 * size * rng.uniform(-1, 1, (T, nq, hd)) * (np.arange(hd) != 3)).astype(np.float32)
    k, v = (rng.standard_normal((n, nkv * hd)).astype(np.float32) for _ in range(2))
    bpt = be.kv_bytes_per_token(KV[kv], nkv * hd)
    bufs = [be.upload(np.zeros(n * bpt, np.uint8)) for _ in range(2)]
    be.kv_write(KV[kv], be.upload(k), be.upload(v), bufs[0], bufs[1], n, nkv * hd, None, n)
    kw = dict(pos_start=n - T) if form == "prompt" else dict(pos=be.upload(np.arange(n - T, n, dtype=np.int32)))
    got = be.read(be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], KV[kv], T, nq, nkv, hd, n, scale=scale, **kw), np.float32, q.shape)
    be.sync()
    ck, cv = (ref.cache_values(KV[kv], be.read(b, np.uint8, (n, bpt)), nkv * hd).reshape(n, nkv, hd) for b in bufs)
    want, of = norms.attention(q, ck, cv, [n - T + t for t in range(T)], scale)
    # as above; and the scale's own last bit, where it is close to f32's smallest numbers
    most = scale * max((np.abs(q[:, h].astype(np.float64)) @ np.abs(ck[:, h // 2]).T).max() for h in range(nq))
    assert np.all(np.linalg.norm(got - want, axis=2) <= (18 * most + 16) * 2.0 ** -22 * of)
