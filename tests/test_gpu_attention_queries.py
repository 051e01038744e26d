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
