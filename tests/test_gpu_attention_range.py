"""f16 prompts over quantised caches whose keys or values f16 does not hold: too large, or all below its normal numbers.  The rows that see them
are computed in f32, and agree with the form for single rows, which never turns the cache into f16."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_KV_Q8_0_WORDS, AGN_Q8_0
from tests import mixers_norms as norms
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu
KV = {"q8_0": AGN_Q8_0, "words": AGN_KV_Q8_0_WORDS}


def attend(be, kv, q, k, v, start, slots, scale, single=False):
    """Writes k and v, attends; (got, the cache's k, its v)."""
    T, nq, hd = q.shape
    nkv, n = k.shape[1], k.shape[0]
    bpt = be.kv_bytes_per_token(KV[kv], nkv * hd)
    bufs = [be.upload(np.zeros(slots * bpt, np.uint8)) for _ in range(2)]
    be.kv_write(KV[kv], be.upload(k.reshape(n, -1).astype(np.float32)), be.upload(v.reshape(n, -1).astype(np.float32)), bufs[0], bufs[1], n, nkv * hd, None, slots)
    kw = dict(pos=be.upload(np.arange(start, start + T, dtype=np.int32))) if single else dict(pos_start=start)
    out = be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], KV[kv], T, nq, nkv, hd, slots, scale=scale, act_dtype=AGN_F16, **kw)
    got = be.read(out, np.float16, q.shape)
    be.sync()
    return [got] + [ref.cache_values(KV[kv], be.read(b, np.uint8, (n, bpt)), nkv * hd).reshape(n, nkv, hd) for b in bufs]


def held(be, kv, q, k, v, start, scale):
    n = k.shape[0]
    got, ck, cv = attend(be, kv, q, k, v, start, n + 3, scale)
    assert be.last_kernel in ("attention_kv_prompt", "attention_kv_join")
    pos = [start + t for t in range(q.shape[0])]
    with np.errstate(over="ignore"):
        want, size = norms.attention(q, ck, cv, pos, scale)
    one = attend(be, kv, q, k, v, start, n + 3, scale, single=True)[0]
    fits = (np.abs(want) < 6e4).all(axis=2)  # 65520 and more are infinity in an f16 result; between the two, rounding decides
    for x in (got, one):
        x = x.astype(np.float64)
        assert np.all(np.isfinite(x[fits])) and np.all(x[np.abs(want) > 7e4] == np.sign(want[np.abs(want) > 7e4]) * np.inf)
        norms.hold(np.where(fits[..., None], x, want), want, size, q, ck, n, scale, "f16")


SHAPES = [(9, 0, 4, 2, 64), (40, 100, 8, 2, 128), (300, 0, 8, 2, 64), (150, 130, 7, 1, 128), (16, 3000, 4, 1, 64), (24, 2000, 8, 2, 128)]


@pytest.mark.parametrize("kv", ["q8_0", "words"])
@pytest.mark.parametrize("T,start,nq,nkv,hd", SHAPES)
def test_large_values(backend, kv, T, start, nq, nkv, hd):
    """Some slots hold values of up to 10^6, in one KV head; their weight is small enough for an f16 result (a key that points away from every query)."""
    rng, n = np.random.default_rng(T), start + T
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in range(2))
    q = rng.standard_normal((T, nq, hd)) + 1.0
    for s in {0, n // 3, n - 1}:
        v[s, 0] *= 3e5
        k[s, 0] = -0.7 * np.ones(hd) * 8 / np.sqrt(hd)
    held(backend, kv, q.astype(np.float16), k, v, start, hd ** -0.5)


@pytest.mark.parametrize("kv", ["q8_0", "words"])
@pytest.mark.parametrize("size", [1e5, 1e6, 2e-6, 3e-7])
@pytest.mark.parametrize("T,start,nq,nkv,hd", SHAPES)
def test_keys_beyond_f16_and_a_scale_that_takes_it_back(backend, kv, size, T, start, nq, nkv, hd):
    if kv == "q8_0" and size < 1e-5:
        size *= 20  # the block's own scale is f16: what it holds itself
    rng, n = np.random.default_rng(T + 1), start + T
    k, v = (rng.standard_normal((n, nkv, hd)) for _ in range(2))
    q = rng.standard_normal((T, nq, hd))
    held(backend, kv, q.astype(np.float16), k * size, v, start, float(np.float32(hd ** -0.5 / size)))


def test_one_large_key_in_a_late_tile(backend):
    """Rows of other tiles and heads stay with the tensor cores; a row that sees the large key gives it all its weight or none."""
    T, nq, nkv, hd = 400, 4, 2, 128
    rng = np.random.default_rng(4)
    k, v = (rng.standard_normal((T, nkv, hd)) for _ in range(2))
    k[300, 1] *= 1e5
    held(backend, "words", rng.standard_normal((T, nq, hd)).astype(np.float16), k, v, 0, hd ** -0.5)
