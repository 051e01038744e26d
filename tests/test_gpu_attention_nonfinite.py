"""Values that are not finite in a slot of hardly any weight: what the row's formula multiplies by a weight above 0 does not vanish, however the slots are shared out."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_F32, AGN_KV_Q8_0_WORDS, AGN_Q8_0

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("T,start", [(16, 4000), (40, 0), (20, 1000)])
@pytest.mark.parametrize("form", ["f32", "f16", "f32 single rows", "f16 single rows"])
def test_a_block_scale_that_is_not_finite(backend, form, T, start, hd, bad):
    """Slot 5's value scale of one block (32 dims of KV head 0), under a weight of about 2^-180 of the largest: every row behind it sees it."""
    be, nq, nkv, n = backend, 4, 2, start + T
    rng, scale = np.random.default_rng(hd), hd ** -0.5
    k = np.ones((n, nkv, hd)) / (scale * hd) + 1e-3 * rng.standard_normal((n, nkv, hd))
    k[:min(128, n // 2)] *= -125.0  # e^-125, and so what the first shares of the slots hold throughout
    q = (1 + 0.01 * rng.standard_normal((T, nq, hd))).astype(np.float16 if form.startswith("f16") else np.float32)
    bpt = be.kv_bytes_per_token(AGN_KV_Q8_0_WORDS, nkv * hd)
    bufs = [be.upload(np.zeros(n * bpt, np.uint8)) for _ in range(2)]
    v = rng.standard_normal((n, nkv * hd)).astype(np.float32)
    be.kv_write(AGN_KV_Q8_0_WORDS, be.upload(k.reshape(n, -1).astype(np.float32)), be.upload(v), bufs[0], bufs[1], n, nkv * hd, None, n)
    raw = be.read(bufs[1], np.uint8, (n, bpt)).copy()
    raw[5, :4] = np.array([bad], np.float32).view(np.uint8)
    be.copy_h2d(bufs[1], raw)
    be.sync()
    kw = dict(pos=be.upload(np.arange(start, n, dtype=np.int32))) if "rows" in form else dict(pos_start=start)
    out = be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], AGN_KV_Q8_0_WORDS, T, nq, nkv, hd, n, act_dtype=AGN_F16 if q.dtype == np.float16 else AGN_F32, **kw)
    got = be.read(out, q.dtype.type, q.shape)
    sees = np.arange(start, n) >= n // 2  # and slots of weight 1 too
    assert not np.isfinite(got[sees][:, :2, :32]).any()
    assert np.isfinite(got[:5] if start == 0 else got[:0]).all() and np.isfinite(got[:, :2, 32:]).all() and np.isfinite(got[:, 2:]).all()


@pytest.mark.parametrize("kv", ["q8_0", "words"])
@pytest.mark.parametrize("act", [AGN_F32, AGN_F16])
@pytest.mark.parametrize("slots", [20, 3000])
def test_a_scale_of_nan_in_a_batch_of_single_rows(backend, act, kv, slots):
    """A value block whose scale is NaN, under a weight like the others': its dims are NaN in every row that sees it, and in no other."""
    be, nq, nkv, hd, n = backend, 8, 2, 64, 3
    rng, dt = np.random.default_rng(slots), AGN_Q8_0 if kv == "q8_0" else AGN_KV_Q8_0_WORDS
    width = nkv * hd
    bpt = be.kv_bytes_per_token(dt, width)
    bufs = [be.upload(np.zeros(n * slots * bpt, np.uint8)) for _ in range(2)]
    for s in range(n):
        k, v = (rng.standard_normal((slots, width)).astype(np.float32) for _ in range(2))
        be.kv_write(dt, be.upload(k), be.upload(v), *(b.data_ptr() + s * slots * bpt for b in bufs), slots, width, None, slots)
    be.sync()
    raw = be.read(bufs[1], np.uint8, (n, slots, bpt)).copy()
    block, scale = (34, np.array([0x7E00], np.uint16)) if kv == "q8_0" else (36, np.array([np.nan], np.float32))
    at = (hd // 32 + 1) * block  # the second block of KV head 1: dims 32 to 63
    raw[1, 11, at:at + scale.nbytes] = scale.view(np.uint8)
    be.copy_h2d(bufs[1], raw)
    be.sync()
    q = rng.standard_normal((4, nq, hd)).astype(np.float32 if act == AGN_F32 else np.float16)
    out = be.launch_attention_kv(be.upload(q), bufs[0], bufs[1], dt, 4, nq, nkv, hd, slots, pos=be.upload(np.array([slots - 1, slots - 1, 10, slots - 1], np.int32)),
                                 seq=be.upload(np.array([0, 1, 1, 2], np.int32)), n_seqs=n, act_dtype=act)
    got = be.read(out, q.dtype.type, q.shape)
    assert np.isnan(got[1, 4:, 32:]).all()
    got[1, 4:, 32:] = 0
    assert np.isfinite(got).all()
