"""agn_attention_kv_* against a 64-bit statement: the three cache layouts, f32 and f16 rows, both forms, lengths at and next to the
tiles' borders, rows that see nothing, whatever stands in the slots that a row does not see, refusals."""
import numpy as np
import pytest

import agention_infer_b200 as agn
from agention_infer_b200 import AGN_F16, AGN_F32, AGN_KV_Q8_0_WORDS, AGN_Q4_K, AGN_Q8_0, BackendError
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu
KV = {"f16": AGN_F16, "q8_0": AGN_Q8_0, "words": AGN_KV_Q8_0_WORDS}
ACT = {"f32": AGN_F32, "f16": AGN_F16}


def np_act(act):
    return np.float32 if act == "f32" else np.float16


class Cache:
    """n sequences of `slots` slots on the GPU: the first lens[s] slots of sequence s written by kv_write, the others left at
    bytes that read as NaN or infinity where the layout can hold them."""

    def __init__(self, be, rng, kv, n, slots, nkv, hd, lens, spread=1.0):
        self.be, self.kv, self.slots, self.nkv, self.hd = be, KV[kv], slots, nkv, hd
        self.bpt = be.kv_bytes_per_token(self.kv, nkv * hd)
        self.bufs = []
        for which in range(2):
            raw = np.full((n, slots, self.bpt), 0xFF, np.uint8)  # f16 0xFFFF and f32 0xFFFFFFFF are NaN
            if kv == "f16":
                raw[:, 1::2] = np.tile(np.array([0x00, 0x7C], np.uint8), self.bpt // 2)  # +infinity
            self.bufs.append(be.upload(raw))
        for s in range(n):
            if lens[s] == 0:
                continue
            k, v = (rng.standard_normal((lens[s], nkv * hd)).astype(np.float32) * np.float32(spread) for _ in range(2))
            at = [b.data_ptr() + s * slots * self.bpt for b in self.bufs]
            be.kv_write(self.kv, be.upload(k), be.upload(v), at[0], at[1], lens[s], nkv * hd, None, slots)
            be.sync()
        self.n = n

    def values(self, s, upto):
        """(k, v) float64 [upto, nkv, hd] of sequence s as the cache holds them."""
        out = []
        for b in self.bufs:
            raw = self.be.read(b.data_ptr() + s * self.slots * self.bpt, np.uint8, (upto, self.bpt))
            out.append(ref.cache_values(self.kv, raw, self.nkv * self.hd).reshape(upto, self.nkv, self.hd))
        return out


def close(got, want, mag, q, k, n, scale, act, operand=None):
    if operand is None:
        operand = 0.0 if act == "f32" else 3 * ref.U16  # f16 kernels may round keys, weights and values
    bound = ref.attention_bound(q, k, mag, n, scale, operand)
    if act == "f16":
        bound = bound + ref.U16 * np.abs(want) + 2.0 ** -25
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= bound), (err.max(), bound.flat[np.argmax(err - bound)])


def run_decode(be, cache, q, pos, seq, act, scale=None, **kw):
    T, nq, hd = q.shape
    out = be.launch_attention_kv(be.upload(q), cache.bufs[0], cache.bufs[1], cache.kv, T, nq, cache.nkv, hd, cache.slots,
                                 pos=be.upload(np.asarray(pos, np.int32)), seq=None if seq is None else be.upload(np.asarray(seq, np.int32)),
                                 n_seqs=cache.n, scale=scale, act_dtype=ACT[act], **kw)
    return be.read(out, np_act(act), q.shape)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("nq,nkv,hd", [(28, 4, 128), (8, 8, 64), (16, 2, 256), (12, 3, 96), (24, 1, 32)])
def test_decode_lengths_and_heads(backend, kv, act, nq, nkv, hd):
    rng = np.random.default_rng(nq * 1000 + hd)
    lens = [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257]
    c = Cache(backend, rng, kv, len(lens), 260, nkv, hd, lens)
    order = [int(s) for s in rng.permutation(len(lens))]
    q = rng.standard_normal((len(lens) + 1, nq, hd)).astype(np_act(act))
    pos = [lens[s] - 1 for s in order] + [-1]
    got = run_decode(backend, c, q, pos, order + [0], act)
    backend.sync()
    assert np.array_equal(got[-1], np.zeros_like(got[-1]))  # a row that sees nothing
    for i, s in enumerate(order):
        k, v = c.values(s, lens[s])
        want, mag = ref.attention(q[i:i + 1], k, v, [lens[s] - 1], hd ** -0.5)
        close(got[i:i + 1], want, mag, q[i:i + 1], k, lens[s], hd ** -0.5, act)


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("T", [1, 3])
def test_long_row_is_split_and_joined(backend, kv, T):
    """Few rows over a long cache: the slots are shared out and the parts joined."""
    nq, nkv, hd, n = 8, 2, 64, 5003
    rng = np.random.default_rng(5)
    c = Cache(backend, rng, kv, 1, n + 9, nkv, hd, [n])
    q = (3 * rng.standard_normal((T, nq, hd))).astype(np.float32)
    pos = [n - 1, 17, 2500][:T]
    got = run_decode(backend, c, q, pos, None, "f32")
    k, v = c.values(0, n)
    want, mag = ref.attention(q, k, v, pos, hd ** -0.5)
    close(got, want, mag, q, k, n, hd ** -0.5, "f32")


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("T,start,nq,nkv,hd", [(1, 0, 4, 2, 64), (5, 0, 28, 4, 128), (70, 0, 28, 4, 128), (33, 100, 8, 8, 64), (131, 61, 7, 1, 128),
                                               (64, 63, 16, 2, 256), (129, 257, 6, 3, 96), (200, 0, 32, 8, 64)])
def test_chunk(backend, kv, act, T, start, nq, nkv, hd):
    rng = np.random.default_rng(T * 7 + start)
    c = Cache(backend, rng, kv, 1, start + T + 5, nkv, hd, [start + T])
    q = rng.standard_normal((T, nq, hd)).astype(np_act(act))
    out = backend.launch_attention_kv(backend.upload(q), c.bufs[0], c.bufs[1], c.kv, T, nq, nkv, hd, c.slots, pos_start=start,
                                      act_dtype=ACT[act])
    got = backend.read(out, np_act(act), q.shape)
    k, v = c.values(0, start + T)
    want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)
    close(got, want, mag, q, k, start + T, hd ** -0.5, act)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_later_tokens_that_are_not_finite_do_not_reach_earlier_rows(backend, act, bad):
    """f16 cache, one chunk: token 40's value row holds one non-finite entry, token 50's key is not finite at all."""
    T, nq, nkv, hd = 90, 4, 2, 64
    rng = np.random.default_rng(3)
    c = Cache(backend, rng, "f16", 1, T, nkv, hd, [T])
    raw = [backend.read(b, np.float16, (T, nkv * hd)).copy() for b in c.bufs]
    raw[1][40, 3] = bad
    raw[0][50, hd:] = bad
    for b, r in zip(c.bufs, raw):
        backend.copy_h2d(b, r)
    q = rng.standard_normal((T, nq, hd)).astype(np_act(act))
    got = backend.read(backend.launch_attention_kv(backend.upload(q), c.bufs[0], c.bufs[1], c.kv, T, nq, nkv, hd, T, act_dtype=ACT[act]),
                       np_act(act), q.shape)
    k, v = (r.astype(np.float64).reshape(T, nkv, hd) for r in raw)
    clean = v.copy()
    clean[40, 0, 3] = 0
    want, mag = ref.attention(q[:50], k[:50], clean[:50], list(range(50)), hd ** -0.5)
    for rows, heads, dims in ((slice(0, 40), slice(0, 4), slice(0, hd)), (slice(40, 50), slice(0, 2), slice(4, hd)),
                              (slice(40, 50), slice(2, 4), slice(0, hd))):
        g, w, m = (x[rows, heads, dims] for x in (got, want, mag))
        operand = 0.0 if act == "f32" else 3 * ref.U16
        bound = ref.attention_bound(q[:50], k[:50], mag, T, hd ** -0.5, operand)[rows, heads, dims] + \
            (ref.U16 * np.abs(w) + 2.0 ** -25 if act == "f16" else 0)
        assert np.all(np.abs(g.astype(np.float64) - w) <= bound)
    sees = got[40:50, :2, 3].astype(np.float64)
    assert np.all(np.isnan(sees)) if np.isnan(bad) else np.all(sees == bad)
    assert np.all(np.isnan(got[50:, 2:]))  # a key that is not finite makes its row's softmax so


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("spread", [1e-6, 3e4])
def test_magnitudes(backend, kv, spread):
    """Values at the ends of f16's range: scores stay moderate (the scale takes the keys' size back)."""
    rng = np.random.default_rng(9)
    c = Cache(backend, rng, kv, 1, 100, 2, 64, [100], spread=min(spread, 8e3))
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    scale = float(np.float32(0.125 / min(spread, 8e3)))
    got = run_decode(backend, c, q, [99, 50], None, "f32", scale=scale)
    k, v = c.values(0, 100)
    want, mag = ref.attention(q, k, v, [99, 50], scale)
    close(got, want, mag, q, k, 100, scale, "f32")


def test_large_queries_and_peaked_rows(backend):
    rng = np.random.default_rng(11)
    c = Cache(backend, rng, "words", 1, 300, 2, 128, [300])
    q = (rng.standard_normal((2, 8, 128)) * np.array([1e5, 1e-5]).reshape(2, 1, 1)).astype(np.float32)
    got = run_decode(backend, c, q, [299, 299], None, "f32", scale=1e-5)
    k, v = c.values(0, 300)
    want, mag = ref.attention(q, k, v, [299, 299], float(np.float32(1e-5)))
    close(got, want, mag, q, k, 300, 1e-5, "f32")


def test_unaligned_cache_and_odd_row_bytes(backend):
    """Caches at the least alignment the layouts ask for, and token rows that are no multiple of 16 bytes."""
    rng = np.random.default_rng(13)
    for kv, skew in (("q8_0", 2), ("f16", 2), ("words", 4)):
        nq, nkv, hd, n = 6, 3, 96, 77
        c = Cache(backend, rng, kv, 1, n, nkv, hd, [n])
        at = []
        for b in c.bufs:
            raw = backend.read(b, np.uint8, (n * c.bpt,))
            moved = backend.empty(n * c.bpt + 64)
            backend.copy_h2d(moved.data_ptr() + skew, raw)
            backend.sync()
            at.append(moved)
        q = rng.standard_normal((3, nq, hd)).astype(np.float32)
        pos = backend.upload(np.array([n - 1, 0, 40], np.int32))
        out = backend.launch_attention_kv(backend.upload(q), at[0].data_ptr() + skew, at[1].data_ptr() + skew, c.kv, 3, nq, nkv, hd, n, pos=pos)
        k, v = c.values(0, n)
        want, mag = ref.attention(q, k, v, [n - 1, 0, 40], hd ** -0.5)
        close(backend.read(out, np.float32, q.shape), want, mag, q, k, n, hd ** -0.5, "f32")
        out = backend.launch_attention_kv(backend.upload(q), at[0].data_ptr() + skew, at[1].data_ptr() + skew, c.kv, 3, nq, nkv, hd, n, pos_start=n - 3)
        want, mag = ref.attention(q, k, v, [n - 3, n - 2, n - 1], hd ** -0.5)
        close(backend.read(out, np.float32, q.shape), want, mag, q, k, n, hd ** -0.5, "f32")


def test_rows_outside_the_cache_are_zero_and_reported(backend):
    rng = np.random.default_rng(2)
    c = Cache(backend, rng, "q8_0", 2, 16, 2, 64, [16, 16])
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    out = backend.launch_attention_kv(backend.upload(q), c.bufs[0], c.bufs[1], c.kv, 5, 4, 2, 64, 16,
                                      pos=backend.upload(np.array([3, 16, -2, 5, 5], np.int32)),
                                      seq=backend.upload(np.array([0, 0, 1, 2, 1], np.int32)), n_seqs=2)
    with pytest.raises(BackendError, match="attention_kv"):
        backend.sync()
    got = backend.read(out, np.float32, q.shape)
    assert not got[1:4].any()
    for i, s, p in ((0, 0, 3), (4, 1, 5)):
        k, v = c.values(s, p + 1)
        want, mag = ref.attention(q[i:i + 1], k, v, [p], 0.125)
        close(got[i:i + 1], want, mag, q[i:i + 1], k, p + 1, 0.125, "f32")
    backend.sync()


def test_refusals(backend):
    be = backend
    buf, big = be.empty(1 << 16), be.empty(1 << 16)
    ok = dict(q=buf, k_cache=big, v_cache=big, kv_dtype=AGN_Q8_0, T=2, n_q_heads=4, n_kv_heads=2, head_dim=64, max_seq_len=16, out=be.empty(4096))

    def refused(status=agn._abi.AGN_EINVAL, **kw):
        with pytest.raises(BackendError) as e:
            be.launch_attention_kv(**{**ok, **kw})
        assert e.value.status == status, e.value

    refused(agn._abi.AGN_EUNSUPPORTED_DTYPE, kv_dtype=AGN_Q4_K)
    refused(n_kv_heads=3)
    refused(head_dim=48)
    refused(head_dim=288)
    refused(T=-1, out=buf)
    refused(max_seq_len=0)
    refused(n_seqs=0)
    refused(scale=0.0)
    refused(scale=float("nan"))
    refused(scale=float("inf"))
    refused(seq=buf)                    # sequences without positions
    refused(pos_start=15)               # 15 + 2 > 16
    refused(pos_start=-1)
    refused(q=None)
    refused(k_cache=None)
    refused(q=ok["out"])                # in place
    refused(q=buf.data_ptr() + 4)
    refused(k_cache=big.data_ptr() + 1)
    refused(kv_dtype=AGN_KV_Q8_0_WORDS, k_cache=big.data_ptr() + 2)
    with pytest.raises(ValueError):
        be.launch_attention_kv(**ok, act_dtype=AGN_Q8_0)
    assert be.launch_attention_kv(**{**ok, "T": 0, "q": None}) is ok["out"]  # nothing to do
    be.sync()


def test_short_workspace_is_refused(backend):
    need = backend.attention_kv_workspace_bytes(1, 8, 2, 128, 4096, True)
    if need:
        buf = backend.empty(1 << 20)
        with pytest.raises(BackendError):
            backend.launch_attention_kv(buf, buf, buf, AGN_Q8_0, 1, 8, 2, 128, 4096, pos=buf, out=backend.empty(4096),
                                        workspace=backend.empty(need - 16))


@pytest.mark.parametrize("form", ["decode", "chunk"])
def test_recorded_chain_write_then_attend(backend, form):
    """A decode step and a prompt piece recorded with the cache write in front of them, replayed with new inputs; a guard
    behind the output stays as it was."""
    be, nq, nkv, hd, slots = backend, 8, 2, 128, 320
    T, start = (1, 255) if form == "decode" else (40, 100)
    rng = np.random.default_rng(21)
    c = Cache(be, rng, "words", 1, slots, nkv, hd, [300])
    dq, dk, dv = be.empty(4 * T * nq * hd), be.empty(4 * T * nkv * hd), be.empty(4 * T * nkv * hd)
    out = be.empty(4 * T * nq * hd + 256)
    pos = be.upload(np.arange(start, start + T, dtype=np.int32)) if form == "decode" else None
    need = be.attention_kv_workspace_bytes(T, nq, nkv, hd, slots, form == "decode")
    ws = be.empty(max(need, 16))

    def chain():
        be.kv_write(c.kv, dk, dv, c.bufs[0], c.bufs[1], T, nkv * hd, pos, slots, pos_start=start)
        be.launch_attention_kv(dq, c.bufs[0], c.bufs[1], c.kv, T, nq, nkv, hd, slots, pos=pos, pos_start=start, out=out, workspace=ws)

    chain()
    be.sync()
    be.graph_begin()
    chain()
    g = be.graph_end()
    be.copy_h2d(out, np.full(4 * T * nq * hd + 256, 0xA5, np.uint8))
    for _ in range(2):
        q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (nq, nkv, nkv))
        for b, x in ((dq, q), (dk, k), (dv, v)):
            be.copy_h2d(b, x)
        be.sync()
        be.graph_launch(g)
        got = be.read(out, np.float32, q.shape)
        kk, vv = c.values(0, start + T)
        want, mag = ref.attention(q, kk, vv, [start + t for t in range(T)], hd ** -0.5)
        close(got, want, mag, q, kk, start + T, hd ** -0.5, "f32")
    assert np.all(be.read(out.data_ptr() + 4 * T * nq * hd, np.uint8, (256,)) == 0xA5)
    be.graph_destroy(g)


def test_same_bits_every_time_and_on_another_stream(backend):
    import torch
    rng = np.random.default_rng(31)
    c = Cache(backend, rng, "q8_0", 3, 700, 4, 128, [700, 300, 45])
    q = rng.standard_normal((3, 28, 128)).astype(np.float32)
    first = run_decode(backend, c, q, [699, 299, 44], [0, 1, 2], "f32")
    assert np.array_equal(first, run_decode(backend, c, q, [699, 299, 44], [0, 1, 2], "f32"))
    s = torch.cuda.Stream()
    try:
        backend.set_stream(s.cuda_stream)
        assert np.array_equal(first, run_decode(backend, c, q, [699, 299, 44], [0, 1, 2], "f32"))
    finally:
        backend.set_stream(None)


def test_cache_beyond_32_bit_offsets(backend):
    """The last sequence of a cache of more than 4 GiB."""
    nkv, hd, slots = 8, 128, 8192
    bpt = backend.kv_bytes_per_token(AGN_F16, nkv * hd)
    n = (1 << 32) // (slots * bpt) + 2
    rng = np.random.default_rng(17)
    bufs = [backend.empty(n * slots * bpt) for _ in range(2)]
    k, v = (rng.standard_normal((50, nkv, hd)).astype(np.float16) for _ in range(2))
    for b, x in zip(bufs, (k, v)):
        backend.copy_h2d(b.data_ptr() + (n - 1) * slots * bpt, x)
    q = rng.standard_normal((1, 32, hd)).astype(np.float32)
    out = backend.launch_attention_kv(backend.upload(q), bufs[0], bufs[1], AGN_F16, 1, 32, nkv, hd, slots,
                                      pos=backend.upload(np.array([49], np.int32)), seq=backend.upload(np.array([n - 1], np.int32)), n_seqs=n)
    got = backend.read(out, np.float32, q.shape)
    want, mag = ref.attention(q, k.astype(np.float64), v.astype(np.float64), [49], hd ** -0.5)
    close(got, want, mag, q, k.astype(np.float64), 50, hd ** -0.5, "f32")
    for b in bufs:
        b.free()
