"""A decode step of a batch: one cache write for the tokens of all sequences (positions s * max_seq_len + p of a cache of n_seqs * max_seq_len slots), then
attention over the sequences."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_KV_Q8_0_WORDS, AGN_Q8_0, BackendError
from tests import mixers_norms as norms
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [AGN_F16, AGN_Q8_0, AGN_KV_Q8_0_WORDS])
def test_steps_of_a_batch_recorded_once(backend, kv):
    """Sequences of different lengths grow by a token each at every replay; one of them is finished and writes and sees nothing."""
    be, n, nq, nkv, hd, slots = backend, 5, 8, 2, 64, 40
    rng, width = np.random.default_rng(kv), 2 * 64
    bpt = be.kv_bytes_per_token(kv, width)
    bufs = [be.upload(np.zeros(n * slots * bpt, np.uint8)) for _ in range(2)]
    lens = np.array([0, 3, 17, 30, 8])
    first = [rng.standard_normal((slots, width)).astype(np.float32) for _ in range(2)]
    for s in range(n):
        if lens[s]:
            be.kv_write(kv, be.upload(first[0]), be.upload(first[1]), *(b.data_ptr() + s * slots * bpt for b in bufs), int(lens[s]), width, None, slots)
    be.sync()
    dq, dk, dv = be.empty(4 * n * nq * hd), be.empty(4 * n * width), be.empty(4 * n * width)
    pos, flat, out = be.empty(4 * n), be.empty(4 * n), be.empty(4 * n * nq * hd)
    seq = be.upload(np.arange(n, dtype=np.int32))
    ws = be.empty(max(16, be.attention_kv_workspace_bytes(n, nq, nkv, hd, slots, True)))

    def chain():
        be.kv_write(kv, dk, dv, bufs[0], bufs[1], n, width, flat, n * slots)
        be.launch_attention_kv(dq, bufs[0], bufs[1], kv, n, nq, nkv, hd, slots, pos=pos, seq=seq, n_seqs=n, out=out, workspace=ws)

    g, done = None, 4
    for step in range(4):
        p = lens + step
        p[done] = -1 if step > 1 else p[done]
        q, k, v = (rng.standard_normal((n, h, hd)).astype(np.float32) for h in (nq, nkv, nkv))
        for b, x in ((dq, q), (dk, k), (dv, v), (pos, p.astype(np.int32)), (flat, np.where(p >= 0, np.arange(n) * slots + p, done * slots + slots - 1).astype(np.int32))):
            be.copy_h2d(b, x)
        be.sync()
        if g is None:
            chain()
            be.sync()
            be.graph_begin()
            chain()
            g = be.graph_end()
        else:
            be.graph_launch(g)
        got = be.read(out, np.float32, q.shape)
        be.sync()
        for s in range(n):
            if p[s] < 0:
                assert not got[s].any()
                continue
            ck, cv = (ref.cache_values(kv, be.read(b, np.uint8, (n, slots, bpt))[s, :p[s] + 1], width).reshape(p[s] + 1, nkv, hd) for b in bufs)
            assert np.abs(ck[-1] - k[s]).max() < 0.05  # the token's own key stands at its place
            want, size = norms.attention(q[s:s + 1], ck, cv, [p[s]], hd ** -0.5)
            norms.hold(got[s:s + 1], want, size, q[s:s + 1], ck, p[s] + 1, hd ** -0.5, "f32")
    be.graph_destroy(g)


def test_a_write_behind_the_last_sequence_is_reported(backend):
    be, n, slots, width = backend, 3, 8, 64
    bpt = be.kv_bytes_per_token(AGN_Q8_0, width)
    bufs = [be.upload(np.zeros((n * slots + 1) * bpt, np.uint8)) for _ in range(2)]
    x = be.upload(np.ones((2, width), np.float32))
    be.kv_write(AGN_Q8_0, x, x, bufs[0], bufs[1], 2, width, be.upload(np.array([n * slots - 1, n * slots], np.int32)), n * slots)
    with pytest.raises(BackendError):
        be.sync()
    raw = be.read(bufs[0], np.uint8, (n * slots + 1, bpt))
    assert raw[n * slots - 1].any() and not raw[n * slots].any() and not raw[:n * slots - 1].any()
