"""The token mixers where their forms change or their inputs are unusual: many single rows, wide caches, every head size, slots shared out over CTAs, values that are
not finite, write strengths and decays outside the usual range, recorded calls, short waits."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, AGN_F32, AGN_Q8_0, BackendError, CudaBackend
from tests import ref_mixers as ref
from tests.test_gpu_attention_kv import ACT, Cache, close, np_act, run_decode
from tests.test_gpu_delta_rule import check, expected, inputs, launch

pytestmark = pytest.mark.gpu


def run_chunk(be, c, q, start, act):
    T, nq, hd = q.shape
    out = be.launch_attention_kv(be.upload(q), c.bufs[0], c.bufs[1], c.kv, T, nq, c.nkv, hd, c.slots, pos_start=start, act_dtype=ACT[act])
    return be.read(out, np_act(act), q.shape)


@pytest.mark.parametrize("T", [511, 512, 513, 700])
def test_more_rows_than_are_shared_out(backend, T):
    rng = np.random.default_rng(T)
    c = Cache(backend, rng, "q8_0", 2, 70, 2, 64, [70, 33])
    q = rng.standard_normal((T, 4, 64)).astype(np.float32)
    seq = rng.integers(0, 2, T)
    pos = np.where(rng.random(T) < 0.1, -1, (rng.random(T) * np.where(seq == 0, 70, 33)).astype(int))
    got = run_decode(backend, c, q, pos, seq, "f32")
    backend.sync()
    for s in range(2):
        k, v = c.values(s, [70, 33][s])
        rows = np.flatnonzero(seq == s)
        want, mag = ref.attention(q[rows], k, v, pos[rows], 0.125)
        close(got[rows], want, mag, q[rows], k, 70, 0.125, "f32")
    assert not got[pos < 0].any()


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("nq,nkv,hd", [(12, 12, 64), (16, 16, 128), (9, 9, 32), (10, 5, 128), (16, 8, 256), (7, 1, 128), (20, 1, 64), (4, 4, 32), (6, 6, 160), (4, 2, 192),
                                       (3, 1, 224)])
def test_head_counts_and_sizes(backend, kv, nq, nkv, hd):
    rng = np.random.default_rng(nq + hd)
    lens = [90, 17]
    c = Cache(backend, rng, kv, 2, 101, nkv, hd, lens)
    q = rng.standard_normal((3, nq, hd)).astype(np.float32)
    got = run_decode(backend, c, q, [89, 16, 40], [0, 1, 0], "f32")
    for i, (s, p) in enumerate(((0, 89), (1, 16), (0, 40))):
        k, v = c.values(s, lens[s])
        want, mag = ref.attention(q[i:i + 1], k, v, [p], hd ** -0.5)
        close(got[i:i + 1], want, mag, q[i:i + 1], k, 90, hd ** -0.5, "f32")
    q = rng.standard_normal((20, nq, hd)).astype(np.float32)
    k, v = c.values(0, 90)
    want, mag = ref.attention(q, k, v, list(range(70, 90)), hd ** -0.5)
    close(run_chunk(backend, c, q, 70, "f32"), want, mag, q, k, 90, hd ** -0.5, "f32")


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 1, 64), (4, 2, 96), (4, 2, 256)])
@pytest.mark.parametrize("T,start", [(16, 4000), (37, 4091)])
def test_piece_behind_a_long_cache(backend, kv, act, nq, nkv, hd, T, start):
    """Few rows over many slots: the slots are shared out over CTAs and the shares joined."""
    rng = np.random.default_rng(T + hd)
    c = Cache(backend, rng, kv, 1, start + T + 3, nkv, hd, [start + T])
    q = (2 * rng.standard_normal((T, nq, hd))).astype(np_act(act))
    got = run_chunk(backend, c, q, start, act)
    assert backend.last_kernel == "attention_kv_join"
    k, v = c.values(0, start + T)
    want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)
    close(got, want, mag, q, k, start + T, hd ** -0.5, act)
    assert np.array_equal(got, run_chunk(backend, c, q, start, act))


@pytest.mark.parametrize("act,hd", [("f32", 64), ("f16", 64), ("f16", 128), ("f32", 256)])
def test_values_that_are_not_finite_behind_a_long_cache(backend, act, hd):
    T, start, nq, nkv = 24, 3000, 4, 2
    rng = np.random.default_rng(hd)
    n = start + T
    c = Cache(backend, rng, "f16", 1, n, nkv, hd, [n])
    raw = backend.read(c.bufs[1], np.float16, (n, nkv * hd)).copy()
    for slot, dim, x in ((start + 5, 3, np.inf), (start + 9, 3, -np.inf), (100, hd + 7, -np.inf), (start + 20, 11, np.nan)):
        raw[slot, dim] = x
    backend.copy_h2d(c.bufs[1], raw)
    backend.sync()
    q = rng.standard_normal((T, nq, hd)).astype(np_act(act))
    got = run_chunk(backend, c, q, start, act).astype(np.float64)
    t = np.arange(T)
    a = got[:, :2, 3]  # heads 0, 1 of KV head 0
    assert np.all(np.isfinite(a[t < 5])) and np.all(a[(t >= 5) & (t < 9)] == np.inf) and np.all(np.isnan(a[t >= 9]))
    assert np.all(np.isfinite(got[t < 20, :2, 11])) and np.all(np.isnan(got[t >= 20, :2, 11]))
    assert np.all(got[:, 2:, 7] == -np.inf)
    rest = got.copy()
    rest[:, :2, 3] = rest[:, :2, 11] = rest[:, 2:, 7] = 0
    assert np.all(np.isfinite(rest))


def test_workspace_of_a_prompt_is_checked(backend):
    need = backend.attention_kv_workspace_bytes(40, 8, 2, 128, 5000, False)
    buf, big = backend.empty(1 << 20), backend.empty(5000 * backend.kv_bytes_per_token(AGN_Q8_0, 256))
    assert need > 0
    with pytest.raises(BackendError):
        backend.launch_attention_kv(buf, big, big, AGN_Q8_0, 40, 8, 2, 128, 5000, pos_start=4960, act_dtype=AGN_F16, out=backend.empty(1 << 20), workspace=backend.empty(64))
    need = backend.gated_delta_rule_workspace_bytes(200, 1, 1, 2, 64, 64)
    with pytest.raises(BackendError):
        backend.launch_gated_delta_rule(buf, buf, buf, buf, buf, None, 200, 1, 1, 2, 64, 64, out=backend.empty(1 << 20), workspace=backend.empty(need - 16))
    backend.sync()


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_prompts_recorded_cold_and_replayed(act):
    """The first call of a process's context is a recorded one; two graphs with a workspace each, replayed in turn."""
    be = CudaBackend(0)
    try:
        rng = np.random.default_rng(2)
        T, start, nq, nkv, hd = 40, 900, 8, 2, 64
        c = Cache(be, rng, "words", 1, start + T, nkv, hd, [start + T])
        qs = [rng.standard_normal((T, nq, hd)).astype(np_act(act)) for _ in range(2)]
        need = max(16, be.attention_kv_workspace_bytes(T, nq, nkv, hd, c.slots, False))
        sets = [(be.upload(q), be.empty(q.nbytes), be.empty(need)) for q in qs]
        graphs = []
        for q, o, ws in sets:
            be.graph_begin()
            be.launch_attention_kv(q, c.bufs[0], c.bufs[1], c.kv, T, nq, nkv, hd, c.slots, pos_start=start, act_dtype=ACT[act], out=o, workspace=ws)
            graphs.append(be.graph_end())
        for g in graphs + graphs[::-1]:
            be.graph_launch(g)
        be.sync()
        k, v = c.values(0, start + T)
        for q, (_, o, _) in zip(qs, sets):
            want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)
            close(be.read(o, np_act(act), q.shape), want, mag, q, k, start + T, hd ** -0.5, act)
        for g in graphs:
            be.graph_destroy(g)
    finally:
        be.close()


def test_two_streams_at_once():
    """Two contexts, a stream and a workspace each, at work on the same cache and on the same inputs of the delta rule."""
    a, b = CudaBackend(0), CudaBackend(0)
    try:
        rng = np.random.default_rng(7)
        c = Cache(a, rng, "q8_0", 1, 2100, 2, 128, [2100])
        q = rng.standard_normal((60, 8, 128)).astype(np.float16)
        dq = a.upload(q)
        x = inputs(rng, [300], 2, 4, 128, 128)
        d = {n: a.upload(v) for n, v in x.items()}
        a.sync()
        outs = []
        for be in (a, b):
            o, ws = be.empty(q.nbytes), be.empty(be.attention_kv_workspace_bytes(60, 8, 2, 128, 2100, False))
            do, ds = be.empty(x["v"].nbytes), be.empty(x["S"].nbytes)
            dws = be.empty(be.gated_delta_rule_workspace_bytes(300, 1, 2, 4, 128, 128))
            outs.append((be, o, ws, do, ds, dws))
        for _ in range(5):
            for be, o, ws, do, ds, dws in outs:
                be.launch_attention_kv(dq, c.bufs[0], c.bufs[1], c.kv, 60, 8, 2, 128, 2100, pos_start=2040, act_dtype=AGN_F16, out=o, workspace=ws)
                be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], d["S"], 300, 1, 2, 4, 128, 128, state_out=ds, out=do, workspace=dws)
        got = [(be.read(o, np.float16, q.shape), be.read(do, np.float32, x["v"].shape), be.read(ds, np.float32, x["S"].shape)) for be, o, _, do, ds, _ in outs]
        for u, w in zip(*got):
            assert np.array_equal(u, w)
        want, wS = expected(x, [300], 128 ** -0.5, 1e-6)
        check(got[0][1], want, x, "out")
        check(got[0][2], wS, x, "state")
    finally:
        a.close()
        b.close()


# ------------------------------------------------------------------------------------------------------- delta rule

@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e30])
@pytest.mark.parametrize("T", [7, 150])
def test_delta_magnitudes(backend, size, T):
    x = inputs(np.random.default_rng(3), [T], 1, 2, 64, 64)
    x["v"] *= np.float32(size)
    x["S"] *= np.float32(size)
    out, S = launch(backend, x, [T], 1, 2, 64, 64)
    want, wS = expected(x, [T], 0.125, 1e-6)
    check(out, want, x, "out")
    check(S, wS, x, "state")


@pytest.mark.parametrize("T", [9, 100])
@pytest.mark.parametrize("what", ["strong", "negative", "growing", "long keys"])
def test_delta_outside_the_bounds_of_the_chunked_form(backend, what, T):
    """Write strengths above 2 or below 0, decays above 1, keys longer than 1: computed row by row."""
    rng = np.random.default_rng(5)
    x = inputs(rng, [T], 1, 2, 64, 64)
    eps = 1e-6
    if what == "strong":
        x["beta"][T // 2] = 2.5
    elif what == "negative":
        x["beta"][T // 2] = -0.3
    elif what == "growing":
        x["g"][::7] = 0.05
    else:
        eps = -1.0
        for n in "qk":
            x[n] /= np.sqrt((x[n] ** 2).sum(-1, keepdims=True))
        x["k"][T // 3] *= 1.3
        x["q"] *= 3
        x["beta"] *= 0.9
    out, S = launch(backend, x, [T], 1, 2, 64, 64, l2norm_eps=eps)
    want, wS = expected(x, [T], 0.125, eps)
    check(out, want, x, "out")
    check(S, wS, x, "state")


@pytest.mark.parametrize("T", [9, 200])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_delta_values_that_are_not_finite(backend, bad, T):
    """A value of one token and column: tokens before it and other columns stay as they are."""
    x = inputs(np.random.default_rng(6), [T], 1, 2, 64, 96)
    at = T * 2 // 3
    clean, _ = expected(x, [T], 0.125, 1e-6)
    x["v"][at, 1, 40] = bad
    out, S = launch(backend, x, [T], 1, 2, 64, 96)
    assert np.all(np.isfinite(out[:at])) and not np.any(np.isfinite(out[at:, 1, 40])) and not np.any(np.isfinite(S[0, 1, :, 40]))
    x["v"][at, 1, 40] = 0
    out[at:, 1, 40] = clean[at:, 1, 40]
    check(out, clean, x, "out")


def test_delta_many_sequences_of_every_length(backend):
    lens = [int(n) for n in np.random.default_rng(1).integers(0, 140, 40)]
    x = inputs(np.random.default_rng(2), lens, 1, 2, 64, 32)
    out, S = launch(backend, x, lens, 1, 2, 64, 32)
    want, wS = expected(x, lens, 0.125, 1e-6)
    check(out, want, x, "out")
    check(S, wS, x, "state")


def test_offsets_out_of_order_stay_inside(backend):
    """Chunked form: reported, and nothing outside out and state is written."""
    be, T = backend, 400
    x = inputs(np.random.default_rng(1), [T], 1, 1, 64, 32)
    d = {n: be.upload(a) for n, a in x.items()}
    S = be.upload(np.zeros((3, 1, 64, 32), np.float32))
    for cu in ([0, 300, 100, 400], [-50, 200, 5000, 390], [399, 0, 0, 0]):
        out = be.upload(np.full(T * 32 + 64, 3.0, np.float32))
        so = be.upload(np.full(3 * 64 * 32 + 64, 3.0, np.float32))
        be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], S, T, 3, 1, 1, 64, 32, cu_seqlens=be.upload(np.array(cu, np.int32)), out=out, state_out=so)
        with pytest.raises(BackendError, match="gated_delta_rule"):
            be.sync()
        assert np.all(be.read(out, np.float32, (T * 32 + 64,))[T * 32:] == 3.0)
        assert np.all(be.read(so, np.float32, (3 * 64 * 32 + 64,))[3 * 64 * 32:] == 3.0)


# ------------------------------------------------------------------------------------------------------- together

def test_layer_of_each_kind(backend):
    """A hybrid model's two layers on one prompt, then one token: qk norm -> rope -> cache write -> attention; delta rule -> gated norm.  The token's attention row is
    checked against the cache as kv_read gives it."""
    be, nq, nkv, hd, slots = backend, 8, 2, 128, 256
    rng = np.random.default_rng(33)
    dk, dv = (be.upload(np.zeros(slots * be.kv_bytes_per_token(AGN_Q8_0, nkv * hd), np.uint8)) for _ in range(2))
    w = [be.upload((1 + 0.02 * rng.standard_normal(hd)).astype(np.float32)) for _ in range(2)]
    state = be.upload(np.zeros((4, 128, 128), np.float32))
    gates = be.upload((1 + 0.02 * rng.standard_normal(128)).astype(np.float32))
    at, S = 0, np.zeros((4, 128, 128))
    for T in (130, 1):
        q, k, v = (rng.standard_normal((T, n * hd)).astype(np.float32) for n in (nq, nkv, nkv))
        dq, kk, vv = be.upload(q), be.upload(k), be.upload(v)
        be.launch_qk_norm_rope_kv_write(dq, kk, vv, w[0], w[1], T, nq, nkv, hd, 1e-6, hd, None, 1e6, AGN_Q8_0, dk, dv, slots, pos_start=at)
        out = be.read(be.launch_attention_kv(dq, dk, dv, AGN_Q8_0, T, nq, nkv, hd, slots, pos_start=at, act_dtype=AGN_F32), np.float32, (T, nq, hd))
        rq = be.read(dq, np.float32, (T, nq, hd))
        ck, cv = (be.read(b, np.float32, (at + T, nkv, hd)).astype(np.float64) for b in be.kv_read(AGN_Q8_0, dk, dv, at + T, nkv * hd))
        want, mag = ref.attention(rq, ck, cv, [at + t for t in range(T)], hd ** -0.5)
        close(out, want, mag, rq, ck, at + T, hd ** -0.5, "f32")
        x = inputs(rng, [T], 2, 4, 128, 128)
        d = {n: be.upload(a) for n, a in x.items()}
        o, _ = be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], state, T, 1, 2, 4, 128, 128, state_out=state)
        z = rng.standard_normal((T * 4, 128)).astype(np.float32)
        y = be.read(be.launch_rms_norm_silu_gate(o, be.upload(z), gates, T * 4, 128, 1e-6), np.float32, (T * 4, 128))
        wo, S = ref.delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], S, 128 ** -0.5, 1e-6)
        got = be.read(o, np.float32, (T, 4, 128))
        check(got, wo, x, "out")
        wy = ref.gated_norm(got.reshape(-1, 128), z, be.read(gates, np.float32, (128,)), 1e-6)
        assert np.all(np.abs(y - wy) <= 1e-5 * np.abs(wy).max(-1, keepdims=True))
        at += T


@pytest.mark.parametrize("T,nq,nkv,hd,slots", [(277, 16, 2, 64, 600), (250, 7, 1, 128, 900), (38, 4, 1, 64, 5000), (64, 4, 1, 256, 3000)])
def test_one_workspace_for_rows_that_end_anywhere(backend, T, nq, nkv, hd, slots):
    rng = np.random.default_rng(T)
    c = Cache(backend, rng, "q8_0", 1, slots, nkv, hd, [slots])
    ws = backend.empty(max(16, backend.attention_kv_workspace_bytes(T, nq, nkv, hd, slots, False)))
    k, v = c.values(0, slots)
    for act in ("f32", "f16"):
        q = rng.standard_normal((T, nq, hd)).astype(np_act(act))
        dq, out = backend.upload(q), backend.empty(q.nbytes)
        for start in list(range(0, slots - T, max(64, (slots - T) // 16 // 64 * 64))) + [slots - T]:
            backend.launch_attention_kv(dq, c.bufs[0], c.bufs[1], c.kv, T, nq, nkv, hd, slots, pos_start=start, act_dtype=ACT[act], out=out, workspace=ws)
        want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)
        close(backend.read(out, np_act(act), q.shape), want, mag, q, k, slots, hd ** -0.5, act)


@pytest.mark.parametrize("form", ["f32", "f16", "f32 rows of their own", "f16 rows of their own"])
def test_keys_of_nan_in_the_last_share_alone(backend, form):
    """Every score that a row has in one of its shares is NaN: so is its result, in that head alone."""
    rng = np.random.default_rng(8)
    act = form[:3]
    T, start, nq, nkv, hd = 40, 2048, 4, 2, 64
    k, v = (rng.standard_normal((start + T, nkv, hd)).astype(np.float16) for _ in range(2))
    k[start:, 0] = np.nan
    q = rng.standard_normal((T, nq, hd)).astype(np_act(act))
    bufs = [backend.upload(x) for x in (q, k, v)]
    kw = dict(pos=backend.upload(np.arange(start, start + T, dtype=np.int32))) if "own" in form else dict(pos_start=start)
    out = backend.launch_attention_kv(bufs[0], bufs[1], bufs[2], AGN_F16, T, nq, nkv, hd, start + T, act_dtype=ACT[act], **kw)
    got = backend.read(out, np_act(act), q.shape)
    assert np.isnan(got[:, :2]).all()
    k, v = k.astype(np.float64), v.astype(np.float64)
    want, mag = ref.attention(q[:, 2:], k[:, 1:], v[:, 1:], [start + t for t in range(T)], hd ** -0.5)
    close(got[:, 2:], want, mag, q[:, 2:], k[:, 1:], start + T, hd ** -0.5, act)


@pytest.mark.parametrize("kv,low,high", [("q8_0", -4, 2), ("words", -6, 6), ("words", 36, 37), ("words", -37, -36), ("words", 0, 1), ("f16", -4, 3)])
@pytest.mark.parametrize("hd", [64, 160])
def test_values_of_very_different_sizes(backend, kv, low, high, hd):
    """V's magnitude changes from slot to slot by up to twelve orders, at both ends of f32's range too; some rows see only small ones."""
    rng = np.random.default_rng(hd + high)
    T, start, nq, nkv = 50, 150, 6, 2
    slots = start + T
    c = Cache(backend, rng, kv, 1, slots, nkv, hd, [slots])
    v = rng.standard_normal((slots, nkv * hd)) * 10.0 ** rng.uniform(low, high, (slots, 1))
    v[start + 20] *= 10.0 if high > 30 else 1.0
    k = rng.standard_normal((slots, nkv * hd)).astype(np.float32)
    backend.kv_write(c.kv, backend.upload(k), backend.upload(v.astype(np.float32)), c.bufs[0], c.bufs[1], slots, nkv * hd, None, slots)
    q = rng.standard_normal((T, nq, hd)).astype(np.float32)
    k, v = c.values(0, slots)
    want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)
    # a row's error is counted against its own weights' sum of |v|: what is small beside a value that the row does not see stays exact
    close(run_chunk(backend, c, q, start, "f32"), want, mag, q, k, slots, hd ** -0.5, "f32")


@pytest.mark.parametrize("kv", ["f16", "q8_0", "words"])
def test_small_weights_beside_a_large_one_on_a_value_of_zero(backend, kv):
    """One slot has nearly all the weight and a V of exactly 0.  The other slots' weights are exact to 2^-30 of it (half of the lower f16 part's smallest step, 2^-25, over
    the 2^6 that weights are brought up by, for scales of half the largest at least): with n of them the row is off by at most n 2^-30 max |v| beside the usual bound."""
    rng = np.random.default_rng(6)
    T, start, nq, nkv, hd = 40, 260, 4, 2, 64
    slots = start + T
    c = Cache(backend, rng, kv, 1, slots, nkv, hd, [slots])
    k, v = (rng.standard_normal((slots, nkv * hd)).astype(np.float32) for _ in range(2))
    v[100] = 0.0
    k[100] = 1.0
    q = (0.2 * rng.standard_normal((T, nq, hd)) + np.linspace(0.5, 4.0, T)[:, None, None]).astype(np.float32)
    backend.kv_write(c.kv, backend.upload(k), backend.upload(v), c.bufs[0], c.bufs[1], slots, nkv * hd, None, slots)
    got = run_chunk(backend, c, q, start, "f32").astype(np.float64)
    k, v = c.values(0, slots)
    want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)
    bound = ref.attention_bound(q, k, mag, slots, hd ** -0.5) + slots * 2.0 ** -30 * np.abs(v).max()
    assert np.all(np.abs(got - want) <= bound)
