"""agn_gated_delta_rule_f32 and agn_rms_norm_silu_gate_* against 64-bit statements."""
import numpy as np
import pytest

import agention_infer_b200 as agn
from agention_infer_b200 import AGN_BF16, AGN_F16, AGN_Q8_0, BackendError
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu

# Both forms hold everything in f32 (24 bits; the chunked form multiplies operands of at least 21 bits).  A write's factor
# I - beta k k^T has norm at most 1 and the decay at most 1, so an error made at one token is not enlarged later: with rounding errors
# of either sign the result is off by a few times 2^-21 of the size of what it is summed from (states and values), and 1e-5 of that
# size, the bar of the other float ops, leaves 20 times of it for the growth over the tokens that a state remembers.
TOL = 1e-5


def inputs(rng, lens, nk, nv, dk, dv, decay=1.0, pad=0):
    T = sum(lens) + pad
    r = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    g = (-decay * np.log1p(np.exp(rng.standard_normal((T, nv)) - 1)) * rng.uniform(0.02, 0.5, nv)).astype(np.float32)
    beta = (1 / (1 + np.exp(-rng.standard_normal((T, nv))))).astype(np.float32)
    return dict(q=r(T, nk, dk), k=r(T, nk, dk), v=r(T, nv, dv), g=g, beta=beta, S=(0.3 * r(len(lens), nv, dk, dv)).astype(np.float32))


def expected(x, lens, scale, eps):
    out, S, at = np.zeros(x["v"].shape), np.zeros(x["S"].shape), 0
    for s, n in enumerate(lens):
        rows = slice(at, at + n)
        out[rows], S[s] = ref.delta_rule(x["q"][rows], x["k"][rows], x["v"][rows], x["g"][rows], x["beta"][rows], x["S"][s], scale, eps)
        at += n
    return out, S


def check(got, want, x, what):
    size = max(np.abs(x["S"]).max(initial=0.0), np.abs(x["v"]).max(initial=0.0), np.abs(want).max(initial=0.0), 1e-30)
    err = np.abs(got.astype(np.float64) - want).max(initial=0.0)
    assert err <= TOL * size, (what, err, size)


def launch(be, x, lens, nk, nv, dk, dv, cu=True, **kw):
    T = x["q"].shape[0]
    d = {n: be.upload(a) for n, a in x.items()}
    offs = be.upload(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)) if cu else None
    out, S = be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], d["S"], T, len(lens), nk, nv, dk, dv, cu_seqlens=offs, **kw)
    got = be.read(out, np.float32, x["v"].shape), be.read(S, np.float32, x["S"].shape)
    be.sync()
    return got


@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [2, 7], [8, 9, 0, 1], [15, 16, 17], [63], [64], [65], [127, 1, 128, 129, 0, 31], [300], [200, 3, 511]])
@pytest.mark.parametrize("nk,nv,dk,dv", [(2, 4, 128, 128), (2, 2, 64, 64)])
def test_lengths(backend, lens, nk, nv, dk, dv):
    rng = np.random.default_rng(sum(lens) + len(lens))
    x = inputs(rng, lens, nk, nv, dk, dv)
    out, S = launch(backend, x, lens, nk, nv, dk, dv)
    want, wS = expected(x, lens, dk ** -0.5, 1e-6)
    check(out, want, x, "out")
    check(S, wS, x, "state")


@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("nk,nv,dk,dv", [(1, 1, 128, 32), (1, 3, 64, 96), (2, 4, 128, 256), (3, 3, 64, 160)])
def test_head_layouts(backend, T, nk, nv, dk, dv):
    x = inputs(np.random.default_rng(T + dv), [T], nk, nv, dk, dv)
    out, S = launch(backend, x, [T], nk, nv, dk, dv, cu=False, scale=1.0)
    want, wS = expected(x, [T], 1.0, 1e-6)
    check(out, want, x, "out")
    check(S, wS, x, "state")


@pytest.mark.parametrize("T", [5, 150])
@pytest.mark.parametrize("decay", [0.0, 1.0, 60.0, np.inf])
def test_decays(backend, T, decay):
    """No decay at all, a strong one (a chunk's product underflows), a state that is dropped at every token (g = -inf)."""
    x = inputs(np.random.default_rng(4), [T], 2, 4, 128, 64, decay=0.0 if np.isinf(decay) else decay)
    if np.isinf(decay):
        x["g"][:] = 0
        x["g"][::3] = -np.inf
    out, S = launch(backend, x, [T], 2, 4, 128, 64)
    want, wS = expected(x, [T], 128 ** -0.5, 1e-6)
    check(out, want, x, "out")
    check(S, wS, x, "state")


@pytest.mark.parametrize("T", [6, 130])
def test_repeated_keys_and_full_writes(backend, T):
    """The same key at every token with beta = 1: each token replaces what the one before wrote (the triangular system at its worst)."""
    x = inputs(np.random.default_rng(8), [T], 1, 2, 64, 64)
    x["k"][:] = x["k"][:1]
    x["beta"][:] = 1
    x["g"][:] = 0
    out, S = launch(backend, x, [T], 1, 2, 64, 64)
    want, wS = expected(x, [T], 0.125, 1e-6)
    check(out, want, x, "out")
    check(S, wS, x, "state")


@pytest.mark.parametrize("T", [4, 100])
def test_zero_rows_no_norm_and_zero_state(backend, T):
    x = inputs(np.random.default_rng(6), [T], 2, 2, 64, 64)
    for n in "qk":
        x[n] /= np.sqrt((x[n] ** 2).sum(-1, keepdims=True))
    x["k"][T // 2] = 0
    x["q"][1] = 0
    x["S"][:] = 0
    T_, be = T, backend
    d = {n: be.upload(a) for n, a in x.items()}
    out, S = be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], None, T_, 1, 2, 2, 64, 64, l2norm_eps=-1.0)
    want, wS = expected(x, [T], 0.125, -1.0)
    check(be.read(out, np.float32, x["v"].shape), want, x, "out")
    check(be.read(S, np.float32, x["S"].shape), wS, x, "state")
    out, S = be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], None, T_, 1, 2, 2, 64, 64)  # zero rows through the norm
    want, wS = expected(x, [T], 0.125, 1e-6)
    check(be.read(out, np.float32, x["v"].shape), want, x, "out")
    check(be.read(S, np.float32, x["S"].shape), wS, x, "state")


@pytest.mark.parametrize("lens", [[3, 2], [100, 70]])
def test_strided_rows_in_place_state_and_rows_behind(backend, lens):
    """q, k, v as parts of one projection's rows; the state advanced in place; rows behind the last sequence stay."""
    be, nk, nv, dk, dv = backend, 2, 4, 64, 64
    T, pad = sum(lens), 5
    x = inputs(np.random.default_rng(12), lens, nk, nv, dk, dv, pad=pad)
    width = 2 * nk * dk + nv * dv + 12
    row = np.full((T + pad, width), np.nan, np.float32)
    row[:, :nk * dk], row[:, nk * dk:2 * nk * dk] = x["q"].reshape(T + pad, -1), x["k"].reshape(T + pad, -1)
    row[:, 2 * nk * dk:2 * nk * dk + nv * dv] = x["v"].reshape(T + pad, -1)
    d, base = {n: be.upload(x[n]) for n in ("g", "beta", "S")}, be.upload(row)
    out = be.upload(np.full(x["v"].shape, 7.0, np.float32))
    cu = be.upload(np.array([0, lens[0], T], np.int32))
    be.launch_gated_delta_rule(base, base.data_ptr() + 4 * nk * dk, base.data_ptr() + 8 * nk * dk, d["g"], d["beta"], d["S"], T + pad, 2, nk, nv, dk,
                               dv, cu_seqlens=cu, q_stride=width, k_stride=width, v_stride=width, state_out=d["S"], out=out)
    got = be.read(out, np.float32, x["v"].shape)
    want, wS = expected(x, lens, 0.125, 1e-6)
    check(got[:T], want[:T], x, "out")
    assert np.all(got[T:] == 7.0)
    check(be.read(d["S"], np.float32, x["S"].shape), wS, x, "state")


@pytest.mark.parametrize("cu,spans", [([0, 5, 3], [(0, 5), (5, 5)]), ([-4, 2, 90], [(0, 2), (2, 6)]), ([2, 4, 6], [(2, 4), (4, 6)])])
def test_offsets_out_of_order_are_cut_and_reported(backend, cu, spans):
    be, x = backend, inputs(np.random.default_rng(1), [6], 1, 1, 64, 32)
    S = np.stack([x["S"][0], x["S"][0] * 2])
    d = {n: be.upload(a) for n, a in x.items()}
    out = be.upload(np.zeros(x["v"].shape, np.float32))
    _, so = be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], be.upload(S), 6, 2, 1, 1, 64, 32,
                                       cu_seqlens=be.upload(np.array(cu, np.int32)), out=out)
    if cu[0] == 2:
        be.sync()  # a first offset behind row 0 is in order
    else:
        with pytest.raises(BackendError, match="gated_delta_rule"):
            be.sync()
    got, gS = be.read(out, np.float32, x["v"].shape), be.read(so, np.float32, S.shape)
    for s, (b, e) in enumerate(spans):
        w, wS = ref.delta_rule(*(x[n][b:e] for n in ("q", "k", "v", "g", "beta")), S[s], 0.125, 1e-6)
        check(got[b:e], w, x, "out")
        check(gS[s], wS, x, "state")


def test_prompt_in_pieces_equals_the_whole(backend):
    """A prompt of 200 tokens at once, and as 70 + 129 + 1 with the state carried over: the same to rounding."""
    be, x = backend, inputs(np.random.default_rng(14), [200], 2, 4, 128, 128)
    out, S = launch(be, x, [200], 2, 4, 128, 128)
    state, at, parts = x["S"], 0, []
    for n in (70, 129, 1):
        piece = {m: (a[at:at + n] if m != "S" else state) for m, a in x.items()}
        o, state = launch(be, piece, [n], 2, 4, 128, 128)
        parts.append(o)
        at += n
    check(np.concatenate(parts), out.astype(np.float64), x, "out")
    check(state, S.astype(np.float64), x, "state")


def test_recorded_layer_and_repeated_bits(backend):
    """The mixer and its gated norm recorded together, replayed with new inputs; the same inputs give the same bits."""
    be, T, nk, nv, D = backend, 150, 2, 4, 128
    rng = np.random.default_rng(16)
    x = inputs(rng, [T], nk, nv, D, D)
    d = {n: be.upload(a) for n, a in x.items()}
    w, z = (1 + 0.02 * rng.standard_normal(D)).astype(np.float32), rng.standard_normal((T, nv, D)).astype(np.float32)
    dw, dz = be.upload(w), be.upload(z)
    out, so, y = be.empty(4 * T * nv * D), be.empty(4 * nv * D * D), be.empty(4 * T * nv * D)
    ws = be.empty(max(16, be.gated_delta_rule_workspace_bytes(T, 1, nk, nv, D, D)))

    def chain():
        be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], d["S"], T, 1, nk, nv, D, D, state_out=so, out=out, workspace=ws)
        be.launch_rms_norm_silu_gate(out, dz, dw, T * nv, D, 1e-6, out=y)

    chain()
    first = be.read(y, np.float32, (T, nv, D))
    be.graph_begin()
    chain()
    g = be.graph_end()
    be.graph_launch(g)
    assert np.array_equal(first, be.read(y, np.float32, (T, nv, D)))
    x2 = inputs(rng, [T], nk, nv, D, D)
    for n, a in x2.items():
        be.copy_h2d(d[n], a)
    be.sync()
    be.graph_launch(g)
    got, gout = be.read(y, np.float32, (T, nv, D)), be.read(out, np.float32, (T, nv, D))
    want, _ = expected(x2, [T], D ** -0.5, 1e-6)
    check(gout, want, x2, "out")
    normed = ref.gated_norm(gout, z, w, 1e-6)
    assert np.all(np.abs(got - normed) <= 1e-5 * np.abs(normed).max(-1, keepdims=True))
    be.graph_destroy(g)


def test_delta_refusals(backend):
    be = backend
    buf, st, o = be.empty(1 << 16), be.empty(1 << 17), be.empty(1 << 16)
    ok = dict(q=buf, k=buf, v=buf, g=buf, beta=buf, state=st, T=4, n_seqs=2, n_k_heads=1, n_v_heads=2, head_k=64, head_v=64, out=o, state_out=st)

    def refused(**kw):
        with pytest.raises(BackendError) as e:
            be.launch_gated_delta_rule(**{**ok, **kw})
        assert e.value.status == agn._abi.AGN_EINVAL

    refused(T=5)                # not two sequences of one length, and no offsets
    refused(T=-1, out=o)
    refused(n_seqs=0)
    refused(n_k_heads=3)
    refused(head_k=96)
    refused(head_v=48)
    refused(head_v=288)
    refused(q_stride=60)
    refused(q_stride=66)
    refused(scale=float("nan"))
    refused(l2norm_eps=float("nan"))
    refused(q=None)
    refused(g=None)
    refused(out=buf)            # in place
    refused(k=buf.data_ptr() + 4)
    refused(state=st.data_ptr() + 8)
    be.launch_gated_delta_rule(**{**ok, "T": 0})  # states are copied
    be.sync()


# ------------------------------------------------------------------------------------------------------- gated norm

@pytest.mark.parametrize("rows,n", [(1, 1), (3, 5), (7, 64), (32, 128), (33, 128), (5, 130), (4, 255), (2, 256), (3, 500), (6, 1000), (2, 1024)])
def test_gated_norm(backend, rows, n):
    rng = np.random.default_rng(rows * n)
    x, z = (rng.standard_normal((rows, n)).astype(np.float32) * np.float32(3) for _ in range(2))
    w = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    if rows > 2:
        x[1] = 0
        z[2] = -200.0  # exp(200) overflows: the gate is -0
    dx, dz, dw = (backend.upload(a) for a in (x, z, w))
    with np.errstate(over="ignore"):
        want = ref.gated_norm(x, z, w, 1e-6)
    got = backend.read(backend.launch_rms_norm_silu_gate(dx, dz, dw, rows, n, 1e-6), np.float32, (rows, n))
    # a product of five factors off by at most 4 steps each (rsqrt 2, exp 2, the rest 1), the sum of squares by n / 32 + 5 adds
    tol = (n / 32 + 30) * 2.0 ** -24
    assert np.all(np.abs(got - want) <= tol * np.abs(want) + 1e-37)
    for dt, np_of in ((AGN_F16, lambda a: a.view(np.float16).astype(np.float64)),
                      (AGN_BF16, lambda a: (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64))):
        o = backend.read(backend.launch_rms_norm_silu_gate_out16(dx, dz, dw, rows, n, 1e-6, dt), np.uint16, (rows, n))
        step = 2.0 ** -11 if dt == AGN_F16 else 2.0 ** -8
        assert np.all(np.abs(np_of(o) - got) <= step * np.abs(got) + 2.0 ** -25)
    out = backend.launch_rms_norm_silu_gate(dx, dz, dw, rows, n, 1e-6, out=dx)  # in place
    assert np.array_equal(backend.read(out, np.float32, (rows, n)), got)


def test_gated_norm_unaligned_and_refusals(backend):
    be, rng = backend, np.random.default_rng(5)
    x, z, w = (rng.standard_normal(s).astype(np.float32) for s in ((6, 64), (6, 64), (64,)))
    b = be.empty(4096 * 3)
    at = [b.data_ptr() + 4, b.data_ptr() + 4096 + 8, b.data_ptr() + 8192 + 4]
    for p, a in zip(at, (x, z, w)):
        be.copy_h2d(p, a)
    got = be.read(be.launch_rms_norm_silu_gate(*at, 6, 64, 1e-6), np.float32, (6, 64))
    want = ref.gated_norm(x, z, w, 1e-6)
    assert np.all(np.abs(got - want) <= 32 * 2.0 ** -24 * np.abs(want))
    for kw in (dict(rows=-1), dict(n=0), dict(n=1025), dict(x=None), dict(x=b.data_ptr() + 2)):
        with pytest.raises(BackendError):
            be.launch_rms_norm_silu_gate(**{**dict(x=at[0], gate=at[1], w=at[2], rows=1, n=64, eps=1e-6, out=b.data_ptr() + 8192 + 1024), **kw})
    with pytest.raises(BackendError) as e:
        be.launch_rms_norm_silu_gate_out16(*at, 1, 64, 1e-6, AGN_Q8_0, out=b)
    assert e.value.status == agn._abi.AGN_EUNSUPPORTED_DTYPE
    with pytest.raises(BackendError):
        be.launch_rms_norm_silu_gate_out16(*at, 1, 64, 1e-6, AGN_F16, out=at[0])
    be.sync()
