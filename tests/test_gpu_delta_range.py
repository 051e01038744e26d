"""The gated delta rule where magnitudes lie far apart: what a column or a row of the result is made of decides how exact it has to be, not what stands in other
columns, in later rows, or in a state that has decayed.  The columns of a state evolve independently, and no row reaches an earlier one."""
import numpy as np
import pytest

from tests.test_gpu_delta_rule import TOL, expected, inputs, launch

pytestmark = pytest.mark.gpu


def hold(got, want, size, what):
    """TOL of `size` (broadcast), the size of what the values are summed from."""
    err = np.abs(got.astype(np.float64) - want) / size
    assert err.max() <= TOL, (what, err.max(), np.unravel_index(np.argmax(err), err.shape))


def columns(x, want, wS):
    """Sizes per (head, column) of one sequence: of its state, values and results."""
    return np.maximum(np.maximum(np.abs(x["S"][0]).max(axis=1), np.abs(wS[0]).max(axis=1)), np.maximum(np.abs(x["v"]).max(axis=0), np.abs(want).max(axis=0)))


@pytest.mark.parametrize("T", [7, 64, 150])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e10, 1e20, 1e-10, 1e-20])
def test_a_column_of_another_size_leaves_its_neighbours_alone(backend, size, dk, T):
    x = inputs(np.random.default_rng(T), [T], 1, 2, dk, 64)
    for c in (3, 40):
        x["v"][:, 1, c] *= np.float32(size)
        x["S"][:, 1, :, c] *= np.float32(size)
    out, S = launch(backend, x, [T], 1, 2, dk, 64)
    want, wS = expected(x, [T], dk ** -0.5, 1e-6)
    of = columns(x, want, wS)
    hold(out, want, of[None], "out")
    hold(S[0], wS[0], of[:, None], "state")


@pytest.mark.parametrize("T", [20, 64, 150])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e15, 1e30])
@pytest.mark.parametrize("what", ["row", "element"])
def test_a_large_late_row_leaves_earlier_rows_alone(backend, what, size, T):
    x = inputs(np.random.default_rng(T), [T], 2, 2, 128, 32)
    late = T - 5
    if what == "row":
        x["v"][late] *= np.float32(size)
    else:
        x["v"][late, 1, 7] = size
    out, S = launch(backend, x, [T], 2, 2, 128, 32)
    want, wS = expected(x, [T], 128 ** -0.5, 1e-6)
    before = max(np.abs(x["S"]).max(), np.abs(x["v"][:late]).max())
    hold(out[:late], want[:late], before, "earlier rows")
    of = columns(x, want, wS)
    hold(out, want, of[None], "out")
    hold(S[0], wS[0], of[:, None], "state")


@pytest.mark.parametrize("T", [20, 64, 150])
@pytest.mark.parametrize("size", [1e4, 1e8, 1e15, 1e30])
@pytest.mark.parametrize("g", [-np.inf, -100.0])
def test_what_has_decayed_leaves_later_rows_alone(backend, g, size, T):
    """A large state and large first rows, dropped by one token's decay: the rows from there on are made of their own values."""
    x = inputs(np.random.default_rng(T), [T], 1, 2, 64, 64)
    drop = T // 2
    x["S"] *= np.float32(size)
    x["v"][:drop] *= np.float32(size)
    x["g"][drop] = g
    out, S = launch(backend, x, [T], 1, 2, 64, 64)
    want, wS = expected(x, [T], 0.125, 1e-6)
    after = np.abs(x["v"][drop:]).max() + size * np.exp(g) * 100
    hold(out[drop:], want[drop:], after, "later rows")
    hold(S, wS, after, "state")
    hold(out, want, max(np.abs(x["S"]).max(), np.abs(x["v"]).max()), "out")


@pytest.mark.parametrize("T", [10, 100])
def test_rows_of_the_state_of_different_sizes(backend, T):
    """Keys and queries along single axes: a query reads one row of the state, whatever stands in the others."""
    x = inputs(np.random.default_rng(1), [T], 1, 1, 64, 32)
    sizes = 10.0 ** np.linspace(-12, 12, 64)
    for n in "qk":
        x[n][:] = 0
        x[n][np.arange(T), 0, (np.arange(T) * 37 + (n == "q") * 11) % 64] = 1
    x["S"] = (x["S"] * sizes[None, None, :, None]).astype(np.float32)
    x["v"] = (x["v"] * sizes[np.argmax(x["k"][:, 0], axis=1), None, None]).astype(np.float32)
    out, S = launch(backend, x, [T], 1, 1, 64, 32, l2norm_eps=-1.0)
    want, wS = expected(x, [T], 0.125, -1.0)
    hold(out, want, 5 * sizes[np.argmax(x["q"][:, 0], axis=1), None, None], "out")
    hold(S[0, 0], wS[0, 0], 5 * sizes[:, None], "state")


def running(x, scale, eps):
    """(out, state, |S| of each head after every row [T, nv]) in float64, one sequence."""
    q, k, v, S = (x[n].astype(np.float64) for n in ("q", "k", "v", "S"))
    if eps >= 0:
        q, k = (a / np.sqrt((a * a).sum(-1, keepdims=True) + eps) for a in (q, k))
    rep, S = v.shape[1] // k.shape[1], S[0]
    q, k = (np.repeat(a, rep, axis=1) for a in (q * scale, k))
    out, size = np.zeros(v.shape), np.zeros(v.shape[:2])
    for t in range(len(v)):
        S = S * np.exp(x["g"][t].astype(np.float64))[:, None, None]
        d = x["beta"][t].astype(np.float64)[:, None] * (v[t] - np.einsum("hkv,hk->hv", S, k[t]))
        S = S + k[t][:, :, None] * d[:, None, :]
        out[t] = np.einsum("hkv,hk->hv", S, q[t])
        size[t] = np.abs(S).max(axis=(1, 2))
    return out, S, size, np.linalg.norm(q, axis=2)


@pytest.mark.parametrize("T", [10, 64, 100])
@pytest.mark.parametrize("what", ["queries", "keys", "both"])
@pytest.mark.parametrize("eps", [-1.0, 1e-6, 1.0])
@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-6, 1e-9])
def test_small_queries_and_keys_keep_their_bits(backend, size, eps, what, T):
    """Taken as they are, or far below the epsilon of their norm: an output row is as large as its query, a state that begins at 0 as its keys."""
    x = inputs(np.random.default_rng(T), [T], 2, 4, 128, 64)
    for n in "qk":
        x[n] /= np.sqrt((x[n] ** 2).sum(-1, keepdims=True))
    if what != "keys":
        x["q"][::2] *= np.float32(size)
    if what != "queries":
        x["k"] *= np.float32(size)
        x["S"][:] = 0
    out, S = launch(backend, x, [T], 2, 4, 128, 64, l2norm_eps=eps)
    want, wS, of_S, of_q = running(x, 128 ** -0.5, eps)
    hold(out, want, (of_S * of_q)[..., None], "out")
    hold(S[0], wS, of_S[-1][:, None, None], "state")


@pytest.mark.parametrize("T", [10, 64, 100])
@pytest.mark.parametrize("low", [1e-3, 1e-6, 1e-9])
def test_weak_writes_keep_their_bits(backend, low, T):
    """Write strengths of all sizes from `low` to 1, growing, on a state of 0: the first rows' results are as small as they are."""
    x = inputs(np.random.default_rng(T), [T], 1, 2, 64, 64)
    x["S"][:] = 0
    x["beta"][:] = np.exp(np.linspace(np.log(low), 0, T))[:, None]
    out, S = launch(backend, x, [T], 1, 2, 64, 64)
    want, wS, of_S, of_q = running(x, 0.125, 1e-6)
    hold(out, want, (of_S * of_q)[..., None], "out")
    hold(S[0], wS, of_S[-1][:, None, None], "state")


@pytest.mark.parametrize("T", [10, 100])
def test_long_queries_taken_as_they_are(backend, T):
    x = inputs(np.random.default_rng(T), [T], 1, 2, 64, 64)
    x["k"] /= np.sqrt((x["k"] ** 2).sum(-1, keepdims=True))
    x["q"] *= (10.0 ** np.random.default_rng(1).uniform(-6, 6, T)[:, None, None]).astype(np.float32)
    out, S = launch(backend, x, [T], 1, 2, 64, 64, l2norm_eps=-1.0)
    want, wS, of_S, of_q = running(x, 0.125, -1.0)
    hold(out, want, (of_S * of_q)[..., None], "out")
    hold(S[0], wS, of_S[-1][:, None, None], "state")


@pytest.mark.parametrize("T", [10, 150])
@pytest.mark.parametrize("size", [1e34, 1e36, 2e37])
@pytest.mark.parametrize("what", ["all", "the state", "a state along the keys", "a late value"])
def test_near_the_end_of_f32s_range(backend, what, size, T):
    """What stays finite token by token stays finite, and exact, whatever the form."""
    x = inputs(np.random.default_rng(T), [T], 1, 2, 128, 64)
    if what == "all":
        x["v"] *= np.float32(size)
    if what == "a state along the keys":  # sums of 128 terms of one sign
        x["k"][:], x["S"][:] = 1, 0.3 * size
    elif what != "a late value":
        x["S"] *= np.float32(size)
    else:
        x["v"][T - 3, 1, 5] = size
    out, S = launch(backend, x, [T], 1, 2, 128, 64)
    want, wS = expected(x, [T], 128 ** -0.5, 1e-6)
    of = columns(x, want, wS)
    hold(out, want, of[None], "out")
    hold(S[0], wS[0], of[:, None], "state")


@pytest.mark.parametrize("T", [10, 64, 150])
@pytest.mark.parametrize("size", [1e-28, 1e-31, 1e-33, 1e-35])
def test_near_the_smallest_numbers_of_f32(backend, size, T):
    x = inputs(np.random.default_rng(T), [T], 1, 2, 64, 64)
    x["v"] *= np.float32(size)
    x["S"] *= np.float32(size)
    out, S = launch(backend, x, [T], 1, 2, 64, 64)
    want, wS = expected(x, [T], 0.125, 1e-6)
    of = columns(x, want, wS)
    hold(out, want, of[None], "out")
    hold(S[0], wS[0], of[:, None], "state")
