"""The row-wise check of attention's results tells right from wrong: rounding passes; a result of zeros, a mask that is off by one slot, operands in too few bits
and lost shares do not.  (On the CPU, on inputs like those of the GPU tests.)"""
import numpy as np
import pytest

from tests import mixers_norms as norms
from tests import ref_mixers as ref

SHAPES = [(16, 4000, 8, 2, 128), (37, 4091, 4, 2, 256), (64, 2936, 4, 1, 256), (20, 70, 8, 2, 64), (200, 0, 8, 2, 64), (40, 100, 8, 2, 128), (24, 2000, 8, 2, 128)]


def data(T, start, nq, nkv, hd, act, seed=0):
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((start + T, nkv, hd)).astype(np.float32).astype(np.float64) for _ in range(2))
    q = rng.standard_normal((T, nq, hd)).astype(np.float32 if act == "f32" else np.float16)
    return q, k, v, [start + t for t in range(T)], hd ** -0.5


def test_the_reference_agrees_with_the_other_one():
    q, k, v, pos, scale = data(30, 50, 6, 2, 32, "f32")
    pos[3] = -1
    want, _ = ref.attention(q, k, v, pos, scale)
    got, size = norms.attention(q, k, v, pos, scale)
    assert np.abs(got - want).max() < 1e-13 and np.all(size[3] == 0)


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_wrong_results_are_rejected(shape, act):
    q, k, v, pos, scale = data(*shape, act)
    n = len(k)
    want, size = norms.attention(q, k, v, pos, scale)

    def rejected(got):  # one row that is further off than allowed is enough to fail a test; what is wrong throughout shows in nearly every row
        return norms.violations(got, want, size, q, k, n, scale, act).mean()

    assert rejected(np.zeros_like(want)) > 0.95
    if pos[0] >= 8:  # a row's own slot, or its last eight, left out: as visible as their weights are
        assert rejected(norms.attention(q, k, v, [p - 1 for p in pos], scale)[0]) > 0.3
        assert rejected(norms.attention(q, k, v, [p - 8 for p in pos], scale)[0]) > 0.9
    b = lambda x: (np.ascontiguousarray(x, np.float32).view(np.uint32) + 0x8000 & 0xFFFF0000).view(np.float32).astype(np.float64)  # noqa: E731
    if act == "f32":
        assert rejected(norms.attention(q.astype(np.float16), k, v, pos, scale)[0]) > 0.95
        assert rejected(norms.attention(q, k, v.astype(np.float16).astype(np.float64), pos, scale)[0]) > 0.95
    else:
        assert rejected(norms.attention(b(q).astype(np.float16), b(k), b(v), pos, scale)[0]) > 0.5


@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [1.0, 3.0])
def test_rounding_passes(shape, act, size):
    """Operands rounded once each to the bits that the bound is made for."""
    q, k, v, pos, scale = data(*shape, act, seed=1)
    q = (q * size).astype(q.dtype)
    want, rows = norms.attention(q, k, v, pos, scale)
    if act == "f16":
        got = norms.attention(q, k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64), pos, scale)[0].astype(np.float16)
    else:
        r = lambda x: x + np.random.default_rng(2).uniform(-1, 1, x.shape) * norms.U["f32"] * np.abs(x)  # noqa: E731
        got = norms.attention(r(q.astype(np.float64)), r(k), r(v), pos, scale)[0].astype(np.float32)
    assert not norms.violations(got, want, rows, q, k, len(k), scale, act).any()
