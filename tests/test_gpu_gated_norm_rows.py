"""agn_rms_norm_silu_gate_* over so many rows that a warp takes two of them: odd counts, rows that no vector fits, 16-bit results, in place; and rows whose
squares leave f32's range."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_BF16, AGN_F16
from tests import ref_mixers as ref

pytestmark = pytest.mark.gpu


def as_f64(bits, dtype):
    return bits.view(np.float16).astype(np.float64) if dtype == AGN_F16 else (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("rows", [9471, 9472, 9473, 9479, 20001])
@pytest.mark.parametrize("n", [128, 127, 64, 33, 4, 1])
@pytest.mark.parametrize("skew", [0, 4])
def test_many_rows(backend, rows, n, skew):
    be, rng = backend, np.random.default_rng(rows + n)
    x, z = (rng.standard_normal((rows, n)).astype(np.float32) * np.float32(2) for _ in range(2))
    w = (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
    x[rows - 1], z[rows - 2] = 0.01, -30.0
    at = []
    for a in (x, z, w):
        b = be.empty(a.nbytes + 16)
        be.copy_h2d(b.data_ptr() + skew, a)
        at.append(b)
    be.sync()
    px, pz, pw = (b.data_ptr() + skew for b in at)
    guard = np.full(rows * n + 64, 7.0, np.float32)
    out = be.upload(guard)
    be.launch_rms_norm_silu_gate(px, pz, pw, rows, n, 1e-6, out=out)
    got = be.read(out, np.float32, (rows * n + 64,))
    assert np.all(got[rows * n:] == 7.0)
    got = got[:rows * n].reshape(rows, n)
    want = ref.gated_norm(x, z, w, 1e-6)
    # five factors off by at most 4 steps each, the sum of squares by n / 32 + 5 additions
    assert np.all(np.abs(got - want) <= (n / 32 + 30) * 2.0 ** -24 * np.abs(want) + 1e-37)
    for dtype, step in ((AGN_F16, 2.0 ** -11), (AGN_BF16, 2.0 ** -8)):
        o = be.upload(np.full(rows * n + 64, 0x4242, np.uint16))
        be.launch_rms_norm_silu_gate_out16(px, pz, pw, rows, n, 1e-6, dtype, out=o)
        bits = be.read(o, np.uint16, (rows * n + 64,))
        assert np.all(bits[rows * n:] == 0x4242)
        assert np.all(np.abs(as_f64(bits[:rows * n].reshape(rows, n), dtype) - got) <= step * np.abs(got) + 2.0 ** -25)
    be.launch_rms_norm_silu_gate(px, pz, pw, rows, n, 1e-6, out=px)  # in place
    assert np.array_equal(be.read(px, np.float32, (rows, n)), got)
    be.copy_h2d(px, x)
    be.sync()
    be.launch_rms_norm_silu_gate(px, pz, pw, rows, n, 1e-6, out=pz)  # over the gate
    assert np.array_equal(be.read(pz, np.float32, (rows, n)), got)
