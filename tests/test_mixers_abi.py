"""Entry points of the token mixers without a GPU: a null context is refused, workspace sizes are host arithmetic."""
import pytest

from agention_infer_b200 import _abi
from agention_infer_b200.build import build_library


@pytest.fixture(scope="module")
def lib():
    build_library()
    return _abi.load()


def test_null_context_is_refused(lib):
    for f in (lib.agn_attention_kv_f32, lib.agn_attention_kv_f16):
        assert f(None, None, None, _abi.AGN_Q8_0, None, None, 1, 4, 2, 64, None, 0, None, 1, 16, 0.125, None, 0) == _abi.AGN_EINVAL
    assert lib.agn_gated_delta_rule_f32(None, *[None] * 8, 1, 1, None, 1, 1, 64, 64, 64, 64, 64, 0.125, 1e-6, None, 0) == _abi.AGN_EINVAL
    assert lib.agn_rms_norm_silu_gate_f32(None, None, None, None, None, 1, 64, 1e-6) == _abi.AGN_EINVAL
    assert lib.agn_rms_norm_silu_gate_f32_out16(None, None, None, None, None, 1, 64, 1e-6, _abi.AGN_F16) == _abi.AGN_EINVAL


@pytest.mark.parametrize("T,nq,nkv,hd,slots", [(-1, 4, 2, 64, 16), (1, 4, 3, 64, 16), (1, 4, 2, 48, 16), (1, 4, 2, 64, 0), (1, 0, 0, 64, 16), (1 << 40, 4, 2, 64, 16)])
def test_workspace_of_refused_sizes_is_zero(lib, T, nq, nkv, hd, slots):
    for has_pos in (0, 1):
        assert lib.agn_attention_kv_workspace_bytes(T, nq, nkv, hd, slots, has_pos) == 0


def test_workspace_sizes_are_not_negative(lib):
    for T in (0, 1, 7, 64, 5000):
        for slots in (1, 100, 32768, 1 << 30):
            for has_pos in (0, 1):
                assert lib.agn_attention_kv_workspace_bytes(T, 28, 4, 128, slots, has_pos) >= 0
        for n in (1, 3, 64):
            assert lib.agn_gated_delta_rule_workspace_bytes(T, n, 16, 32, 128, 128) >= 0
    assert lib.agn_gated_delta_rule_workspace_bytes(10, 1, 3, 4, 128, 128) == 0


@pytest.mark.parametrize("T,nq,nkv,hd", [(277, 16, 2, 64), (250, 7, 1, 128), (38, 4, 1, 64), (556, 14, 2, 64), (64, 4, 1, 256), (129, 8, 1, 96)])
def test_a_longer_cache_never_asks_for_less_workspace(lib, T, nq, nkv, hd):
    """Rows may end anywhere in the cache, so that a size is enough for every shorter one."""
    sizes = [lib.agn_attention_kv_workspace_bytes(T, nq, nkv, hd, slots, 0) for slots in range(T, T + 6000, 16)]
    assert all(b >= a for a, b in zip(sizes, sizes[1:]))
