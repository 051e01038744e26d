"""Calls of the token mixers that are refused before anything is launched."""
import pytest

import agention_infer_b200 as agn
from agention_infer_b200 import AGN_Q8_0, BackendError

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["g", "beta", "cu_seqlens"])
@pytest.mark.parametrize("T", [4, 200])
@pytest.mark.parametrize("skew", [1, 2, 3])
def test_delta_rule_refuses_floats_and_offsets_between_elements(backend, which, T, skew):
    """Both forms (the recurrent and the chunked one): g and beta are read as floats, cu_seqlens as 32-bit numbers."""
    be = backend
    buf, out, state = be.empty(1 << 18), be.empty(1 << 18), be.empty(1 << 16)
    args = dict(q=buf, k=buf, v=buf, g=buf, beta=buf, state=state, T=T, n_seqs=1, n_k_heads=1, n_v_heads=2, head_k=64, head_v=64,
                out=out, state_out=state)
    launches = be.launch_count
    with pytest.raises(BackendError) as e:
        be.launch_gated_delta_rule(**{**args, which: buf.data_ptr() + skew})
    assert e.value.status == agn._abi.AGN_EINVAL and which in str(e.value)
    assert be.launch_count == launches


@pytest.mark.parametrize("which", ["pos", "seq"])
@pytest.mark.parametrize("skew", [1, 2])
def test_attention_refuses_positions_between_elements(backend, which, skew):
    be = backend
    buf, cache, out = be.empty(1 << 16), be.empty(1 << 16), be.empty(1 << 16)
    args = dict(q=buf, k_cache=cache, v_cache=cache, kv_dtype=AGN_Q8_0, T=2, n_q_heads=4, n_kv_heads=2, head_dim=64, max_seq_len=16,
                pos=buf, seq=buf, out=out)
    launches = be.launch_count
    with pytest.raises(BackendError) as e:
        be.launch_attention_kv(**{**args, which: buf.data_ptr() + skew})
    assert e.value.status == agn._abi.AGN_EINVAL and which in str(e.value)
    assert be.launch_count == launches
