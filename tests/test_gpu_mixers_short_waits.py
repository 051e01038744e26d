"""Waits of the token mixers that run out: each of their kernels' waits is bounded by the option "mbar_spin_limit", and a call whose waits ran
out is reported by the next sync.  So whatever the limit, a call either gives its result or raises; it never does neither."""
import numpy as np
import pytest

from agention_infer_b200 import AGN_F16, BackendError, _abi
from tests import ref_mixers as ref
from tests.test_gpu_attention_kv import Cache, close
from tests.test_gpu_delta_rule import check, expected, inputs

pytestmark = pytest.mark.gpu

LIMITS = [1, 1, 1, 1, 2, 2, 3, 4, 6, 8, 16, 64, 1025]


def attempt(be, limit, call):
    """True: the call's waits ran out and sync said so."""
    be.set_option("mbar_spin_limit", limit)
    try:
        call()
        be.sync()
        return False
    except BackendError as e:
        assert e.status == _abi.AGN_ETIMEOUT and "wait" in str(e), e
        return True
    finally:
        be.set_option("mbar_spin_limit", 1 << 22)


@pytest.mark.parametrize("T", [40, 64, 65, 130, 300])
@pytest.mark.parametrize("nk,nv", [(1, 1), (4, 8)])
def test_delta_rule_gives_its_result_or_says_that_it_did_not(backend, T, nk, nv):
    be, rng = backend, np.random.default_rng(T)
    x = inputs(rng, [T], nk, nv, 128, 128)
    d = {n: be.upload(a) for n, a in x.items()}
    want, wS = expected(x, [T], 128 ** -0.5, 1e-6)
    out, S = be.empty(x["v"].nbytes), be.empty(x["S"].nbytes)
    ws = be.empty(be.gated_delta_rule_workspace_bytes(T, 1, nk, nv, 128, 128))
    blank = np.full(max(x["v"].size, x["S"].size), np.nan, np.float32)

    def call():
        be.launch_gated_delta_rule(d["q"], d["k"], d["v"], d["g"], d["beta"], d["S"], T, 1, nk, nv, 128, 128, state_out=S, out=out, workspace=ws)

    for limit in LIMITS:
        be.copy_h2d(out, blank[:x["v"].size])
        be.copy_h2d(S, blank[:x["S"].size])
        be.sync()
        if not attempt(be, limit, call):
            check(be.read(out, np.float32, x["v"].shape), want, x, "out")
            check(be.read(S, np.float32, x["S"].shape), wS, x, "state")
    call()  # and the context is as good as before
    check(be.read(out, np.float32, x["v"].shape), want, x, "out")
    be.sync()


@pytest.mark.parametrize("T,start,hd", [(9, 0, 64), (40, 100, 128), (300, 0, 128), (16, 3000, 64)])
def test_f16_prompts_give_their_result_or_say_that_they_did_not(backend, T, start, hd):
    """One tile, a few, several row tiles, and slots that are shared out."""
    be, rng, nq, nkv = backend, np.random.default_rng(T), 8, 2
    n = start + T
    c = Cache(be, rng, "q8_0", 1, n, nkv, hd, [n])
    q = rng.standard_normal((T, nq, hd)).astype(np.float16)
    dq, out = be.upload(q), be.empty(q.nbytes)
    ws = be.empty(be.attention_kv_workspace_bytes(T, nq, nkv, hd, n, False))
    k, v = c.values(0, n)
    want, mag = ref.attention(q, k, v, [start + t for t in range(T)], hd ** -0.5)

    def call():
        be.launch_attention_kv(dq, c.bufs[0], c.bufs[1], c.kv, T, nq, nkv, hd, n, pos_start=start, act_dtype=AGN_F16, out=out, workspace=ws)

    for limit in LIMITS:
        be.copy_h2d(out, np.full(q.shape, np.nan, np.float16))
        be.sync()
        if not attempt(be, limit, call):
            close(be.read(out, np.float16, q.shape), want, mag, q, k, n, hd ** -0.5, "f16")
    call()
    close(be.read(out, np.float16, q.shape), want, mag, q, k, n, hd ** -0.5, "f16")
    be.sync()
