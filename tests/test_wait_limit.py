"""Waits inside the chunked delta rule that run out: told by NaN outputs, caches that keep their states, and
the device status word, whether index checks are on or off."""

import itertools

import pytest
import torch

import causal_conv1d_cute as C
from causal_conv1d_cute import _lib
from test_gated_delta import BF, F16, F32, gpu, make


def test_limit_is_checked():
    lib = _lib.load()
    assert lib.cc1d_set_wait_limit(-1) == 1 and b"limit" in lib.cc1d_last_error()
    assert lib.cc1d_set_wait_limit(2_000_000_000) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("checks", [True, False])
@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (BF, BF), (F16, F32)])
@pytest.mark.parametrize("hk,hv,dv", [(1, 2, 128), (20, 40, 128), (40, 40, 256)])  # 32, 64 and 128 columns
def test_waits_that_run_out(request, hk, hv, dv, dtype, sdtype, checks):
    """Nothing is copied, so that every wait is for something that never comes."""
    request.node._expect_status = True
    lengths = [65, 3, 0, 130, 64]
    q, k, v, g, b, A, dt = (gpu(t) for t in make(sum(lengths), hk, hv, 128, dv, dtype))
    start = torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int32, device="cuda")
    idx = torch.tensor([4, 0, 1, 5, 2], dtype=torch.int32, device="cuda")
    hinit = torch.tensor([1, 0, 1, 0, 1], dtype=torch.bool, device="cuda")
    before = torch.randn(6, hv, 128, dv, device="cuda").to(sdtype)
    whole = torch.full((sum(lengths) + 2, hv, dv), 7.0, device="cuda", dtype=dtype)
    C.set_device_checks(checks)
    lib = _lib.load()

    def run(states):
        return C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, idx, hinit, states, A_log=A, dt_bias=dt, qk_l2norm=True,
                                            out=whole[1:-1])

    good = before.clone()
    want = run(good).clone()
    assert C.device_status() == 0 and torch.isfinite(want.float()).all()
    states = before.clone()
    assert lib.cc1d_set_wait_limit(0) == 0
    try:
        got = run(states)
        assert C.device_status() == _lib.DEV_TIMEOUT
    finally:
        assert lib.cc1d_set_wait_limit(2_000_000_000) == 0
    assert torch.isnan(got).all() and torch.equal(states, before)
    assert (whole[0] == 7).all() and (whole[-1] == 7).all()
    # The context and the next call are as before.
    again = run(states)
    assert C.device_status() == 0
    assert torch.equal(again, want) and torch.equal(states, good)
