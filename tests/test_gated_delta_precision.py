"""The final fp32 states of the chunked gated delta rule hold the precision of fp32.

Tolerance, as the 2-norm of the difference over the 2-norm of the state, for each head of each
sequence: 2^-19, which is 32 roundings of fp32 (2^-24): operands of the products hold 24 bits, and what
is left are the sums of five products in a row, the norms, and decays of a few ulp."""

import itertools

import pytest
import torch

import causal_conv1d_cute as C
from test_gated_delta import BF, F16, gates, gpu, make, near, rule

TOL = 2.0**-19


def states_case(lengths, hk, hv, dtype, dv=128, raw=True, seed=0, change=None, tol=TOL):
    T, n = sum(lengths), len(lengths)
    q, k, v, g, b, A, dt = make(T, hk, hv, 128, dv, dtype, raw, seed, unit=not raw)
    if change is not None:
        change(q, k, v, g, b)
    start = [0, *itertools.accumulate(lengths)]
    gg, bb = gates(g, b, A, dt)
    st = torch.randn(n, hv, 128, dv, generator=torch.Generator().manual_seed(seed)) * 0.3
    got = gpu(st)
    out = C.gated_delta_rule_varlen_fn(
        gpu(q), gpu(k), gpu(v), gpu(g), gpu(b), torch.tensor(start, dtype=torch.int32, device="cuda"), None,
        torch.ones(n, dtype=torch.bool, device="cuda"), got, A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=raw)
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    for i in range(n):
        s = slice(start[i], start[i + 1])
        want, S = rule(q[s], k[s], v[s], gg[s], bb[s], st[i], 128**-0.5, raw)
        off = (got[i] - S).flatten(1).norm(dim=1) / S.flatten(1).norm(dim=1)
        assert off.max() <= tol, f"sequence {i}: {off.max():.3g} off"
        near(out[s], want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("lengths,hk,hv,dv", [
    ([700], 1, 3, 128),  # few heads: tiles of 32 columns
    ([130, 64, 65, 200], 20, 40, 128),  # more: 64 (bf16)
    ([65, 130, 64, 90, 20, 97, 10, 33], 20, 40, 128),  # many: 128
    ([129, 77, 300], 1, 2, 256),
])
def test_states_of_random_keys(lengths, hk, hv, dv, dtype):
    states_case(lengths, hk, hv, dtype, dv, seed=dv + hv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("hk,hv", [(1, 2), (40, 40)])
def test_states_without_decay(hk, hv, dtype):
    """Nothing is forgotten: every chunk's error stays in the state."""

    def change(q, k, v, g, b):
        g.zero_()

    states_case([400, 150, 64, 100, 66, 70, 80, 90], hk, hv, dtype, raw=False, change=change)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("hk,hv", [(1, 2), (40, 40)])
def test_states_of_equal_keys(hk, hv, dtype):
    """One key throughout: u cancels over the tokens of a chunk, which leaves a state some twenty times
    smaller than what was added to it. Tolerance: that of fp32 results everywhere, 2e-5."""

    def change(q, k, v, g, b):
        k[:] = k[:1]

    states_case([400, 150, 64, 100, 66, 70, 80, 90], hk, hv, dtype, change=change, tol=2e-5)
