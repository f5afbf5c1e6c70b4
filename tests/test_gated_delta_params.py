"""Parameters of raw gates as weights come: of two dtypes, or views of wider tensors."""

import itertools

import pytest
import torch

import causal_conv1d_cute as C
from causal_conv1d_cute import gated_delta as G
from test_gated_delta import BF, F16, F32, gpu, make


@pytest.mark.gpu
@pytest.mark.parametrize("adtype,ddtype", list(itertools.product([F32, BF, F16], repeat=2)))
@pytest.mark.parametrize("strided", [False, True])
def test_dtypes_and_strides(adtype, ddtype, strided):
    """The same bits as with fp32 copies of the values."""
    T = 130
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, 1, 3, 128, 128, BF))
    A, dt = A.to(adtype), dt.to(ddtype)
    given = (torch.stack([A, A], 1)[:, 0], torch.stack([dt, dt], 1)[:, 1]) if strided else (A, dt)
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda")

    def run(A_log, dt_bias):
        kw = dict(A_log=A_log, dt_bias=dt_bias, qk_l2norm=True)
        st, sd = torch.zeros(1, 3, 128, 128, device="cuda"), torch.zeros(T, 3, 128, 128, device="cuda")
        o = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, None, st, **kw)
        d, fin = C.gated_delta_rule_fn(*(t[None] for t in (q, k, v, g, b)), None, True, **kw)
        return o, st, d, fin, C.gated_delta_rule_update(q, k, v, g, b, sd, **kw), sd

    for x, y in zip(run(*given), run(A.float(), dt.float())):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_other_dtypes_are_refused():
    q, k, v, g, b, A, dt = (gpu(t) for t in make(3, 1, 2, 128, 128, BF))
    for bad in ((A.double(), dt), (A, dt.double()), (A, dt.int())):
        assert "dtypes" in G.gated_delta_rule_reason(q, k, v, g, b, None, *bad)
        with pytest.raises(C.Unsupported, match="A_log"):
            C.gated_delta_rule_update(q, k, v, g, b, torch.zeros(3, 2, 128, 128, device="cuda"), A_log=bad[0], dt_bias=bad[1])
