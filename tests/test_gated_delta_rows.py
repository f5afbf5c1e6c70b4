"""The gated delta rule row by row: the output of every token and head, and the state of every head, is within
the tolerance by itself, so that no wrong column or token hides in the norm of the rest.

Tolerances, in 2-norms. A head's state S is within 2e-5 of its norm. An output is scale S^T q with |q| = 1, so
that an error of S of 2e-5 leaves one of 2e-5 scale |S|, however small the output itself has become. To
either comes the rounding to its type: the unit roundoff times each value, and for values of fp16 below its
normal range half of their spacing, 2^-25."""

import itertools

import pytest
import torch

import causal_conv1d_cute as C
from test_gated_delta import BF, F16, F32, UNIT, gates, gpu, make, rule


class Norms(list):
    """Takes the states after each token, and keeps the norm of each head's."""

    def append(self, S):
        super().append(S.flatten(1).norm(dim=1))


def rows_near(got, ref, axes, norms=None):
    """Norms over the last `axes` axes; norms: of what the rows were made of, if not of themselves."""
    unit, tiny = UNIT[got.dtype], 2.0**-25 if got.dtype == F16 else 0.0
    got, ref = got.double().cpu().flatten(-axes), ref.double().cpu().flatten(-axes)
    assert got.shape == ref.shape and torch.isfinite(got).all()
    off, norm = (got - ref).norm(dim=-1), ref.norm(dim=-1)
    most = 2e-5 * (norm if norms is None else norms) + unit * norm + tiny * ref.shape[-1] ** 0.5
    bad = (off > most).nonzero()
    assert not len(bad), f"{len(bad)} rows, first {bad[0].tolist()}: {(off / most).max():.3g} of what is allowed"


def recorded_case(B, steps, hk, hv, dv, dtype, sdtype, update, pads=(), seed=0):
    """Decode with the state recorded after every token; 128 x dv states."""
    d = 128
    q, k, v, g, b, A, dt = make(B * steps, hk, hv, d, dv, dtype, seed=seed)
    q, k, v, g, b = (t.unflatten(0, (B, steps)) for t in (q, k, v, g, b))
    r = torch.Generator().manual_seed(seed + 1)
    st = torch.randn(B + 2, hv, d, dv, generator=r).mul(0.3).to(sdtype)
    idx, iidx = torch.randperm(B + 2, generator=r)[:B].int(), torch.randperm(B + 1, generator=r)[:B].int()
    for p in pads:
        idx[p] = -1
    inter = torch.full((B + 1, steps, hv, d, dv), 3.0).to(sdtype)
    ds, di = gpu(st), gpu(inter)
    got = C.gated_delta_rule_update(
        *(gpu(t) for t in (q, k, v, g, b)), ds, idx.cuda(), A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=True,
        intermediate_states=di, intermediate_state_indices=iidx.cuda(), update_states=update).cpu()
    gg, bb = gates(g, b, A, dt)
    want_st, want_in, ds, di = st.double(), inter.double(), ds.cpu(), di.cpu()
    for i in range(B):
        if idx[i] < 0:
            continue
        rec = []
        want, S = rule(q[i], k[i], v[i], gg[i], bb[i], st[idx[i]], d**-0.5, True, rec)
        rows_near(got[i], want, 1, d**-0.5 * torch.stack(rec).flatten(2).norm(dim=2))
        want_in[iidx[i]] = torch.stack(rec)
        if update:
            want_st[idx[i]] = S
    rows_near(ds, want_st, 2)
    rows_near(di, want_in, 2)
    used = idx[idx >= 0].tolist() if update else []
    rest = [s for s in range(B + 2) if s not in used]
    assert torch.equal(ds[rest], st[rest])
    rest = [s for s in range(B + 1) if s not in iidx[idx >= 0].tolist()]
    assert torch.equal(di[rest], inter[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sdtype", [(BF, BF), (F16, F16)])
@pytest.mark.parametrize("steps", [1, 2, 4, 7, 16])
@pytest.mark.parametrize("dv", [128, 256])
@pytest.mark.parametrize("update", [True, False])
def test_recorded_16_bit_states(dtype, sdtype, steps, dv, update):
    """Whole heads to a CTA, whatever their number."""
    recorded_case(3, steps, 1, 3, dv, dtype, sdtype, update, pads=(1,) if steps == 4 else (), seed=steps)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("update", [True, False])
def test_recorded_fp32_states_of_many_heads(dtype, update):
    """From 740 heads on whole heads to a CTA; below that (the last case) tiles of 32 columns."""
    recorded_case(62, 3, 4, 12, 128, dtype, F32, update, pads=(5, 61))
    recorded_case(31, 2, 4, 12, 256, dtype, F32, update)
    recorded_case(61, 2, 4, 12, 128, dtype, F32, update)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (BF, BF), (F16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("lengths,hk,hv,dv", [
    ([1, 63, 64, 65, 130, 200, 7], 1, 2, 128),  # few heads: tiles of 32 columns
    ([1, 63, 64, 65, 130, 20, 7], 11, 22, 128),  # 64 (bf16)
    ([1, 63, 64, 65, 130, 20, 7], 22, 44, 128),  # 128
    ([1, 63, 64, 65, 130, 20, 7], 1, 2, 96),
    ([2] * 40 + [130, 33] + [1] * 20, 1, 2, 128),  # long ones among short ones
])
def test_prefill_rows(lengths, hk, hv, dv, dtype, sdtype):
    T, n = sum(lengths), len(lengths)
    q, k, v, g, b, A, dt = make(T, hk, hv, 128, dv, dtype, seed=dv + hv)
    start = [0, *itertools.accumulate(lengths)]
    st = torch.randn(n, hv, 128, dv, generator=torch.Generator().manual_seed(1)).mul(0.3).to(sdtype)
    ds = gpu(st)
    got = C.gated_delta_rule_varlen_fn(
        gpu(q), gpu(k), gpu(v), gpu(g), gpu(b), torch.tensor(start, dtype=torch.int32, device="cuda"), None,
        torch.ones(n, dtype=torch.bool, device="cuda"), ds, A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=True).cpu()
    gg, bb = gates(g, b, A, dt)
    for i in range(n):
        s = slice(start[i], start[i + 1])
        norms = Norms()
        want, S = rule(q[s], k[s], v[s], gg[s], bb[s], st[i], 128**-0.5, True, norms)
        rows_near(got[s], want, 1, 128**-0.5 * torch.stack(norms))
        rows_near(ds[i], S, 2)
