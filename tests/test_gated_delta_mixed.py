"""Batches of mostly short sequences that hold long ones: those go chunk by chunk, the rest token by token."""

import ctypes
import itertools

import pytest
import torch

import causal_conv1d_cute as C
from causal_conv1d_cute import _lib
from test_gated_delta import BF, F16, F32, gpu, make, varlen_case

MIXED = {
    "one": [1] * 60 + [300] + [1] * 20,
    "some": [1] * 90 + [0] * 50 + [129] + [2] * 30 + [65] + [33, 32, 31] + [1] * 20,
    "padded": [0] * 100 + [400] + [0] * 10,
    "short": [3] * 60,
    "many": [33] * 40 + [64, 65, 70] + [0] * 200,  # more than a list holds: those above 64
    "first-and-last": [70] + [1] * 40 + [40],
    "steps-of-1024": [1] * 1000 + [50] + [0] * 23 + [45] + [1] * 1100 + [100],
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(MIXED))
def test_mixed_lengths(name):
    lengths = MIXED[name]
    assert 128 <= sum(lengths) < 12 * len(lengths)
    varlen_case(lengths, hk=1, hv=2, seed=len(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sdtype", [(BF, BF), (F16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("hk,hv,dv", [(2, 6, 128), (1, 1, 256), (3, 3, 64)])
def test_mixed_types_and_heads(dtype, sdtype, hk, hv, dv):
    varlen_case([2] * 40 + [130, 33] + [1] * 20, hk=hk, hv=hv, dv=dv, dtype=dtype, sdtype=sdtype, seed=hv)


@pytest.mark.gpu
@pytest.mark.parametrize("states,pad", [(False, None), (True, 41), (True, 3)])
def test_mixed_without_cache_and_with_a_pad(states, pad):
    varlen_case([2] * 40 + [33, 130] + [1] * 20, states=states, pad=pad)


def block(rows, tokens, hk=16, hv=48, longest=0):
    """A packed argument block of bf16 tensors, for questions that touch no memory."""
    d, at = 128, 1 << 20
    heads = (0, (2 * hk + hv) * d, d, 1)
    return _lib.GDR_ARGS.pack(at, at, at, at, at, 0, 0, at, at, 0, 0, 0, at, 0, 0, 0, *heads, *heads, *heads, 0, hv * d, d, 1,
                              0, hv, 1, 0, hv, 1, hv * d * d, d * d, d, 0, 0, 0, 0, rows, tokens, rows, 0, 0,
                              longest, hk, hv, d, d, 0, 0, 0, 2, 2, 1, 1, -1, 1.0)


def workspace(*args, **kw):
    need = ctypes.c_int64(-1)
    assert _lib.load().cc1d_gdr_workspace(block(*args, **kw), ctypes.byref(need)) == 0
    return need.value


@pytest.mark.gpu
def test_workspace_of_mixed_batches():
    """A long prompt may be among them: room for the chunks of 32 sequences, or of as many as can be long."""
    chunk = 48 * 49936
    assert workspace(513, 512 + 4096) >= (4608 // 64 + 32) * chunk
    assert workspace(513, 512 + 4096) < (4608 // 64 + 34) * chunk
    assert (2 + 4) * chunk > workspace(20, 130) >= (2 + 3) * chunk
    assert workspace(64, 127) == 0 and workspace(10, 119) == 0
    assert workspace(10, 120) >= (1 + 10) * chunk


@pytest.mark.gpu
def test_no_long_ones_are_looked_for_where_there_are_none():
    assert workspace(64, 512) > 0 and workspace(64, 512, longest=33) == workspace(64, 512)
    assert workspace(64, 512, longest=8) == 0 and workspace(64, 512, longest=32) == 0
    assert workspace(4, 512, longest=128) == workspace(4, 512) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("B,L", [(20, 7), (13, 11), (12, 40)])
def test_dense_batches_of_short_sequences(B, L):
    """The same bits as the packed call, which does not know the lengths."""
    q, k, v, g, b, A, dt = (gpu(t) for t in make(B * L, 1, 2, 128, 128, BF))
    args = dict(A_log=A, dt_bias=dt, qk_l2norm=True)
    st = torch.randn(B, 2, 128, 128, device="cuda")
    out, fin = C.gated_delta_rule_fn(*(t.unflatten(0, (B, L)) for t in (q, k, v, g, b)), st, True, **args)
    start = torch.arange(0, B * L + 1, L, dtype=torch.int32, device="cuda")
    hinit = torch.ones(B, dtype=torch.bool, device="cuda")
    packed = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, hinit, st, **args)
    assert torch.equal(out.flatten(0, 1), packed) and torch.equal(fin, st)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("limit", [1, 3_000_000])
def test_mixed_in_groups_of_heads(monkeypatch, limit, dtype):
    from causal_conv1d_cute import _ops

    lengths = [1] * 30 + [100, 65] + [3] * 20
    q, k, v, g, b, A, dt = (gpu(t) for t in make(sum(lengths), 5, 10, 128, 128, dtype))
    start = torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int32, device="cuda")

    def run():
        s = torch.ones(len(lengths), 10, 128, 128, device="cuda")
        hinit = torch.ones(len(lengths), dtype=torch.bool, device="cuda")
        return C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, hinit, s, A_log=A, dt_bias=dt, qk_l2norm=True), s

    o0, s0 = run()
    monkeypatch.setattr(_ops, "_GDR_WORKSPACE", limit)
    o1, s1 = run()
    assert torch.equal(o0, o1) and torch.equal(s0, s1)


@pytest.mark.gpu
def test_bad_bounds_among_mixed(request):
    request.node._expect_status = True
    lengths = [1] * 40 + [100] + [1] * 20
    T = sum(lengths)
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, 1, 2, 128, 128, BF))
    start = torch.tensor([0, *itertools.accumulate(lengths)], dtype=torch.int32, device="cuda")
    st = torch.randn(len(lengths), 2, 128, 128, device="cuda")
    want = st.clone()
    args = dict(A_log=A, dt_bias=dt, qk_l2norm=True)
    C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, None, want, **args)
    start[-1] = T + 1
    got = st.clone()
    C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, None, got, **args)
    assert C.device_status() == _lib.DEV_BAD_QSL
    assert torch.equal(got[:-1], want[:-1]) and torch.equal(got[-1], st[-1])
