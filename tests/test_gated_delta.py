"""Gated delta rule (packed and dense prefill, decode) and gated RMS norm against their definitions
in 64 bits.

Tolerances, as the 2-norm of the difference over the 2-norm of the result: fp32 results 2e-5 (the
chunked kernel splits fp32 operands into two bf16 parts, 2^-17 apart from them, through five
products in a row); results of 16 bits the unit roundoff of their type (2^-8, 2^-11) more."""

import itertools

import pytest
import torch

import causal_conv1d_cute as C
from causal_conv1d_cute import _lib
from causal_conv1d_cute import gated_delta as G

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF: 2.0**-8, F16: 2.0**-11, F32: 0.0}
TOL = {t: 2e-5 + u for t, u in UNIT.items()}


def near(got, ref, dtype=None):
    tol = TOL[dtype or got.dtype]
    got, ref = got.double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    off, norm = (got - ref).norm().item(), ref.norm().item()
    assert off <= tol * norm, f"{off / max(norm, 1e-300):.3g} off, {tol:.3g} allowed"


def gates(g, beta, A_log=None, dt_bias=None):
    g, beta = g.double(), beta.double()
    if A_log is not None:
        x = g + dt_bias.double()
        g = -A_log.double().exp() * (x.clamp_min(0) + torch.log1p((-x.abs()).exp()))
        beta = 1 / (1 + (-beta).exp())
    return g, beta


def rule(q, k, v, g, beta, S, scale, l2norm, record=None):
    """One sequence, token by token, in 64 bits: q, k (T, HK, dk), v (T, HV, dv), S (HV, dk, dv)."""
    q, k, v = q.double(), k.double(), v.double()
    if l2norm:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    S = S.double().clone()
    out = torch.empty(v.shape, dtype=torch.float64)
    for t in range(v.shape[0]):
        S = S * g[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
        S = S + k[t][:, :, None] * u[:, None, :]
        out[t] = scale * torch.einsum("hkv,hk->hv", S, q[t])
        if record is not None:
            record.append(S.clone())
    return out, S


def make(T, hk, hv, dk, dv, dtype, raw=True, seed=0, unit=False):
    """Inputs on the CPU; q, k, v are column views of one row, as the conv hands them over."""
    r = torch.Generator().manual_seed(seed)
    x = torch.randn(T, 2 * hk * dk + hv * dv, generator=r)
    if unit:  # keys of unit length for calls without the l2 norm
        kk = x[:, hk * dk : 2 * hk * dk].view(T, hk, dk)
        kk /= kk.norm(dim=-1, keepdim=True)
    x = x.to(dtype)
    q, k, v = x.split([hk * dk, hk * dk, hv * dv], 1)
    q, k, v = q.view(T, hk, dk), k.view(T, hk, dk), v.view(T, hv, dv)
    if raw:
        g = torch.randn(T, hv, generator=r).to(dtype)
        b = torch.randn(T, hv, generator=r).to(dtype)
        A = torch.empty(hv).uniform_(0.05, 16, generator=r).log()
        dt = torch.randn(hv, generator=r) - 3
        return q, k, v, g, b, A, dt
    g = -torch.rand(T, hv, generator=r) * 0.5
    b = torch.rand(T, hv, generator=r)
    return q, k, v, g, b, None, None


def gpu(t):
    """To the GPU with the same strides."""
    if t is None:
        return None
    d = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda")
    return d.copy_(t)


def varlen_case(lengths, hk=2, hv=6, dk=128, dv=128, dtype=BF, sdtype=F32, raw=True, l2norm=True,
                states=True, scale=None, seed=0, pad=None, change=None):
    """Run the packed prefill and compare outputs and the whole cache with the definition."""
    T, n = sum(lengths), len(lengths)
    q, k, v, g, b, A, dt = make(T, hk, hv, dk, dv, dtype, raw, seed, unit=not l2norm)
    if change is not None:
        change(q, k, v, g, b)
    r = torch.Generator().manual_seed(seed + 1)
    cache = torch.randn(n + 2, hv, dk, dv, generator=r).mul(0.3).to(sdtype) if states else None
    idx = torch.randperm(n + 2, generator=r)[:n].int()
    if pad is not None:
        idx[pad] = -1
    hinit = torch.rand(n, generator=r) < 0.6
    start = torch.tensor([0] + list(itertools.accumulate(lengths)), dtype=torch.int32)
    gg, bb = gates(g, b, A, dt)
    want, want_cache = torch.zeros(T, hv, dv, dtype=torch.float64), None if cache is None else cache.double().clone()
    sc = dk**-0.5 if scale is None else scale
    for i, L in enumerate(lengths):
        if L == 0 or (states and idx[i] < 0):
            continue
        s = slice(int(start[i]), int(start[i + 1]))
        S0 = torch.zeros(hv, dk, dv)
        if states and hinit[i]:
            S0 = cache[idx[i]]
        want[s], S = rule(q[s], k[s], v[s], gg[s], bb[s], S0, sc, l2norm)
        if states:
            want_cache[idx[i]] = S
    dc = gpu(cache)
    got = C.gated_delta_rule_varlen_fn(
        gpu(q), gpu(k), gpu(v), gpu(g), gpu(b), start.cuda(), idx.cuda() if states else None,
        hinit.cuda() if states else None, dc, A_log=gpu(A), dt_bias=gpu(dt), scale=scale, qk_l2norm=l2norm)
    if pad is not None:
        s = slice(int(start[pad]), int(start[pad + 1]))
        got[s] = 0
    near(got, want)
    if states:
        near(dc, want_cache)
        # untouched slots, bit for bit
        used = {int(idx[i]) for i, L in enumerate(lengths) if L and idx[i] >= 0}
        for s in set(range(n + 2)) - used:
            assert torch.equal(dc[s].cpu(), cache[s])
    return got, dc


# ------------------------------------------------------------------------------------------ host


def test_shape_errors():
    q, k, v, g, b, A, dt = make(5, 2, 4, 16, 16, F32)
    qsl = torch.tensor([0, 5], dtype=torch.int32)
    st = torch.zeros(1, 4, 16, 16)
    bad = [
        dict(k=k[:, :, :8]), dict(v=v[:, :3]), dict(g=g[:, :2]), dict(beta=b[:4]), dict(A_log=None),
        dict(dt_bias=dt[:2]), dict(states=st[:, :, :8]), dict(states=st[0]), dict(query_start_loc=None),
        dict(cache_indices=torch.zeros(2, dtype=torch.int32)), dict(has_initial_state=torch.zeros(2)),
        dict(q=q[0], k=k[0]),
    ]
    for change in bad:
        args = dict(q=q, k=k, v=v, g=g, beta=b, query_start_loc=qsl, states=st, A_log=A, dt_bias=dt)
        args.update(change)
        with pytest.raises(ValueError):
            C.gated_delta_rule_varlen_fn(**args)
    with pytest.raises(ValueError):
        C.gated_delta_rule_update(q, k, v, g, b, st[:, :3], A_log=A, dt_bias=dt)
    with pytest.raises(ValueError):
        C.gated_delta_rule_update(q, k, v, g, b, torch.zeros(5, 4, 16, 16), torch.zeros(3), A_log=A, dt_bias=dt)
    with pytest.raises(ValueError):
        C.gated_delta_rule_update(q, k, v, g, b, torch.zeros(5, 4, 16, 16), intermediate_states=torch.zeros(5, 2, 4, 16, 16),
                                  A_log=A, dt_bias=dt)
    with pytest.raises(ValueError):
        C.gated_delta_rule_fn(q, k, v, g, b)
    with pytest.raises(ValueError):
        C.rms_norm_gated(v, v[:, :2], torch.ones(16))
    with pytest.raises(ValueError):
        C.rms_norm_gated(v, v, torch.ones(8))


def test_no_cpu_fallback_and_no_gradients():
    q, k, v, g, b, A, dt = make(5, 2, 4, 16, 16, F32)
    qsl = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(C.Unsupported, match="not a CUDA tensor"):
        C.gated_delta_rule_varlen_fn(q, k, v, g, b, qsl, A_log=A, dt_bias=dt)
    with pytest.raises(C.Unsupported, match="not a CUDA tensor"):
        C.gated_delta_rule_update(q, k, v, g, b, torch.zeros(5, 4, 16, 16), A_log=A, dt_bias=dt)
    with pytest.raises(C.Unsupported, match="not a CUDA tensor"):
        C.gated_delta_rule_fn(*(t[None] for t in (q, k, v, g, b)), A_log=A, dt_bias=dt)
    with pytest.raises(C.Unsupported):
        C.rms_norm_gated(v, v, torch.ones(16))
    assert "gradients" in G.gated_delta_rule_reason(q.clone().requires_grad_(), k, v, g, b)
    assert "backward" in G.gated_delta_rule_reason(q, k, v, g, b, None, A.clone().requires_grad_(), dt)
    with pytest.raises(C.Unsupported, match="backward"):
        C.rms_norm_gated(v.clone().requires_grad_(), v, torch.ones(16))


def test_c_abi_refuses_before_launch():
    lib = _lib.load()

    def block(**kw):
        """An argument block with made-up pointers; everything refused here is refused on the host."""
        f = dict(dict(states=1, nslots=4, rows=2, tokens=8, steps=1, hk=2, hv=4, dk=16, dv=16, dtype=2, sdtype=2,
                      a_log=0, dt=0, q=1, inter=0), **kw)
        return _lib.GDR_ARGS.pack(f["q"], 1, 1, 1, 1, f["a_log"], f["dt"], 1, f["states"], f["inter"], 0, 0, 1, 0, 0, 0,
                                  *[0] * 29, f["rows"], f["tokens"], f["nslots"], 0, 0, f["steps"], f["hk"], f["hv"],
                                  f["dk"], f["dv"], f["dtype"], 2, 2, 2, f["sdtype"], 0, 1, -1, 1.0)

    up, var = lib.cc1d_gdr_update, lib.cc1d_gdr_varlen
    assert up(None, None) == 1 and var(None, None) == 1
    assert up(block(dtype=7), None) == 2
    assert up(block(dtype=0, sdtype=1), None) == 2
    assert up(block(hv=3), None) == 1
    assert up(block(dk=257), None) == 1
    assert up(block(dk=0), None) == 1
    assert up(block(steps=0), None) == 1
    assert up(block(a_log=1), None) == 1
    assert up(block(q=0), None) == 1
    assert up(block(rows=5), None) == 1 and b"slots" in lib.cc1d_last_error()
    assert up(block(rows=0), None) == 0
    assert var(block(tokens=2**31), None) == 1
    assert var(block(inter=1), None) == 1
    assert var(block(tokens=0), None) == 0

    def norm(dtype=0, wdtype=2, n0=1, dim=8, x=1):
        return _lib.NORM_ARGS.pack(x, 0, 1, 1, *[8] * 6, n0, 1, dim, dtype, wdtype, 1e-6)

    f = lib.cc1d_rms_norm_gated
    assert f(None, None) == 1 and f(norm(dtype=5), None) == 2 and f(norm(wdtype=1), None) == 2
    assert f(norm(dim=0), None) == 1 and f(norm(x=0), None) == 1 and f(norm(n0=0), None) == 0


def test_schemas_mark_what_is_written():
    written = {
        "gdr_update": {"out", "states", "inter"}, "gdr_varlen": {"out", "states"}, "rms_norm_gated": {"out"},
        "slots_copy": {"caches"}, "slots_compact": {"caches", "remap", "count", "moves"},
    }
    for name, names in written.items():
        schema = getattr(torch.ops.cc1d, name).default._schema
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == names


# --------------------------------------------------------------------------------------- prefill


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (BF, BF), (F16, F32), (F16, F16), (F32, F32)])
def test_varlen_lengths(dtype, sdtype):
    """Every length around a chunk of 64 and a tile of 4 tokens, empty sequences among them."""
    varlen_case([1, 0, 2, 63, 64, 65, 0, 3, 128, 5, 200, 127, 4, 129], dtype=dtype, sdtype=sdtype)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1], [64], [65], [700], [0, 0, 300, 0], [1] * 40, [17, 330]])
def test_varlen_batches(lengths):
    varlen_case(lengths, seed=len(lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [13, 25, 60, 300])
@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (BF, BF), (F16, F32), (F16, F16)])
def test_varlen_many_sequences(n, dtype, sdtype):
    """Enough (sequence, head) pairs to fill the GPU with each width of a work tile; uneven lengths."""
    r = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 150, (n,), generator=r).tolist()
    varlen_case(lengths, hk=1, hv=6, dtype=dtype, sdtype=sdtype, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 3), (2, 2), (4, 8), (3, 6)])
def test_varlen_head_groups(hk, hv):
    varlen_case([100, 31, 70], hk=hk, hv=hv, seed=hk)


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 64), (64, 128), (128, 256), (256, 128), (96, 80), (1, 1), (7, 9), (200, 33), (128, 130)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_varlen_head_dims(dk, dv, dtype):
    varlen_case([70, 1, 90], hk=1, hv=2, dk=dk, dv=dv, dtype=dtype, seed=dk)


@pytest.mark.gpu
@pytest.mark.parametrize("raw,l2norm,scale", [(False, False, None), (False, True, 0.5), (True, False, 1.0)])
def test_varlen_options(raw, l2norm, scale):
    varlen_case([150, 66], raw=raw, l2norm=l2norm, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_varlen_without_cache(dtype):
    varlen_case([150, 3, 66], states=False, dtype=dtype)


@pytest.mark.gpu
def test_varlen_pad_slot_is_skipped():
    varlen_case([80, 70, 65], pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_varlen_strong_and_total_decay(dtype):
    """Log decays of 0, very large ones and -inf (which clears the state), beta of 0 and 1."""

    def change(q, k, v, g, b):
        g[10:20] = -200.0
        g[40] = -float("inf")
        g[64] = -float("inf")
        g[90:140] = 0.0
        g[150:152] = -1e30
        b[30:40] = 0.0
        b[100:110] = 1.0

    varlen_case([230, 70], raw=False, change=change, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_varlen_sequences_do_not_see_each_other(bad, dtype):
    """Values that are not finite in one sequence stay in it, tails of its chunks included."""
    lengths = [70, 33, 129, 64]
    T = sum(lengths)
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, 2, 4, 128, 128, dtype))
    start = torch.tensor([0] + list(itertools.accumulate(lengths)), dtype=torch.int32)
    st = torch.randn(4, 4, 128, 128, device="cuda")
    hinit = torch.ones(4, dtype=torch.bool, device="cuda")

    def run():
        s = st.clone()
        o = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start.cuda(), None, hinit, s, A_log=A, dt_bias=dt, qk_l2norm=True)
        return o, s

    o0, s0 = run()
    q[70:103] = bad
    k[70:103] = bad
    v[70:103] = bad
    st[1] = bad
    o1, s1 = run()
    keep = torch.ones(T, dtype=torch.bool)
    keep[70:103] = False
    assert torch.equal(o0[keep.cuda()], o1[keep.cuda()])
    for i in (0, 2, 3):
        assert torch.equal(s0[i], s1[i])
    assert not torch.isfinite(o1[70:103].float()).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (F16, F16)])
@pytest.mark.parametrize("dv,states,raw,pad", [(128, True, False, 3), (256, True, True, None), (128, False, True, None)])
def test_varlen_wide_tiles(dtype, sdtype, dv, states, raw, pad):
    """Batches with work for the widest tile: several tiles of a head, made gates, no cache, a pad."""
    varlen_case([65, 1, 0, 130, 64, 3, 20, 97], hk=20, hv=40, dv=dv, dtype=dtype, sdtype=sdtype, states=states, raw=raw,
                pad=pad, seed=dv)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_varlen_wide_tiles_do_not_see_each_other(bad, dtype):
    """The same as above for one sequence among many heads; the outputs of the others bit for bit."""
    lengths = [70, 33, 129, 64, 1, 90, 15, 66]
    T, n, hv = sum(lengths), len(lengths), 40
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, 20, hv, 128, 128, dtype))
    start = torch.tensor([0] + list(itertools.accumulate(lengths)), dtype=torch.int32).cuda()
    st = torch.randn(n, hv, 128, 128, device="cuda")
    hinit = torch.ones(n, dtype=torch.bool, device="cuda")

    def run():
        s = st.clone()
        o = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, hinit, s, A_log=A, dt_bias=dt, qk_l2norm=True)
        return o, s

    o0, s0 = run()
    for x in (q, k, v):
        x[70:103] = bad
    st[1] = bad
    o1, s1 = run()
    assert torch.equal(o0[:70], o1[:70]) and torch.equal(o0[103:], o1[103:])
    for i in (0, *range(2, n)):
        assert torch.equal(s0[i], s1[i])
    assert not torch.isfinite(o1[70:103].float()).any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_varlen_later_tokens_do_not_reach_back(bad):
    """A value that is not finite shows from its own token on, and in no chunk of 64 before."""
    T = 150
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, 1, 2, 128, 128, BF))
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    args = dict(A_log=A, dt_bias=dt, qk_l2norm=True)
    o0 = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, **args)
    v[101] = bad
    o1 = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, **args)
    assert torch.equal(o0[:64], o1[:64])
    assert not torch.isfinite(o1[101:].float()).any()


@pytest.mark.gpu
def test_varlen_strides_and_out():
    """Heads before tokens, an inner stride of 2, gates of another dtype and order, a given output."""
    T, hk, hv, d = 140, 2, 4, 128
    q, k, v, g, b, A, dt = make(T, hk, hv, d, d, BF)
    gg, bb = gates(g, b, A, dt)
    want, S = rule(q, k, v, gg, bb, torch.zeros(hv, d, d), d**-0.5, True)
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    layouts = [
        lambda t: gpu(t.transpose(0, 1).contiguous().transpose(0, 1)),
        lambda t: gpu(torch.stack([t, t], -1)[..., 0]),
        lambda t: gpu(torch.cat([t[:, :, :1], t], -1)[..., 1:]),  # rows off 16-byte boundaries
    ]
    for lay in layouts:
        out = torch.full((T, hv, 2 * d), 7.0, device="cuda", dtype=BF)
        st = torch.zeros(1, hv, d, d, device="cuda")
        got = C.gated_delta_rule_varlen_fn(
            lay(q), lay(k), lay(v), gpu(g.t().contiguous().t()), gpu(b.float()), start, None, None, st,
            A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=True, out=out[..., :d])
        near(got, want)
        near(st[0], S)
        assert (out[..., d:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [lambda s: (s[0], s[1] + 1, s[2], s[3]), lambda s: (s[0], s[1], s[2], s[3] + 3)])
def test_varlen_strided_cache(shape):
    """A cache that is a view of a wider one, with aligned and with unaligned rows."""
    T, hk, hv, d = 100, 1, 2, 128
    q, k, v, g, b, A, dt = make(T, hk, hv, d, d, BF)
    whole = torch.randn(shape((3, hv, d, d)))
    gg, bb = gates(g, b, A, dt)
    want, S = rule(q, k, v, gg, bb, whole[1, :hv, :, :d], d**-0.5, True)
    dev = whole.cuda()
    view = dev[:, :hv, :, :d]
    got = C.gated_delta_rule_varlen_fn(
        gpu(q), gpu(k), gpu(v), gpu(g), gpu(b), torch.tensor([0, T], dtype=torch.int32, device="cuda"),
        torch.tensor([1], dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.bool, device="cuda"), view,
        A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=True)
    near(got, want)
    near(view[1], S)
    dev[1, :hv, :, :d] = whole[1, :hv, :, :d].cuda()
    assert torch.equal(dev.cpu(), whole)


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [1, 500_000, 1_300_000])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_varlen_in_groups_of_heads(monkeypatch, limit, dtype):
    """A workspace above its limit: the heads in groups, uneven ones too, bit for bit the same."""
    from causal_conv1d_cute import _ops

    lengths = [100, 65, 3]
    q, k, v, g, b, A, dt = (gpu(t) for t in make(sum(lengths), 5, 10, 128, 128, dtype))
    start = torch.tensor([0] + list(itertools.accumulate(lengths)), dtype=torch.int32, device="cuda")

    def run():
        s = torch.ones(3, 10, 128, 128, device="cuda")
        hinit = torch.ones(3, dtype=torch.bool, device="cuda")
        return C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, hinit, s, A_log=A, dt_bias=dt, qk_l2norm=True), s

    o0, s0 = run()
    monkeypatch.setattr(_ops, "_GDR_WORKSPACE", limit)
    o1, s1 = run()
    assert torch.equal(o0, o1) and torch.equal(s0, s1)


@pytest.mark.gpu
def test_strided_index_tensors():
    q, k, v, g, b, A, dt = (gpu(t) for t in make(130, 1, 2, 128, 128, BF))
    kw = dict(A_log=A, dt_bias=dt, qk_l2norm=True)
    wide = lambda x, t: torch.stack([torch.tensor(x, dtype=t), torch.full((len(x),), 7, dtype=t)], 1).cuda()[:, 0]  # noqa: E731
    i32 = torch.int32
    a, s = [], []
    for view in (lambda t: t, lambda t: t.contiguous()):
        st = torch.ones(4, 2, 128, 128, device="cuda")
        a.append(C.gated_delta_rule_varlen_fn(q, k, v, g, b, view(wide([0, 70, 130], i32)), view(wide([3, 0], i32)),
                                              view(wide([1, 0], torch.uint8)), st, **kw))
        a.append(C.gated_delta_rule_update(q[:2], k[:2], v[:2], g[:2], b[:2], st, view(wide([2, 3], i32)), **kw))
        s.append(st)
    assert torch.equal(a[0], a[2]) and torch.equal(a[1], a[3]) and torch.equal(s[0], s[1])


@pytest.mark.gpu
def test_varlen_bad_indices_are_skipped_and_reported(request):
    request.node._expect_status = True
    lengths = [65, 66, 67]
    q, k, v, g, b, A, dt = (gpu(t) for t in make(sum(lengths), 1, 2, 128, 128, BF))
    st = torch.randn(3, 2, 128, 128, device="cuda")
    before = st.clone()
    qsl = torch.tensor([0, 65, 131, 198], dtype=torch.int32, device="cuda")
    idx = torch.tensor([0, 3, 2], dtype=torch.int32, device="cuda")
    C.gated_delta_rule_varlen_fn(q, k, v, g, b, qsl, idx, None, st, A_log=A, dt_bias=dt, qk_l2norm=True)
    assert C.device_status() == _lib.DEV_BAD_SLOT
    assert torch.equal(st[1], before[1]) and not torch.equal(st[0], before[0])
    st = before.clone()
    qsl[2] = 50
    qsl[3] = 199
    C.gated_delta_rule_varlen_fn(q, k, v, g, b, qsl, None, None, st, A_log=A, dt_bias=dt, qk_l2norm=True)
    assert C.device_status() == _lib.DEV_BAD_QSL
    assert torch.equal(st[1:], before[1:]) and not torch.equal(st[0], before[0])


@pytest.mark.gpu
def test_varlen_repeats_bit_for_bit_and_on_a_side_stream():
    lengths = [300, 77, 512]
    q, k, v, g, b, A, dt = (gpu(t) for t in make(sum(lengths), 2, 6, 128, 128, BF))
    start = torch.tensor([0] + list(itertools.accumulate(lengths)), dtype=torch.int32, device="cuda")

    def run():
        s = torch.zeros(3, 6, 128, 128, device="cuda")
        return C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, None, s, A_log=A, dt_bias=dt, qk_l2norm=True), s

    o0, s0 = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o1, s1 = run()
    side.synchronize()
    assert torch.equal(o0, o1) and torch.equal(s0, s1)


@pytest.mark.gpu
def test_prefill_in_pieces_equals_prefill_at_once():
    """A prompt cut at any place, its state carried in the cache, gives the same rows."""
    T = 330
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, 1, 3, 128, 128, BF))
    one = torch.zeros(1, 3, 128, 128, device="cuda")
    kw = dict(A_log=A, dt_bias=dt, qk_l2norm=True)
    at = lambda x: torch.tensor([0, x], dtype=torch.int32, device="cuda")  # noqa: E731
    want = C.gated_delta_rule_varlen_fn(q, k, v, g, b, at(T), None, None, one, **kw)
    two, got = torch.zeros_like(one), []
    first = 0
    for n in (64, 1, 100, 165):
        s = slice(first, first + n)
        got.append(C.gated_delta_rule_varlen_fn(q[s], k[s], v[s], g[s], b[s], at(n), None,
                                                torch.tensor([first > 0], device="cuda"), two, **kw))
        first += n
    near(torch.cat(got), want.double())
    near(two, one.double())


@pytest.mark.gpu
@pytest.mark.parametrize("B,L", [(3, 130), (2, 1), (1, 64), (2, 0), (0, 5)])
@pytest.mark.parametrize("initial", [False, True])
def test_dense_prefill(B, L, initial):
    hk, hv, d = 2, 4, 128
    q, k, v, g, b, A, dt = make(max(B * L, 1), hk, hv, d, d, BF)
    q, k, v, g, b = (t[: B * L].unflatten(0, (B, L)) for t in (q, k, v, g, b))
    S0 = torch.randn(B, hv, d, d) * 0.3
    gg, bb = gates(g, b, A, dt)
    want = [rule(q[i], k[i], v[i], gg[i], bb[i], S0[i] if initial else torch.zeros(hv, d, d), d**-0.5, True) for i in range(B)]
    dS = gpu(S0)
    got, fin = C.gated_delta_rule_fn(gpu(q), gpu(k), gpu(v), gpu(g), gpu(b), dS if initial else None, True,
                                     A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=True)
    assert got.shape == (B, L, hv, d) and fin.shape == (B, hv, d, d) and fin.dtype == F32
    assert torch.equal(dS.cpu(), S0)
    if B:
        near(got, torch.stack([w[0] for w in want]))
        near(fin, torch.stack([w[1] for w in want]))
    if B * L:
        alone = C.gated_delta_rule_fn(gpu(q), gpu(k), gpu(v), gpu(g), gpu(b), dS if initial else None,
                                      A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=True)
        assert torch.equal(alone, got)


# ---------------------------------------------------------------------------------------- decode


def update_case(B, steps, hk, hv, dk, dv, dtype, sdtype, raw=True, l2norm=True, record=False, update=True,
                pads=(), single=False, seed=0):
    q, k, v, g, b, A, dt = make(B * steps, hk, hv, dk, dv, dtype, raw, seed, unit=not l2norm)
    q, k, v, g, b = (t.unflatten(0, (B, steps)) for t in (q, k, v, g, b))
    r = torch.Generator().manual_seed(seed + 7)
    slots = B + 3
    st = torch.randn(slots, hv, dk, dv, generator=r).mul(0.3).to(sdtype)
    idx = torch.randperm(slots, generator=r)[:B].int()
    for p in pads:
        idx[p] = -1
    inter = torch.full((B + 1, steps, hv, dk, dv), 3.0).to(sdtype) if record else None
    iidx = torch.randperm(B + 1, generator=r)[:B].int() if record else None
    gg, bb = gates(g, b, A, dt)
    want, want_st = torch.zeros(v.shape, dtype=torch.float64), st.double().clone()
    want_in = inter.double().clone() if record else None
    for i in range(B):
        if idx[i] < 0:
            continue
        rec = []
        want[i], S = rule(q[i], k[i], v[i], gg[i], bb[i], st[idx[i]], dk**-0.5, l2norm, rec)
        if update:
            want_st[idx[i]] = S
        if record:
            want_in[iidx[i]] = torch.stack(rec)
    args = [gpu(t[:, 0] if single else t) for t in (q, k, v, g, b)]
    ds, di = gpu(st), gpu(inter)
    got = C.gated_delta_rule_update(
        *args, ds, idx.cuda(), A_log=gpu(A), dt_bias=gpu(dt), qk_l2norm=l2norm, intermediate_states=di,
        intermediate_state_indices=None if iidx is None else iidx.cuda(), update_states=update)
    got = got.unsqueeze(1) if single else got
    live = idx >= 0
    near(got.cpu()[live], want[live])
    near(ds, want_st)
    untouched = sorted(set(range(slots)) - set(idx[live].tolist())) if update else list(range(slots))
    assert torch.equal(ds.cpu()[untouched], st[untouched])
    if record:
        near(di, want_in)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,sdtype", [(BF, F32), (BF, BF), (F16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("single", [True, False])
def test_update_types(dtype, sdtype, single):
    update_case(5, 1, 2, 6, 128, 128, dtype, sdtype, single=single)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [2, 3, 4, 5, 8, 16])
@pytest.mark.parametrize("record,update", [(True, True), (True, False), (False, True)])
def test_update_steps(steps, record, update):
    update_case(3, steps, 1, 3, 128, 128, BF, F32, record=record, update=update, seed=steps)


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 256), (256, 256), (96, 80), (1, 1), (7, 9), (200, 33), (128, 130)])
def test_update_head_dims(dk, dv):
    update_case(3, 2, 1, 2, dk, dv, BF, F32, record=True, seed=dk)
    update_case(3, 1, 1, 2, dk, dv, F16, F16, seed=dv)


@pytest.mark.gpu
@pytest.mark.parametrize("raw,l2norm", [(False, False), (False, True), (True, False)])
def test_update_options(raw, l2norm):
    update_case(4, 3, 2, 4, 128, 128, BF, F32, raw=raw, l2norm=l2norm)


@pytest.mark.gpu
def test_update_pad_rows():
    update_case(6, 2, 1, 2, 128, 128, BF, F32, record=True, pads=(0, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 33, 130])
def test_update_batches(B):
    update_case(B, 1, 1, 3, 128, 128, BF, F32, seed=B)


@pytest.mark.gpu
def test_update_bad_slot_is_skipped_and_reported(request):
    request.node._expect_status = True
    q, k, v, g, b, A, dt = (gpu(t) for t in make(3, 1, 2, 128, 128, BF))
    st = torch.randn(3, 2, 128, 128, device="cuda")
    before = st.clone()
    inter = torch.zeros(2, 1, 2, 128, 128, device="cuda")
    C.gated_delta_rule_update(q, k, v, g, b, st, torch.tensor([0, 3, -7], dtype=torch.int32, device="cuda"),
                              A_log=A, dt_bias=dt, qk_l2norm=True)
    assert C.device_status() == _lib.DEV_BAD_SLOT
    assert torch.equal(st[1:], before[1:]) and not torch.equal(st[0], before[0])
    C.gated_delta_rule_update(q, k, v, g, b, st, A_log=A, dt_bias=dt, qk_l2norm=True, intermediate_states=inter)
    assert C.device_status() == _lib.DEV_BAD_INTER_SLOT


@pytest.mark.gpu
def test_update_of_infinite_decay_clears_the_state():
    q, k, v, g, b, _, _ = (gpu(t) for t in make(2, 1, 2, 128, 128, F32, raw=False))
    g[0] = -float("inf")
    st = torch.randn(2, 2, 128, 128, device="cuda")
    C.gated_delta_rule_update(q, k, v, g, b, st, qk_l2norm=True)
    kk = k[0, 0] / (k[0, 0].square().sum() + 1e-6).sqrt()
    near(st[0], torch.einsum("k,hv->hkv", kk.double(), (b[0, :, None] * v[0]).double()))


@pytest.mark.gpu
def test_decode_equals_prefill():
    """Tokens one at a time, in steps of 16 and as one packed sequence agree."""
    T, hk, hv, d = 48, 1, 3, 128
    q, k, v, g, b, A, dt = (gpu(t) for t in make(T, hk, hv, d, d, F32))
    kw = dict(A_log=A, dt_bias=dt, qk_l2norm=True)
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    s0, s1, s2 = (torch.zeros(1, hv, d, d, device="cuda") for _ in range(3))
    want = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, None, s0, **kw)
    one = [C.gated_delta_rule_update(*(t[i : i + 1] for t in (q, k, v, g, b)), s1, **kw) for i in range(T)]
    many = [C.gated_delta_rule_update(*(t[i : i + 16][None] for t in (q, k, v, g, b)), s2, **kw) for i in range(0, T, 16)]
    near(torch.cat(one), want.double())
    near(torch.cat(many, 1)[0], want.double())
    near(s1, s0.double())
    near(s2, s0.double())


@pytest.mark.gpu
def test_calls_in_a_graph():
    q, k, v, g, b, A, dt = (gpu(t) for t in make(130, 1, 3, 128, 128, BF))
    start = torch.tensor([0, 100, 130], dtype=torch.int32, device="cuda")
    st, sd = torch.zeros(2, 3, 128, 128, device="cuda"), torch.zeros(130, 3, 128, 128, device="cuda")
    w = torch.ones(128, device="cuda")
    kw = dict(A_log=A, dt_bias=dt, qk_l2norm=True)

    def step():
        o = C.gated_delta_rule_varlen_fn(q, k, v, g, b, start, None, None, st, **kw)
        return C.rms_norm_gated(o, v, w), C.gated_delta_rule_update(q, k, v, g, b, sd, **kw)

    want = [t.clone() for t in step()]
    sd.zero_()
    st.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        sd.zero_()
        st.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------ norm


def norm_ref(x, z, w, eps):
    x, w = x.double(), w.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    return y if z is None else y * z.double() / (1 + (-z.double()).exp())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("shape", [(1, 128), (5, 3, 128), (7, 64), (3, 2, 256), (2, 5, 512), (4, 1000), (3, 1024), (2, 2304),
                                   (3, 1), (5, 7), (6, 130), (0, 4, 128), (2, 3, 4, 128), (128,), (257, 6, 128)])
@pytest.mark.parametrize("gate", [True, False])
def test_norm(dtype, shape, gate):
    r = torch.Generator().manual_seed(3)
    x, z = (torch.randn(shape, generator=r).to(dtype) for _ in range(2))
    w = torch.rand(shape[-1], generator=r) + 0.5
    for wd in {F32, dtype}:
        got = C.rms_norm_gated(x.cuda(), z.cuda() if gate else None, w.to(wd).cuda(), 1e-5)
        near(got, norm_ref(x, z if gate else None, w.to(wd), 1e-5))


@pytest.mark.gpu
def test_norm_strides_and_in_place():
    r = torch.Generator().manual_seed(4)
    rows = torch.randn(20, 2 * 6 * 128 + 4, generator=r).to(BF)
    w = torch.rand(128, generator=r)
    x, z = rows[:, :768].unflatten(1, (6, 128)), rows[:, 768:1536].unflatten(1, (6, 128))
    ref = norm_ref(x, z, w, 1e-6)
    d = rows.cuda()
    dx, dz = d[:, :768].unflatten(1, (6, 128)), d[:, 768:1536].unflatten(1, (6, 128))
    near(C.rms_norm_gated(dx, dz, w.cuda()), ref)
    odd = torch.empty(20, 1, 6, 129, dtype=BF, device="cuda")[..., 1:]
    near(C.rms_norm_gated(dx[:, None], dz[:, None], w.cuda(), out=odd), ref[:, None])
    t = torch.randn(128, 6, generator=r).to(BF)
    near(C.rms_norm_gated(t.cuda().t(), None, w.cuda()), norm_ref(t.t(), None, w, 1e-6))
    assert C.rms_norm_gated(dx, dz, w.cuda(), out=dx) is dx
    near(dx, ref)
    assert torch.equal(d[:, 768:].cpu(), rows[:, 768:])


@pytest.mark.gpu
def test_norm_extremes():
    """Zero rows give zeros; gates far out saturate; large values do not overflow in fp32."""
    x = torch.zeros(4, 128, device="cuda")
    x[1] = 1e15
    x[2] = -3.0
    x[3] = 1e-20
    z = torch.full((4, 128), 200.0, device="cuda")
    z[2] = -200.0
    w = torch.ones(128, device="cuda")
    got = C.rms_norm_gated(x, z, w, 1e-6).cpu()
    assert torch.equal(got[0], torch.zeros(128))
    near(got, norm_ref(x.cpu(), z.cpu(), w.cpu(), 1e-6))
    b = C.rms_norm_gated(x.to(BF), z.to(BF), w, 1e-6).cpu()
    assert torch.isfinite(b).all() and (b[2] == 0).all() and (b[1] == 200).all()
