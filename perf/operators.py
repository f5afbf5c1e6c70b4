"""Cases for the operators of a Gated DeltaNet layer behind its causal conv: the gated delta rule
(packed chunked prefill, recurrent decode), the gated RMS norm, and the slot moves of the state caches.

Head counts are the serving shape that bench.py times for the fused decode (16 query/key heads and
48 value heads of 128, conv rows of 10240 = 2 * 16 * 128 + 48 * 128 columns) and its tensor-parallel
slices. q, k and v are column views of the conv's output rows, and the gates are raw projections, as
the conv + unpack step hands them over.

With `own` false, run() computes each operator in plain fp32 torch; with `own` true it calls the
package.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

D = 128  # head dim of keys and values
CHUNK = 64  # chunk of the plain prefill
L2_EPS = 1e-6
NORM_EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    """The package lives in a folder whose name is no Python identifier; it is imported by path."""
    root = str(Path(__file__).resolve().parent.parent / "causal-conv1d-cute_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import causal_conv1d_cute

    return causal_conv1d_cute


# ------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # The last pieces of four prompts on one of eight tensor-parallel ranks: latency counts.
        dict(name="prefill-tails", op="prefill", tokens=61, seqs=4, hk=2, dtype="bf16", state="f32", initial=True),
        # One long prompt on one of four ranks: 12 heads, a long chain over few rows.
        dict(name="prefill-one-long", op="prefill", tokens=8192, seqs=1, hk=4, dtype="bf16", state="f32", initial=False),
        # A packed batch of the size of the packed conv benchmark: 32 prompts of uneven length, all heads.
        dict(name="prefill-packed", op="prefill", tokens=40807, seqs=32, hk=16, dtype="bf16", state="f32", initial=True),
        # One user's decode step on one of eight ranks: the smallest call.
        dict(name="decode-one", op="decode", rows=1, steps=1, slots=16, hk=2, dtype="bf16", state="f32", record=False),
        # The serving decode batch of the fused conv + unpack benchmark.
        dict(name="decode-256", op="decode", rows=256, steps=1, slots=310, hk=16, dtype="bf16", state="f32", record=False),
        # Verification of four drafted tokens, the state after each step kept.
        dict(name="verify-4", op="decode", rows=37, steps=4, slots=64, hk=16, dtype="f16", state="f16", record=True),
        # Output norm of a decode batch, and of a packed prefill.
        dict(name="norm-decode", op="norm", tokens=64, heads=48, dtype="bf16"),
        dict(name="norm-prefill", op="norm", tokens=40807, heads=48, dtype="bf16"),
        # A prompt's state forked to three continuations on one of eight ranks; two slots freed.
        dict(name="slots-fork", op="copy", layers=12, slots=24, pairs=5, freed=2, hk=2, dtype="bf16", state="f32"),
        # Many slots at once, all heads.
        dict(name="slots-copy", op="copy", layers=6, slots=96, pairs=40, freed=3, hk=16, dtype="bf16", state="f32"),
        # Live slots moved to the front after a third of the requests ended, on one of four ranks; and a
        # larger cache of one of two ranks.
        dict(name="slots-compact-few", op="compact", layers=4, slots=13, live=8, moves=3, hk=4, dtype="bf16", state="f32"),
        dict(name="slots-compact", op="compact", layers=12, slots=97, live=64, moves=21, hk=8, dtype="bf16", state="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "decode", "norm", "copy", "compact"])
    hk = rng.choice([1, 2, 4, 8, 16])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    state = rng.choice(["f32", "f32", dtype])
    if op == "prefill":
        tokens = _log_int(rng, 16, 40000)
        seqs = min(_log_int(rng, 1, 32), max(1, tokens // 4))
        if tokens > 12000:
            seqs = max(seqs, 4)  # no longer chain than the listed cases have
        return dict(op=op, tokens=tokens, seqs=seqs, hk=hk, dtype=dtype, state=state, initial=rng.random() < 0.5)
    if op == "decode":
        steps = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
        rows = _log_int(rng, 1, max(1, 250 // (2 * steps) if steps > 1 else 250))
        return dict(op=op, rows=rows, steps=steps, slots=rows + rng.randint(0, 40), hk=hk, dtype=dtype, state=state,
                    record=steps > 1 and rng.random() < 0.7)
    if op == "norm":
        return dict(op=op, tokens=_log_int(rng, 1, 40000), heads=3 * hk, dtype=dtype)
    layers = rng.randint(1, 12)
    if op == "copy":
        pairs = _log_int(rng, 1, 36)
        freed = rng.randint(0, pairs // 3)
        slots = 2 * pairs + rng.randint(1, 16)
        layers = max(1, min(layers, 480 // (slots * hk // 4 + 1)))
        return dict(op=op, layers=layers, slots=slots, pairs=pairs, freed=freed, hk=hk, dtype=dtype, state=state)
    live = _log_int(rng, 2, 48)
    moves = rng.randint(1, (live + 1) // 2)
    slots = live + moves + rng.randint(0, 24)
    layers = max(1, min(layers, 480 // (slots * hk // 4 + 1)))
    return dict(op=op, layers=layers, slots=slots, live=live, moves=moves, hk=hk, dtype=dtype, state=state)


def _size(dtype):
    return 4 if dtype == "f32" else 2


def _slot_bytes(case):
    hk, hv = case["hk"], 3 * case["hk"]
    return (2 * hk + hv) * D * 3 * _size(case["dtype"]) + hv * D * D * _size(case["state"])


def work(case):
    op = case["op"]
    if op == "norm":
        n = case["tokens"] * case["heads"] * D
        return {"bytes": 3 * n * _size(case["dtype"]) + 4 * D, "flops": 10 * n}
    if op == "copy":
        moved = case["pairs"] - case["freed"]
        return {"bytes": case["layers"] * (2 * moved + case["freed"]) * _slot_bytes(case), "flops": 0}
    if op == "compact":
        return {"bytes": case["layers"] * 2 * case["moves"] * _slot_bytes(case), "flops": 0}
    hk, hv, e, es = case["hk"], 3 * case["hk"], _size(case["dtype"]), _size(case["state"])
    if op == "prefill":
        tokens, rows, recorded = case["tokens"], case["seqs"], 0
        reads = rows if case["initial"] else 0
    else:
        tokens, rows = case["rows"] * case["steps"], case["rows"]
        recorded, reads = (tokens if case["record"] else 0), rows
    tensors = tokens * (2 * hk * D + 2 * hv * D + 2 * hv) * e
    return {"bytes": tensors + (reads + rows + recorded) * hv * D * D * es, "flops": 6 * D * D * hv * tokens}


# ------------------------------------------------------------------------------------------ inputs


def _gates(tokens, hv, dtype, gen):
    """Raw a and b projections and the layer's decay parameters, spread as such layers keep them."""
    dev = gen.device
    a = torch.randn(tokens, hv, device=dev, generator=gen).to(dtype)
    b = torch.randn(tokens, hv, device=dev, generator=gen).to(dtype)
    A_log = torch.empty(hv, device=dev).uniform_(0.05, 16.0, generator=gen).log()
    dt = torch.empty(hv, device=dev).uniform_(math.log(1e-3), math.log(1e-1), generator=gen).exp()
    dt_bias = dt + torch.log(-torch.expm1(-dt))
    return a, b, A_log, dt_bias


def _qkv(rows, hk, hv, dtype, gen):
    """Rows of the conv's output (SiLU of a near-normal value) and the q, k, v views of their columns."""
    x = torch.nn.functional.silu(torch.randn(rows, (2 * hk + hv) * D, device=gen.device, generator=gen)).to(dtype)
    q, k, v = x.split([hk * D, hk * D, hv * D], 1)
    return q.view(rows, hk, D), k.view(rows, hk, D), v.view(rows, hv, D)


def _lengths(case, rng):
    """Uneven lengths that add up to the case's tokens: shares of a lognormal, one token at least."""
    n, total = case["seqs"], case["tokens"]
    share = rng.lognormal(0.0, 1.0, n)
    cuts = np.floor(np.cumsum(share / share.sum()) * (total - n)).astype(int)
    cuts[-1] = total - n
    return (np.diff(cuts, prepend=0) + 1).tolist()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 32))
    s = {"case": case}
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    if op == "norm":
        n, h = case["tokens"], case["heads"]
        s["x"] = torch.randn(n, h, D, device=dev, generator=gen).mul_(0.2).to(dtype)
        s["z"] = torch.randn(n, h, D, device=dev, generator=gen).to(dtype)
        s["weight"] = torch.empty(D, device=dev).uniform_(0.5, 1.5, generator=gen)
        return s
    hk, hv = case["hk"], 3 * case["hk"]
    state = DTYPES[case["state"]]

    def states(slots):
        return torch.randn(slots, hv, D, D, device=dev, generator=gen).mul_(0.1).to(state)

    if op in ("copy", "compact"):
        caches = []
        for _ in range(case["layers"]):
            caches.append(torch.randn(case["slots"], (2 * hk + hv) * D, 3, device=dev, generator=gen).to(dtype))
            caches.append(states(case["slots"]))
        s["caches"] = caches
        perm = rng.permutation(case["slots"])
        if op == "copy":
            # Few sources (prompts that fork), distinct destinations; the first pairs free their slot.
            n = case["pairs"]
            src = perm[n : n + (n + 2) // 3][rng.randint(0, (n + 2) // 3, n)]
            src[: case["freed"]] = -1
            s["src"] = torch.tensor(src, dtype=torch.int32, device=dev)
            s["dst"] = torch.tensor(perm[:n], dtype=torch.int32, device=dev)
        else:
            live = np.zeros(case["slots"], bool)
            live[: case["live"]] = True
            live[rng.choice(case["live"], case["moves"], replace=False)] = False
            live[case["live"] + rng.choice(case["slots"] - case["live"], case["moves"], replace=False)] = True
            s["live"] = torch.tensor(live, device=dev)
        return s
    if op == "prefill":
        n, tokens = case["seqs"], case["tokens"]
        lengths = _lengths(case, rng)
        start = np.concatenate([[0], np.cumsum(lengths)])
        s["lengths"] = lengths
        s["query_start_loc"] = torch.tensor(start, dtype=torch.int32, device=dev)
        s["has_initial_state"] = torch.tensor(rng.rand(n) < (0.5 if case["initial"] else 0.0), device=dev)
        s["states"] = states(n + 3)
        s["indices"] = torch.tensor(rng.permutation(n + 3)[:n], dtype=torch.int32, device=dev)
        s["q"], s["k"], s["v"] = _qkv(tokens, hk, hv, dtype, gen)
        s["a"], s["b"], s["A_log"], s["dt_bias"] = _gates(tokens, hv, dtype, gen)
        return s
    n, steps = case["rows"], case["steps"]
    q, k, v = _qkv(n * steps, hk, hv, dtype, gen)
    s["q"], s["k"], s["v"] = (t.unflatten(0, (n, steps)) for t in (q, k, v))
    a, b, s["A_log"], s["dt_bias"] = _gates(n * steps, hv, dtype, gen)
    s["a"], s["b"] = a.view(n, steps, hv), b.view(n, steps, hv)
    s["states"] = states(case["slots"])
    s["indices"] = torch.tensor(rng.permutation(case["slots"])[:n], dtype=torch.int32, device=dev)
    s["record"] = torch.zeros(n, steps, hv, D, D, device=dev, dtype=state) if case["record"] else None
    s["record_indices"] = torch.arange(n, dtype=torch.int32, device=dev)
    return s


# --------------------------------------------------------------------------------------------- run


def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "copy": _own_copy, "compact": _own_compact, "prefill": _own_prefill, "decode": _own_decode}[op](s)
    return {"norm": _norm, "copy": _copy, "compact": _compact, "prefill": _prefill, "decode": _decode}[op](s)


def _own_norm(s):
    return _package().rms_norm_gated(s["x"], s["z"], s["weight"], NORM_EPS)


def _handle(s):
    """The engine's handle on its caches, made once."""
    if "handle" not in s:
        s["handle"] = _package().StateSlots(s["caches"])
    return s["handle"]


def _own_copy(s):
    _handle(s).copy(s["src"], s["dst"])
    return s["caches"]


def _own_compact(s):
    remap, count = _handle(s).compact(s["live"])
    return {"caches": s["caches"], "remap": remap, "count": count}


def _own_prefill(s):
    out = _package().gated_delta_rule_varlen_fn(
        s["q"], s["k"], s["v"], s["a"], s["b"], s["query_start_loc"], s["indices"], s["has_initial_state"], s["states"],
        A_log=s["A_log"], dt_bias=s["dt_bias"], qk_l2norm=True)
    return {"out": out, "states": s["states"]}


def _own_decode(s):
    out = _package().gated_delta_rule_update(
        s["q"], s["k"], s["v"], s["a"], s["b"], s["states"], s["indices"],
        A_log=s["A_log"], dt_bias=s["dt_bias"], qk_l2norm=True,
        intermediate_states=s["record"], intermediate_state_indices=s["record_indices"] if s["record"] is not None else None)
    got = {"out": out, "states": s["states"]}
    if s["record"] is not None:
        got["record"] = s["record"]
    return got


# ------------------------------------------------------------------------- the plain forms (fp32)


def _norm(s):
    x, z = s["x"].float(), s["z"].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + NORM_EPS) * s["weight"]
    return (y * z * torch.sigmoid(z)).to(s["x"].dtype)


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    clear = src < 0
    for c in s["caches"]:
        rows = c[src.clamp_min(0)]
        shape = (-1,) + (1,) * (c.dim() - 1)
        c[dst] = torch.where(clear.view(shape), torch.zeros((), dtype=c.dtype, device=c.device), rows)
    return s["caches"]


def _compact(s):
    live = s["live"]
    at = torch.arange(live.numel(), device=live.device)
    count = live.sum()
    holes, movers = (~live & (at < count)).nonzero()[:, 0], (live & (at >= count)).nonzero()[:, 0]
    remap = torch.where(live, at, -1)
    remap[movers] = holes
    for c in s["caches"]:
        c[holes] = c[movers]
    return {"caches": s["caches"], "remap": remap.int(), "count": count.int()}


def _gate(s):
    """log decay and beta of the raw projections, in fp32."""
    g = -torch.exp(s["A_log"].float()) * torch.nn.functional.softplus(s["a"].float() + s["dt_bias"].float())
    return g, torch.sigmoid(s["b"].float())


def _unit(x):
    return x * torch.rsqrt(x.square().sum(-1, keepdim=True) + L2_EPS)


def _prefill(s):
    q, k, v = s["q"], s["k"], s["v"]
    T, hk, hv = q.shape[0], q.shape[1], v.shape[1]
    dev, group = q.device, v.shape[1] // q.shape[1]
    # Chunks of every sequence, longest sequence first: rows[c] are a chunk's tokens (T: no token).
    order = sorted(range(len(s["lengths"])), key=lambda n: -s["lengths"][n])
    length = np.array([s["lengths"][n] for n in order])
    start = np.concatenate([[0], np.cumsum(s["lengths"])])[order]
    per = (length + CHUNK - 1) // CHUNK
    base = np.concatenate([[0], np.cumsum(per)])
    seq = np.repeat(np.arange(len(order)), per)
    first = (np.arange(base[-1]) - base[seq]) * CHUNK
    tok = first[:, None] + np.arange(CHUNK)
    rows = np.where(tok < length[seq][:, None], start[seq][:, None] + tok, T)
    rows = torch.from_numpy(rows).to(dev)
    base, active = base.tolist(), [int((per > c).sum()) for c in range(int(per[0]))]
    heads = torch.tensor(base[:-1], device=dev)

    def chunks(x):  # (T, H, ...) -> (chunks, H, 64, ...), fp32, zeros where there is no token
        x = torch.cat([x.float(), torch.zeros_like(x[:1], dtype=torch.float32)])
        return x[rows].transpose(1, 2)

    g, beta = _gate(s)
    g, beta = chunks(g), chunks(beta)
    qc, kc, vc = _unit(chunks(q)) * D**-0.5, _unit(chunks(k)), chunks(v)
    kk, qk = kc @ kc.mT, qc @ kc.mT
    decay = g.cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=dev).tril()
    ratio = torch.exp((decay.unsqueeze(-1) - decay.unsqueeze(-2)).masked_fill(~low, -math.inf))
    kk, qk, qc, kc = (x.repeat_interleave(group, 1) for x in (kk, qk, qc, kc))
    lower = (beta.unsqueeze(-1) * kk * ratio).tril(-1)
    qk = qk * ratio
    grow = torch.exp(decay).unsqueeze(-1)
    right = torch.cat([vc, kc * grow], -1) * beta.unsqueeze(-1)
    right = torch.linalg.solve_triangular(lower, right, upper=False, unitriangular=True)
    u, w = right.split(D, -1)
    qc = qc * grow
    last = decay[..., -1:]
    kc = kc * torch.exp(last - decay).unsqueeze(-1)
    last = torch.exp(last).unsqueeze(-1)
    slots = s["indices"].long()[torch.tensor(order, device=dev)]
    fresh = ~s["has_initial_state"][torch.tensor(order, device=dev)]
    S = s["states"][slots].float().masked_fill(fresh.view(-1, 1, 1, 1), 0.0)
    out = torch.empty(base[-1], hv, CHUNK, D, device=dev)
    for c, n in enumerate(active):  # the chain over chunks, all sequences that reach chunk c at once
        at = heads[:n] + c
        new = u[at] - w[at] @ S[:n]
        out[at] = qc[at] @ S[:n] + qk[at] @ new
        S[:n] = S[:n] * last[at] + kc[at].mT @ new
    s["states"][slots] = S.to(s["states"].dtype)
    packed = torch.empty(T + 1, hv, D, device=dev, dtype=q.dtype)
    packed[rows] = out.transpose(1, 2).to(q.dtype)
    return {"out": packed[:T], "states": s["states"]}


def _decode(s):
    steps, group = s["q"].shape[1], s["v"].shape[2] // s["q"].shape[2]
    g, beta = _gate(s)
    q = (_unit(s["q"].float()) * D**-0.5).repeat_interleave(group, 2)
    k = _unit(s["k"].float()).repeat_interleave(group, 2)
    v, alpha = s["v"].float(), torch.exp(g)
    slots = s["indices"].long()
    S = s["states"][slots].float()
    out = torch.empty_like(v)
    for t in range(steps):
        S = S * alpha[:, t, :, None, None]
        kt = k[:, t].unsqueeze(-1)
        u = beta[:, t].unsqueeze(-1) * (v[:, t] - (S * kt).sum(-2))
        S = S + kt * u.unsqueeze(-2)
        out[:, t] = (S * q[:, t].unsqueeze(-1)).sum(-2)
        if s["record"] is not None:
            s["record"][s["record_indices"].long(), t] = S.to(s["record"].dtype)
    s["states"][slots] = S.to(s["states"].dtype)
    got = {"out": out.to(s["q"].dtype), "states": s["states"]}
    if s["record"] is not None:
        got["record"] = s["record"]
    return got


# -------------------------------------------------------------------------------- 64-bit definition


def exact(case, seed):
    s = prepare(case, seed) if not own else None
    op = case["op"]
    if op == "norm":
        x, z, w = (s[n].double() for n in ("x", "z", "weight"))
        return x / (x.pow(2).sum(-1, keepdim=True) / D + NORM_EPS).sqrt() * w * z / (1 + torch.exp(-z))
    if op in ("copy", "compact"):
        return None  # values are only moved
    f = {n: s[n].double() for n in ("q", "k", "v", "a", "b")}
    arg = f["a"] + s["dt_bias"].double()
    alpha = torch.exp(-torch.exp(s["A_log"].double()) * torch.log1p(torch.exp(arg)))
    beta = 1 / (1 + torch.exp(-f["b"]))
    q, k = (x / (x.pow(2).sum(-1, keepdim=True) + L2_EPS).sqrt() for x in (f["q"], f["k"]))
    q, v = q / math.sqrt(D), f["v"]
    if op == "decode":
        q, k, v, alpha, beta = (x.flatten(0, 1) for x in (q, k, v, alpha, beta))
        lengths = [case["steps"]] * case["rows"]
        fresh = [False] * case["rows"]
    else:
        lengths, fresh = s["lengths"], (~s["has_initial_state"]).tolist()
    hk, hv = q.shape[1], v.shape[1]
    first = np.concatenate([[0], np.cumsum(lengths)])[:-1]
    order = np.argsort([-x for x in lengths], kind="stable")
    at = torch.tensor(first[order], device=q.device)
    slots = s["indices"].long()[torch.tensor(order, device=q.device)]
    S = s["states"][slots].double().view(len(lengths), hk, hv // hk, D, D)
    S[torch.tensor([fresh[i] for i in order], device=q.device)] = 0
    out = torch.empty(q.shape[0], hv, D, device=q.device, dtype=torch.float64)
    record = torch.zeros(s["record"].shape, device=q.device, dtype=torch.float64) if s.get("record") is not None else None
    lengths = np.array(lengths)[order]
    for t in range(int(lengths[0])):  # token by token, every sequence that has one
        n = int((lengths > t).sum())
        i = at[:n] + t
        kt, qt = k[i][:, :, None, None, :], q[i][:, :, None, None, :]
        X = S[:n]
        X *= alpha[i].view(n, hk, -1, 1, 1)
        u = beta[i].view(n, hk, -1, 1, 1) * (v[i].view(n, hk, -1, 1, D) - kt @ X)
        X += kt.mT * u
        out[i] = (qt @ X).view(n, hv, D)
        if record is not None:
            record[torch.tensor(order, device=q.device), t] = X.view(n, hv, D, D)
    states = s["states"].double()
    states[slots] = S.view(-1, hv, D, D)
    if op == "decode":
        out = out.view(case["rows"], case["steps"], hv, D)
    got = {"out": out, "states": states}
    if record is not None:
        got["record"] = record
    return got
