"""The operators behind the conv of a Gated DeltaNet layer: the gated delta rule (packed and dense
prefill, recurrent decode) and the gated RMS norm.

Per value head, with a (dk, dv) state S and its query/key head (value heads share query/key heads in
groups), each token does in fp32

    S <- exp(g) S;   u = beta (v - S^T k);   S <- S + k u^T;   out = scale S^T q.

g is the log decay (<= 0) and beta the update rate. With A_log and dt_bias, g and beta are the
layer's raw projections (the a and b that causal_conv1d_update_unpack returns): the log decay is
-exp(A_log) softplus(g + dt_bias) and the rate sigmoid(beta).

q, k and v may be column views of the conv's output rows; they are read in place. As everywhere in
this package, calls the kernels cannot serve (CPU tensors, gradients, other dtypes) raise
functional.Unsupported.
"""

import torch

from . import _ops
from .functional import _DTYPES, MAX_STEPS, PAD_SLOT_ID, _flags, _int32, _unsupported


def _shapes(q, k, v, g, beta, lead, A_log, dt_bias):
    """Reject shapes inconsistent with a gated delta rule over lead leading axes."""
    qs, vs = q.shape, v.shape
    if not len(qs) == k.dim() == len(vs) == lead + 2:
        raise ValueError(f"q, k, v must have {lead + 2} axes, got {q.dim()}, {k.dim()}, {v.dim()}")
    if qs != k.shape or qs[:lead] != vs[:lead]:
        raise ValueError(
            f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not go together"
        )
    hk, hv = qs[-2], vs[-2]
    if hk < 1 or hv < 1 or hv % hk:
        raise ValueError(f"{hv} value heads are not a multiple of {hk} query/key heads")
    if qs[-1] < 1 or vs[-1] < 1:
        raise ValueError("head dims must be at least 1")
    want = vs[:-1]
    if g.shape != want or beta.shape != want:
        raise ValueError(f"g {tuple(g.shape)} and beta {tuple(beta.shape)} must have shape {tuple(want)}")
    if (A_log is None) != (dt_bias is None):
        raise ValueError("A_log and dt_bias come together")
    if A_log is not None and (A_log.shape != (hv,) or dt_bias.shape != (hv,)):
        raise ValueError(f"A_log and dt_bias must have shape ({hv},)")


def _state_shape(states, v, dk, what="states"):
    want = (v.shape[-2], dk, v.shape[-1])
    if states.dim() != 4 or tuple(states.shape[1:]) != want:
        raise ValueError(f"{what} shape {tuple(states.shape)} is not (slots, {want[0]}, {want[1]}, {want[2]})")


def gated_delta_rule_reason(q, k, v, g, beta, states=None, A_log=None, dt_bias=None):
    """Why the kernels cannot serve these tensors, or None."""
    grad, device = torch.is_grad_enabled(), q.device
    apart = False
    for t in (q, k, v, g, beta, states, A_log, dt_bias):
        if t is not None:
            if grad and t.requires_grad:
                return "gradients are required and the kernels have no backward pass"
            apart = apart or t.device != device
    if not q.is_cuda:
        return "input is not a CUDA tensor"
    if apart:
        return "tensors are on different devices"
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        return f"dtypes {q.dtype}, {k.dtype}, {v.dtype} are not one of bf16, fp16 or fp32"
    if g.dtype not in _DTYPES or beta.dtype not in _DTYPES:
        return f"gate dtypes {g.dtype}, {beta.dtype} are not bf16, fp16 or fp32"
    if A_log is not None and (A_log.dtype not in _DTYPES or dt_bias.dtype not in _DTYPES):
        return f"A_log and dt_bias dtypes {A_log.dtype}, {dt_bias.dtype} are not bf16, fp16 or fp32"
    if q.shape[-1] > 256:
        return f"a key head dim of {q.shape[-1]} is above 256"
    if states is not None:
        if states.dtype not in (torch.float32, q.dtype):
            return f"state dtype {states.dtype} is neither fp32 nor the input dtype"
        if states.stride(-1) != 1:
            return f"state strides {states.stride()} (the last axis must be contiguous)"
    return None


def _params(A_log, dt_bias):
    """The gates' parameters contiguous and of one dtype, as the kernels read them (fp32 holds all)."""
    if A_log is None:
        return None, None
    if A_log.dtype != dt_bias.dtype:
        A_log, dt_bias = A_log.float(), dt_bias.float()
    return A_log.contiguous(), dt_bias.contiguous()


def _index(index, device):
    """Slot indices as contiguous int32 on device; None stays None."""
    index = _int32(index, device)
    return index if index is None or index.is_contiguous() else index.contiguous()


def gated_delta_rule_varlen_fn(
    q,
    k,
    v,
    g,
    beta,
    query_start_loc,
    cache_indices=None,
    has_initial_state=None,
    states=None,
    A_log=None,
    dt_bias=None,
    scale=None,
    qk_l2norm=False,
    pad_slot_id=PAD_SLOT_ID,
    out=None,
):
    """Gated delta rule over a packed variable-length batch (the prefill of a serving step).

    Args:
        q, k: (total_tokens, heads_k, dk), any strides.
        v: (total_tokens, heads_v, dv), heads_v a multiple of heads_k.
        g, beta: (total_tokens, heads_v) log decays and rates, or raw projections with A_log.
        query_start_loc: int32 (batch + 1,) cumulative sequence lengths.
        cache_indices: optional (batch,) slot of each sequence (default: slot i).
        has_initial_state: optional (batch,) bool/uint8: start from the cached state.
        states: optional (slots, heads_v, dk, dv) cache of fp32 or the input dtype, updated in
            place with the final state of each sequence (sequences of zero tokens leave theirs).
        A_log, dt_bias: optional (heads_v,) parameters of raw gates (where their dtypes differ, or for
            strided views, the call makes copies).
        scale: output scale (default dk ** -0.5).
        qk_l2norm: scale q and k to unit length first (eps 1e-6 under the root).
        pad_slot_id: cache_indices value marking sequences to skip (their outputs are undefined
            and their slots untouched).
        out: optional output of the shape and dtype of v.

    Two forms serve a call. Chunk by chunk of 64 tokens on the tensor cores: bf16 and fp16 with dk = 128,
    dv a multiple of 32 and rows on 16-byte boundaries, where sequences have 12 tokens on average; in other
    batches of 128 tokens and more the long sequences (above 32 tokens, or where there are more than 32
    such above 64, 128, ..). Token by token: all else. Both hold the precision of fp32 (the operands of the
    tensor cores have its 24 bits, in three parts), but they round differently, so that the last bits of a
    sequence depend on the batch it came in, and where a value is not finite the chunked form spoils
    the rows of its whole chunk, earlier ones included, token by token only its own and later ones. The
    chunked form's temporary takes 49,936 bytes per value head for each of tokens / 64 + batch chunks
    (32 or fewer instead of batch for long sequences alone), and 1024 bytes per token and key head more for fp16
    (in groups of heads from 4 GiB on).

    The chunked kernels wait for copies of their own. Should such a wait ever take above two seconds,
    the outputs that depend on it are NaN, the slot keeps its state, and device_status() says so
    (_lib.DEV_TIMEOUT).

    Returns:
        (total_tokens, heads_v, dv) output.
    """
    _shapes(q, k, v, g, beta, 1, A_log, dt_bias)
    if query_start_loc is None or query_start_loc.dim() != 1 or query_start_loc.numel() < 1:
        raise ValueError("a packed batch needs query_start_loc of shape (batch + 1,)")
    n = query_start_loc.numel() - 1
    if states is not None:
        _state_shape(states, v, q.shape[-1])
    for t, what in ((cache_indices, "cache_indices"), (has_initial_state, "has_initial_state")):
        if t is not None and tuple(t.shape) != (n,):
            raise ValueError(f"{what} must have shape ({n},), got {tuple(t.shape)}")
    why = gated_delta_rule_reason(q, k, v, g, beta, states, A_log, dt_bias)
    if why is None and query_start_loc.dtype != torch.int32:
        why = "query_start_loc is not int32"
    if why is not None:
        _unsupported(why)
    if states is not None and cache_indices is None and states.shape[0] < n:
        raise ValueError(f"states has {states.shape[0]} slots for {n} sequences and no cache_indices")
    out = _output(out, v)
    dev = q.device
    qsl = _index(query_start_loc, dev)
    idx = _index(cache_indices, dev) if states is not None else None
    hinit = _flags(has_initial_state, dev) if states is not None else None
    if hinit is not None and not hinit.is_contiguous():
        hinit = hinit.contiguous()
    _ops.gdr_varlen(q, k, v, g, beta, *_params(A_log, dt_bias), out, states, qsl, idx, hinit,
                    q.shape[-1] ** -0.5 if scale is None else scale, qk_l2norm, pad_slot_id)
    return out


def _output(out, v):
    if out is None:
        return torch.empty(v.shape, dtype=v.dtype, device=v.device)
    if out.shape != v.shape or out.dtype != v.dtype or out.device != v.device:
        raise ValueError(f"out must have the shape, dtype and device of v, got {tuple(out.shape)} {out.dtype}")
    return out


def gated_delta_rule_fn(
    q,
    k,
    v,
    g,
    beta,
    initial_states=None,
    return_final_states=False,
    A_log=None,
    dt_bias=None,
    scale=None,
    qk_l2norm=False,
):
    """Gated delta rule over a dense batch of sequences of one length.

    Args:
        q, k: (batch, seqlen, heads_k, dk); v: (batch, seqlen, heads_v, dv); g, beta: (batch,
            seqlen, heads_v). Batches whose rows follow one another evenly are read in place,
            others are packed first.
        initial_states: optional (batch, heads_v, dk, dv) states (zeros when None), not changed.
        return_final_states: also return the (batch, heads_v, dk, dv) fp32 final states.
        A_log, dt_bias, scale, qk_l2norm: as in gated_delta_rule_varlen_fn.

    Returns:
        (batch, seqlen, heads_v, dv) output, or (output, final states).
    """
    _shapes(q, k, v, g, beta, 2, A_log, dt_bias)
    B, L, hv, dv = v.shape
    dk = q.shape[-1]
    if initial_states is not None and tuple(initial_states.shape) != (B, hv, dk, dv):
        raise ValueError(f"initial_states shape {tuple(initial_states.shape)} is not {(B, hv, dk, dv)}")
    why = gated_delta_rule_reason(q, k, v, g, beta, None, A_log, dt_bias)
    if why is None and initial_states is not None and initial_states.device != q.device:
        why = "initial_states is on another device"
    if why is None and initial_states is not None and torch.is_grad_enabled() and initial_states.requires_grad:
        why = "gradients are required and the kernels have no backward pass"
    if why is not None:
        _unsupported(why)
    final = None
    if initial_states is not None:
        final = initial_states.to(torch.float32, copy=True).contiguous()
    elif return_final_states:
        final = torch.zeros((B, hv, dk, dv), dtype=torch.float32, device=q.device)
    out = torch.empty((B, L, hv, dv), dtype=v.dtype, device=v.device)
    if B > 0 and L > 0:
        qsl = torch.arange(0, (B + 1) * L, L, dtype=torch.int32, device=q.device)
        hinit = None
        if initial_states is not None:
            hinit = torch.ones(B, dtype=torch.uint8, device=q.device)
        _ops.gdr_varlen(*(t.flatten(0, 1) for t in (q, k, v, g, beta)), *_params(A_log, dt_bias),
                        out.flatten(0, 1), final, qsl, None, hinit,
                        dk**-0.5 if scale is None else scale, qk_l2norm, PAD_SLOT_ID, L)
    return (out, final) if return_final_states else out


def gated_delta_rule_update(
    q,
    k,
    v,
    g,
    beta,
    states,
    state_indices=None,
    A_log=None,
    dt_bias=None,
    scale=None,
    qk_l2norm=False,
    pad_slot_id=PAD_SLOT_ID,
    intermediate_states=None,
    intermediate_state_indices=None,
    update_states=True,
):
    """Advance the state of each row by one or more tokens and compute their outputs (decode).

    Args:
        q, k: (batch, heads_k, dk) for one token, or (batch, steps, heads_k, dk) with 1 <= steps
            <= 16 for the multi-token step that verifies speculative drafts; any strides.
        v: (batch[, steps], heads_v, dv); g, beta: (batch[, steps], heads_v).
        states: (slots, heads_v, dk, dv) cache of fp32 or the input dtype, updated in place.
        state_indices: optional int32 (batch,) slot of each row (default: row b, slot b).
        A_log, dt_bias, scale, qk_l2norm: as in gated_delta_rule_varlen_fn.
        pad_slot_id: slot value marking rows to skip (state untouched, output undefined).
        intermediate_states: optional (slots, steps, heads_v, dk, dv) cache of the dtype of
            states, receiving the state after every token.
        intermediate_state_indices: optional int32 (batch,) slots of that cache (default:
            state_indices).
        update_states: False leaves states unchanged (a draft whose accepted length is not yet
            known; StateSlots.copy commits one of the intermediate states).

    Returns:
        Output of the shape of v.
    """
    single = q.dim() == 3
    _shapes(q, k, v, g, beta, 1 if single else 2, A_log, dt_bias)
    B = q.shape[0]
    _state_shape(states, v, q.shape[-1])
    for t, what in ((state_indices, "state_indices"), (intermediate_state_indices, "intermediate_state_indices")):
        if t is not None and tuple(t.shape) != (B,):
            raise ValueError(f"{what} must have shape ({B},), got {tuple(t.shape)}")
    inter = intermediate_states
    if inter is not None:
        want = (1 if single else q.shape[1], *states.shape[1:])
        if inter.dim() != 5 or tuple(inter.shape[1:]) != want:
            raise ValueError(f"intermediate_states shape {tuple(inter.shape)} is not (slots, {want})")
    why = gated_delta_rule_reason(q, k, v, g, beta, states, A_log, dt_bias)
    if why is None and not single and not 1 <= q.shape[1] <= MAX_STEPS:
        why = f"{q.shape[1]} steps is outside 1..{MAX_STEPS}"
    if why is None and inter is not None and (
        inter.dtype != states.dtype or inter.device != q.device or inter.stride(-1) != 1
    ):
        why = f"intermediate states {inter.dtype} with strides {inter.stride()} on {inter.device}"
    if why is not None:
        _unsupported(why)
    if state_indices is None and states.shape[0] < B:
        raise ValueError(f"states has {states.shape[0]} slots for {B} rows and no state_indices")
    out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    dev = q.device
    idx = _index(state_indices, dev)
    iidx = _index(intermediate_state_indices, dev) if inter is not None else None
    _ops.gdr_update(q, k, v, g, beta, *_params(A_log, dt_bias), out, states, idx, inter, iidx,
                    q.shape[-1] ** -0.5 if scale is None else scale, qk_l2norm, update_states,
                    pad_slot_id)
    return out


def rms_norm_gated(x, z, weight, eps=1e-6, out=None):
    """x rsqrt(mean(x^2) + eps) weight silu(z) over the last axis, in fp32, rounded once.

    Args:
        x: (..., dim) rows, for a Gated DeltaNet layer (tokens, heads_v, dv).
        z: gate of the shape of x (the z of causal_conv1d_update_unpack, viewed per head), or None.
        weight: (dim,) of fp32 or the dtype of x.
        eps: added to the mean square.
        out: optional output of the shape and dtype of x; it may be x itself.

    Returns:
        Output of the shape of x.
    """
    if x.dim() < 1 or weight.dim() != 1 or x.shape[-1] != weight.shape[0] or x.shape[-1] < 1:
        raise ValueError(f"weight {tuple(weight.shape)} does not fit x {tuple(x.shape)}")
    if z is not None and z.shape != x.shape:
        raise ValueError(f"z {tuple(z.shape)} must have the shape of x {tuple(x.shape)}")
    tensors = [x, weight] + ([] if z is None else [z])
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        _unsupported("gradients are required and the kernels have no backward pass")
    if not x.is_cuda:
        _unsupported("input is not a CUDA tensor")
    if x.dtype not in _DTYPES or (z is not None and z.dtype != x.dtype):
        _unsupported(f"dtype {x.dtype} with gate {None if z is None else z.dtype}")
    if weight.dtype not in (torch.float32, x.dtype) or any(t.device != x.device for t in tensors):
        _unsupported("weight must be fp32 or of the input dtype, on its device")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"out must have the shape, dtype and device of x, got {tuple(out.shape)} {out.dtype}")

    def rows(t):
        # (n0, n1, dim) view, or a copy where the leading axes or the last one do not allow a view.
        t = t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()
        return t if t.dim() == 3 else t.reshape(-1, 1, t.shape[-1])

    w = weight if weight.is_contiguous() else weight.contiguous()
    if out.dim() != 3 and not out.is_contiguous() or out.stride(-1) != 1 and out.shape[-1] != 1:
        out.copy_(rms_norm_gated(x, z, weight, eps))
        return out
    _ops.rms_norm_gated(rows(x), None if z is None else rows(z), w, float(eps), rows(out))
    return out
