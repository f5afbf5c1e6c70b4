"""A Gated DeltaNet layer served with this package: packed prefill, a fork of the cached state, decode
steps, verification of drafted tokens, and compaction of the cache.

    python examples/gated_deltanet.py

Random weights; the run checks that every way to the same tokens gives the same result (a prompt in
one piece, in two, token by token, and as a verified draft), within the rounding of bf16.
"""

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "causal-conv1d-cute_b200"))

import causal_conv1d_cute as C  # noqa: E402
from causal_conv1d_cute.unpack import causal_conv1d_update_unpack  # noqa: E402

HEADS_K, HEADS_V, DIM, WIDTH = 2, 6, 128, 4  # the 16/48-head serving shape on one of eight ranks


class GatedDeltaNet:
    """One layer: projections, conv, gated delta rule, gated norm, output projection.

    conv_states (slots, conv channels, width - 1) and delta_states (slots, heads, dim, dim) are its
    caches; a request owns one slot in both.
    """

    def __init__(self, hidden, slots, device="cuda", dtype=torch.bfloat16, seed=0):
        r = torch.Generator(device).manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, device=device, generator=r) * shape[-1] ** -0.5).to(dtype)

        self.conv_dim = (2 * HEADS_K + HEADS_V) * DIM
        self.in_qkvz = weight(self.conv_dim + HEADS_V * DIM, hidden)
        self.in_ba = weight(2 * HEADS_V, hidden)
        self.conv = weight(self.conv_dim, WIDTH)
        self.A_log = torch.empty(HEADS_V, device=device).uniform_(1, 16, generator=r).log()
        self.dt_bias = torch.randn(HEADS_V, device=device, generator=r) - 4
        self.norm = torch.rand(DIM, device=device, generator=r) + 0.5
        self.out = weight(hidden, HEADS_V * DIM)
        self.conv_states = torch.zeros(slots, self.conv_dim, WIDTH - 1, device=device, dtype=dtype)
        self.delta_states = torch.zeros(slots, HEADS_V, DIM, DIM, device=device)
        self.slots = C.StateSlots([self.conv_states, self.delta_states])

    def _heads(self, conv_out, lead):
        q, k, v = conv_out.split([HEADS_K * DIM, HEADS_K * DIM, HEADS_V * DIM], -1)
        return q.unflatten(-1, (HEADS_K, DIM)), k.unflatten(-1, (HEADS_K, DIM)), v.unflatten(-1, (HEADS_V, DIM))

    def _finish(self, o, z):
        y = C.rms_norm_gated(o, z.unflatten(-1, (HEADS_V, DIM)), self.norm)
        return y.flatten(-2) @ self.out.t()

    def prefill(self, x, query_start_loc, slots, has_initial_state):
        """x: (tokens, hidden), packed."""
        qkvz, ba = x @ self.in_qkvz.t(), x @ self.in_ba.t()
        conv = C.causal_conv1d_varlen_fn(qkvz[:, : self.conv_dim].t(), self.conv, None, query_start_loc, slots,
                                         has_initial_state, self.conv_states, "silu").t()
        q, k, v = self._heads(conv, 1)
        b, a = ba.chunk(2, -1)
        o = C.gated_delta_rule_varlen_fn(q, k, v, a, b, query_start_loc, slots, has_initial_state, self.delta_states,
                                         A_log=self.A_log, dt_bias=self.dt_bias, qk_l2norm=True)
        return self._finish(o, qkvz[:, self.conv_dim :])

    def decode(self, x, slots):
        """x: (rows, hidden), one token each."""
        qkvz, ba = x @ self.in_qkvz.t(), x @ self.in_ba.t()
        conv, z, b, a = causal_conv1d_update_unpack(qkvz, ba, self.conv_states, self.conv, None, slots, HEADS_V, "silu", -1)
        q, k, v = self._heads(conv, 1)
        o = C.gated_delta_rule_update(q, k, v, a, b, self.delta_states, slots, A_log=self.A_log, dt_bias=self.dt_bias,
                                      qk_l2norm=True)
        return self._finish(o, z)

    def verify(self, x, slots, accepted):
        """x: (rows, steps, hidden) drafted tokens; the states after accepted (rows,) of them are kept."""
        rows, steps = x.shape[:2]
        qkvz, ba = x @ self.in_qkvz.t(), x @ self.in_ba.t()
        windows = torch.empty(rows, steps, self.conv_dim, WIDTH - 1, device=x.device, dtype=x.dtype)
        states = torch.empty(rows, steps, *self.delta_states.shape[1:], device=x.device)
        own = torch.arange(rows, dtype=torch.int32, device=x.device)
        conv = C.causal_conv1d_update(qkvz[..., : self.conv_dim].transpose(1, 2), self.conv_states, self.conv, None, "silu",
                                      slots, intermediate_conv_window=windows, intermediate_state_indices=own)
        q, k, v = self._heads(conv.transpose(1, 2), 2)
        b, a = ba.chunk(2, -1)
        o = C.gated_delta_rule_update(q, k, v, a, b, self.delta_states, slots, A_log=self.A_log, dt_bias=self.dt_bias,
                                      qk_l2norm=True, intermediate_states=states, intermediate_state_indices=own,
                                      update_states=False)
        # Commit: step accepted - 1 of each row, from the recorded states to the caches.
        recorded = C.StateSlots([windows.flatten(0, 1), states.flatten(0, 1)])
        self.slots.copy(own * steps + accepted - 1, slots, source=recorded)
        return self._finish(o, qkvz[..., self.conv_dim :])


def main(hidden=256, prompt=150, more=6):
    dev = "cuda"
    layer = GatedDeltaNet(hidden, slots=8)
    x = torch.randn(prompt + more, hidden, device=dev).to(torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    flag = lambda *v: torch.tensor(v, dtype=torch.bool, device=dev)  # noqa: E731

    # All tokens at once in slot 0; the prompt alone in slot 5, in two pieces.
    whole = layer.prefill(x, i32(0, prompt + more), i32(0), flag(False))
    cut = prompt // 3
    layer.prefill(x[:cut], i32(0, cut), i32(5), flag(False))
    layer.prefill(x[cut:prompt], i32(0, prompt - cut), i32(5), flag(True))

    # Fork the prompt to slots 2 and 7: one goes on token by token, one as a verified draft.
    layer.slots.copy(i32(5, 5), i32(2, 7))
    steps = torch.cat([layer.decode(x[prompt + i : prompt + i + 1], i32(2)) for i in range(more)])
    draft = layer.verify(x[prompt:][None], i32(7), i32(more))[0]

    # Free slots 0 and 5, and move the two live slots to the front.
    final = layer.delta_states[0].clone()
    layer.slots.copy(i32(-1, -1), i32(0, 5))
    remap, count = layer.slots.compact(flag(False, False, True, False, False, False, False, True))
    assert int(count) == 2 and remap.tolist() == [-1, -1, 0, -1, -1, -1, -1, 1], remap.tolist()

    def off(a, b):
        return ((a.double() - b.double()).norm() / b.double().norm()).item()

    errors = {"decode": off(steps, whole[prompt:]), "draft": off(draft, whole[prompt:]),
              "state, decode": off(layer.delta_states[0], final), "state, draft": off(layer.delta_states[1], final)}
    # Each way rounds the projections and the conv to bf16 on its own, with other sums before the
    # rounding: a few parts in 2^8.
    assert all(e < 0.03 for e in errors.values()), errors
    return errors


if __name__ == "__main__":
    for name, e in main().items():
        print(f"{name:14s} {e:.2e} from the prefill of all tokens")
