"""Goals over a video's history: training with cross attention, rollout from the 8-bit cache.

A few goal queries attend to the states of the events that fired so far
(ragged event counts, dead slots), as the goal transformer of the world model
does (hclsm/dynamics/level2_goal.py:88-141), with the queries and keys of each
head normalised and rotated by event time.  Training runs over all states at
once; a rollout appends one event's states a step to an 8-bit cache and asks
again.

    PYTHONPATH=. python examples/goal_memory.py
"""
from __future__ import annotations

import torch
import torch.nn as nn

from hclsm_b200.kernels import (Kv8Cache, cross_attention, kv8_attention, kv8_write, qk_norm_rope, rope_tables)


class GoalMemory(nn.Module):
    """Goals (B, G, d_model) attend to states (B, K, N, d_model) of K events with N slots."""

    def __init__(self, d_model=384, heads=6, kv_heads=3, max_events=512, device="cuda", dtype=torch.bfloat16):
        super().__init__()
        if d_model % heads:
            raise ValueError(f"d_model {d_model} must be a multiple of heads {heads}")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, d_model // heads
        kw = dict(bias=False, device=device, dtype=dtype)
        self.q = nn.Linear(d_model, heads * self.head_dim, **kw)
        self.kv = nn.Linear(d_model, 2 * kv_heads * self.head_dim, **kw)
        self.out = nn.Linear(heads * self.head_dim, d_model, **kw)
        self.q_weight = nn.Parameter(torch.ones(self.head_dim, device=device))
        self.k_weight = nn.Parameter(torch.ones(self.head_dim, device=device))
        self.cos, self.sin = rope_tables(max_events, self.head_dim, device=device)

    def _queries(self, goals):
        return self.q(goals).unflatten(-1, (self.heads, self.head_dim))

    def _keys_values(self, states):
        return self.kv(states).unflatten(-1, (2, self.kv_heads, self.head_dim)).unbind(-3)

    def forward(self, goals, states, now, counts=None, alive=None):
        """All states at once: now (B,) the goals' time, counts (B,) events that count, alive (B, N) bool slots."""
        B, K, N, _ = states.shape
        q = self._queries(goals)
        k, v = self._keys_values(states.flatten(1, 2))  # views of one projection
        times = torch.arange(K, device=k.device, dtype=torch.int32).repeat_interleave(N).expand(B, K * N)
        q, k = qk_norm_rope(q, k, self.q_weight, self.k_weight, self.cos, self.sin,
                            q_pos=now[:, None].expand(B, q.shape[1]), k_pos=times)
        o = cross_attention(q, k, v, kv_lens=None if counts is None else counts * N,
                            key_mask=None if alive is None else alive[:, None].expand(B, K, N).flatten(1))
        return self.out(o.flatten(2))

    def cache(self, batch, events, slots):
        return Kv8Cache.empty(batch, events * slots, self.kv_heads, self.head_dim, dtype=self.q.weight.dtype,
                              device=self.q.weight.device)

    @torch.no_grad()
    def step(self, cache, goals, states, now, start):
        """One rollout step: the N states of the event at time ``now`` (B,) join the ``start`` (B,) cached ones,
        and the goals attend to all of them."""
        B, N, _ = states.shape
        k, v = self._keys_values(states)
        q, k = qk_norm_rope(self._queries(goals), k, self.q_weight, self.k_weight, self.cos, self.sin,
                            q_pos=now[:, None].expand(B, goals.shape[1]), k_pos=now[:, None].expand(B, N))
        kv8_write(cache, k, v, start)
        return self.out(kv8_attention(q, cache, start + N).flatten(2))


def main(steps=30, B=8, K=24, N=32, G=4, d=384):
    torch.manual_seed(0)
    model = GoalMemory(d)
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    goals, states = (torch.randn(*s, device="cuda", dtype=torch.bfloat16) for s in ((B, G, d), (B, K, N, d)))
    counts = torch.randint(K // 2, K + 1, (B,), device="cuda", dtype=torch.int32)
    alive = torch.rand(B, N, device="cuda") > 0.1
    target, now = states.mean((1, 2))[:, None].expand(B, G, d).float(), counts - 1
    losses = []
    for _ in range(steps):
        loss = (model(goals, states, now, counts, alive).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    losses = torch.stack(losses).tolist()
    cache, far = model.cache(B, K, N), []
    for t in range(K):
        at = torch.full((B,), t, device="cuda", dtype=torch.int32)
        got = model.step(cache, goals, states[:, t], at, at * N)
        with torch.no_grad():
            want = model(goals, states[:, :t + 1], at)
        far.append((got.float() - want.float()).norm() / want.float().norm())
    far = float(torch.stack(far).max())
    print(f"loss {losses[0]:.5f} -> {losses[-1]:.5f}; rollout from the 8-bit cache: {far:.4f} from full attention")
    return losses, far


if __name__ == "__main__":
    main()
