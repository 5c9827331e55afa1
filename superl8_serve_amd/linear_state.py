"""States of the linear-attention layers of a hybrid model: what ``PagedKVCache``
is to its attention layers (the role of the reference's ``RecurrentStateCache``,
superl8serve/models/cache.py).

A sequence holds one slot in every layer; a slot's state is fp32
``[heads, head_dim, head_dim]`` and does not grow with the context.  Handing a
slot out clears nothing: the first call on it in a layer starts from an empty
state (``reset``).  The calls here build their index tensors from lists, as
``PagedKVCache``'s do; a step that is captured into a graph calls ``ops`` with
tensors of its own and ``state[layer]``.
"""

from __future__ import annotations

import itertools

import torch

from . import ops


class LinearStateCache:
    def __init__(self, num_layers: int, num_slots: int, num_heads: int, head_dim: int, *, device):
        self.num_layers, self.num_slots = num_layers, num_slots
        self.device = device
        self.state = torch.zeros((num_layers, num_slots, num_heads, head_dim, head_dim), device=device)
        self._free_slots: list[int] = list(range(num_slots))  # LIFO, as PagedKVCache's pools
        self._fresh: list[set[int]] = [set() for _ in range(num_layers)]  # slots a layer has not used yet

    def alloc(self) -> int:
        if not self._free_slots:
            raise RuntimeError("LinearStateCache: no free slots")
        slot = self._free_slots.pop()
        for fresh in self._fresh:
            fresh.add(slot)
        return slot

    def free(self, slot: int) -> None:
        if not 0 <= slot < self.num_slots or slot in self._free_slots:
            raise ValueError(f"LinearStateCache: slot {slot} is not in use")
        self._free_slots.append(slot)

    def has_free_slot(self) -> bool:
        return bool(self._free_slots)

    def _rows(self, layer: int, slots: list[int]):
        """Device slots, and the mask of those that start empty (None: no such)."""
        if len(set(slots)) != len(slots):
            raise ValueError(f"LinearStateCache: slots {slots} repeat")
        if not all(0 <= s < self.num_slots for s in slots):
            raise ValueError(f"LinearStateCache: slots {slots} must be in [0, {self.num_slots})")
        new = [s in self._fresh[layer] for s in slots]
        reset = torch.tensor(new, device=self.device) if any(new) else None
        return torch.tensor(slots, dtype=torch.int32, device=self.device), reset

    def attn_varlen(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    slots: list[int], lens: list[int], *, scale: float) -> torch.Tensor:
        """Prompts (or chunks of them) of ``lens[i]`` tokens behind each other:
        ``q`` ``[T, Hq, D]``, ``k``, ``v`` ``[T, Hkv, D]``; every slot's state
        moves on by its tokens."""
        if len(slots) != len(lens) or sum(lens) != q.shape[0] or min(lens, default=0) < 0:
            raise ValueError(f"LinearStateCache: {len(slots)} slots, lengths {lens} for {q.shape[0]} tokens")
        at, reset = self._rows(layer, slots)
        cu = torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device=self.device)
        out = ops.linear_attn_varlen(q, k, v, log_decay, self.state[layer], cu, max(lens, default=0), state_slots=at,
                                     reset=reset, scale=scale)
        self._fresh[layer].difference_update(slots)  # (a refused call leaves its slots fresh)
        return out

    def attn_decode(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                    slots: list[int], *, scale: float) -> torch.Tensor:
        """One token per slot: ``q`` ``[B, Hq, D]``, ``k``, ``v`` ``[B, Hkv, D]``."""
        at, reset = self._rows(layer, slots)
        out = ops.linear_attn_decode(q, k, v, log_decay, self.state[layer], state_slots=at, reset=reset, scale=scale)
        self._fresh[layer].difference_update(slots)
        return out
