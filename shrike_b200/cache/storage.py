"""Device memory behind the cache manager's ids.

Each group of key/value caches is one tensor
`[caches in group, planes, pages, page_size, kv heads, head size]` in the engine dtype (planes 2:
keys and values; 1: one tensor a token that serves as both, a cached latent):
the layout Azimml/shrike uses for its single pool
(shrike/engine/model_runner.py:52-60, per layer viewed as pages at :74-75), once
per group.  A quantised pool keeps int8 codes of that shape and beside them float32 scales
`[caches in group, planes, pages, kv heads, page_size]` (`cache/quantised.py`).  Per-request state of fixed size is one tensor `[slots, *shape]` per
cache id that asked for it; `zero_slots` clears the slots of requests that were just opened,
which the step function calls before their first token runs (a part never has to).
"""

from __future__ import annotations

import torch

from .manager import KVGroupSpec
from .quantised import QuantisedPages


def page_bytes(group: KVGroupSpec, page_size: int, element_size: int, quantised: bool = False) -> int:
    row = group.head_dim + 4 if quantised else group.head_dim * element_size   # a head's elements of one token, with their scale
    return len(group.cache_ids) * group.planes * page_size * group.num_kv_heads * row


def state_bytes(state_needs: dict, max_slots: int) -> int:
    """Bytes of all per-request state: every stateful cache holds `max_slots` slots of its shape."""
    total = 0
    for need in state_needs.values():
        count = 1
        for extent in need.shape:
            count *= extent
        total += max_slots * count * torch.empty((), dtype=getattr(torch, need.dtype)).element_size()
    return total


class CacheStorage:
    def __init__(self, groups, page_size, num_pages, state_needs, max_slots, dtype, device, quantised: bool = False):
        self.groups = list(groups)
        self.page_size = page_size
        self.quantised = quantised
        self.scales: list[torch.Tensor] = []
        self._pages: dict[int, tuple] = {}   # cache id -> (keys, values) of a quantised pool
        self.group_of_cache: dict[int, tuple[int, int]] = {}
        self.kv: list[torch.Tensor] = []
        counts = [num_pages] * len(self.groups) if isinstance(num_pages, int) else list(num_pages)
        for index, (group, count) in enumerate(zip(self.groups, counts)):
            self.kv.append(
                torch.zeros(
                    len(group.cache_ids), group.planes, count, page_size, group.num_kv_heads, group.head_dim,
                    dtype=torch.int8 if quantised else dtype, device=device,
                )
            )
            if quantised:
                self.scales.append(torch.zeros(len(group.cache_ids), group.planes, count, group.num_kv_heads, page_size,
                                               dtype=torch.float32, device=device))
            for position, cache_id in enumerate(group.cache_ids):
                self.group_of_cache[cache_id] = (index, position)
                if quantised:
                    self._pages[cache_id] = tuple(QuantisedPages(self.kv[index][position][plane], self.scales[index][position][plane])
                                                  for plane in (0, -1))
        self.state: dict[int, torch.Tensor] = {
            cache_id: torch.zeros((max_slots, *need.shape), dtype=getattr(torch, need.dtype), device=device)
            for cache_id, need in state_needs.items()
        }

    def zero_slots(self, slots: list[int]) -> None:
        """Zeroes the state of `slots` in every stateful cache: one launch for all of them."""
        if not slots or not self.state:
            return
        torch._foreach_zero_([tensor[slot] for tensor in self.state.values() for slot in slots])

    def keys_values(self, cache_id: int):
        """(group index, keys, values), each `[pages, page_size, kv heads, head size]`; in a group of one
        plane both are the same tensor.  In a quantised pool both are `QuantisedPages`."""
        group, position = self.group_of_cache[cache_id]
        if self.quantised:
            return group, *self._pages[cache_id]
        slab = self.kv[group][position]
        return group, slab[0], slab[-1]

    def bytes(self) -> int:
        total = sum(t.numel() * t.element_size() for t in self.kv + self.scales)
        return total + sum(t.numel() * t.element_size() for t in self.state.values())
