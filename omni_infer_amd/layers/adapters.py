"""Low-rank adapters of many requests beside the replicated projections.

The quantised weights of a served model cannot take an adapter in, and a batch mixes requests of many adapters (and
of none), so every projection keeps a set of adapters of its own beside its shared weight and adds each token's
update to the shared product (``hip_ops.adapter_linear``).  ``ReplicatedLinear`` / ``MergedReplicatedLinear``
(omni/models/common/layers/linear.py:620-762) are where they hang:

    layer.enable_adapters(max_adapters=32, max_rank=16)
    layer.adapters.set_adapter(slot, lora_a, lora_b, scaling)     # scaling = alpha / rank
    batch = AdapterBatch(adapter_ids, max_adapters=32)            # once for a batch, -1: no adapter
    y, _ = layer(x, batch)
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Union

import torch
import torch.nn as nn

from .. import hip_ops as ops


class AdapterBatch:
    """Which adapter each token of a batch uses, sorted once for all projections of all layers, on whatever streams they
    run (``hip_ops.adapter_plan`` for what holds under graph capture)."""

    def __init__(self, adapter_ids: torch.Tensor, max_adapters: int):
        self.max_adapters = int(max_adapters)
        self.plan = ops.adapter_plan(adapter_ids, self.max_adapters)


class AdapterSlots(nn.Module):
    """The adapters of one projection with the output widths ``output_sizes`` (one, or the shards of a stacked one).
    A slot that holds nothing has the scale 0, which adds nothing whatever the rows hold.  Shorter ranks and shards that an
    adapter leaves alone are filled up with zeros to ``max_rank``, which is rounded up to a multiple of 8: a row of x that
    is not finite comes out as NaN there, where infinities times those zeros meet."""

    def __init__(self, input_size: int, output_sizes: Sequence[int], max_adapters: int, max_rank: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        if input_size % 8 or any(w % 8 for w in output_sizes):
            raise ValueError(f"adapters need widths that are multiples of 8, not {input_size} and {list(output_sizes)}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"adapters are bf16 or fp16, not {dtype}")
        if max_adapters < 1 or not 1 <= max_rank <= 256:
            raise ValueError("adapters need at least one slot and a rank between 1 and 256")
        self.output_sizes: List[int] = list(output_sizes)
        self.max_adapters, self.rank = int(max_adapters), (int(max_rank) + 7) // 8 * 8
        S, N = len(self.output_sizes), sum(self.output_sizes)
        zeros = lambda *s, dt=dtype: nn.Parameter(torch.zeros(*s, dtype=dt, device=device), requires_grad=False)  # noqa: E731
        self.a = zeros(max_adapters, S * self.rank, input_size)
        self.b = zeros(max_adapters, N, self.rank)
        self.scale = zeros(max_adapters, dt=torch.float32)

    def set_adapter(self, slot: int, lora_a: Union[torch.Tensor, Sequence[Optional[torch.Tensor]]],
                    lora_b: Union[torch.Tensor, Sequence[Optional[torch.Tensor]]], scaling: float = 1.0) -> None:
        """``lora_a`` [rank, input_size] and ``lora_b`` [width, rank], as checkpoints hold them; for a stacked
        projection one of each per shard, None where the adapter leaves a shard alone."""
        lora_a = [lora_a] if isinstance(lora_a, torch.Tensor) else list(lora_a)
        lora_b = [lora_b] if isinstance(lora_b, torch.Tensor) else list(lora_b)
        self._check_slot(slot)
        S, n0 = len(self.output_sizes), 0
        if len(lora_a) != S or len(lora_b) != S:
            raise ValueError(f"set_adapter: {S} shards want as many pairs of matrices")
        for a, b, width in zip(lora_a, lora_b, self.output_sizes):
            if (a is None) != (b is None):
                raise ValueError("set_adapter: the matrices of a shard come together")
            if a is not None and (a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.a.shape[2] or
                                  tuple(b.shape) != (width, a.shape[0]) or a.shape[0] > self.rank):
                raise ValueError(f"set_adapter: [rank, {self.a.shape[2]}] and [{width}, rank] with a rank up to "
                                 f"{self.rank}, not {tuple(a.shape)} and {tuple(b.shape)}")
        new_a, new_b = torch.zeros_like(self.a.data[slot]), torch.zeros_like(self.b.data[slot])
        for j, (a, b, width) in enumerate(zip(lora_a, lora_b, self.output_sizes)):
            if a is not None:
                k = a.shape[0]
                new_a[j * self.rank:j * self.rank + k].copy_(a)
                new_b[n0:n0 + width, :k].copy_(b)
            n0 += width
        self.a.data[slot].copy_(new_a)   # all at once: what was given may lie in this slot
        self.b.data[slot].copy_(new_b)
        self.scale.data[slot] = float(scaling)

    def clear(self, slot: int) -> None:
        self._check_slot(slot)
        for t in (self.a, self.b, self.scale):
            t.data[slot].zero_()

    def _check_slot(self, slot: int) -> None:
        if not 0 <= slot < self.max_adapters:
            raise ValueError(f"adapter slot {slot} outside [0, {self.max_adapters})")

    def add_to(self, base: torch.Tensor, x: torch.Tensor, batch: AdapterBatch) -> torch.Tensor:
        """Adds each token's update to ``base``, the shared product of ``x``, in place."""
        if batch.max_adapters != self.max_adapters:
            raise ValueError(f"a batch of {batch.max_adapters} adapters for a layer with {self.max_adapters}")
        return ops.adapter_linear(x, base, self.a.data, self.b.data, batch.plan, self.scale.data,
                                  slices=self.output_sizes, out=base)
