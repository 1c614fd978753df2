"""Dense 8-bit KV blocks of a model: the cache that evicts nothing.

The reference's BlockManager and its slot mappings (block_manager.py:8-119,
model_runner.py:594-679, 713-772) keep tables on the host and send them every step;
here the host keeps token counts only, and a step's tables, slots and positions
come from one launch (layers.block_kv.prepare_block_tables).  A step covers
every slot of the manager, the idle ones with no new token, so its launches
have the same shapes from step to step.
"""
from __future__ import annotations

import torch

from ..layers.block_kv import BlockTables, allocate_block_kvcache, prepare_block_tables
from ..utils.context import reset_context, set_context


class BlockKVManager:
    """``num_blocks`` blocks per layer and up to ``max_seqs`` sequences of up to
    ``max_model_len`` tokens.  One table serves all layers: a block id is the
    same rows of each layer's cache.

    For eager steps: the host plans each from its counts, and ``free_count`` is
    another tensor after a step or a release.  A captured step calls
    ``prepare_block_tables`` on tensors of its own."""

    def __init__(self, *, num_layers: int, num_kv_heads: int, head_dim: int, num_blocks: int, max_seqs: int,
                 max_model_len: int, block_size: int = 256, dtype: torch.dtype = torch.int8, device="cuda"):
        self.block_size = block_size
        self.num_blocks = num_blocks
        self.max_model_len = max_model_len
        self.device = torch.device(device)
        self.caches = [allocate_block_kvcache(num_blocks, num_kv_heads, block_size, head_dim, dtype, self.device)
                       for _ in range(num_layers)]
        width = -(-max_model_len // block_size)
        self.block_tables = torch.full((max_seqs, width), -1, device=self.device, dtype=torch.int32)
        self.free_blocks = torch.arange(num_blocks, device=self.device, dtype=torch.int32)
        self.free_count = torch.full((1,), num_blocks, device=self.device, dtype=torch.int32)
        self.free = num_blocks               # the host's copy of free_count
        self.cached = [0] * max_seqs         # tokens each slot's sequence holds
        self.slots: dict[int, int] = {}      # sequence id -> slot
        self._pin = self.device.type == "cuda"

    def attach_attention_modules(self, modules) -> None:
        for layer_id, (module, cache) in enumerate(zip(modules, self.caches, strict=True)):
            module.layer_id = layer_id
            module.block_kv_cache = cache

    def _blocks(self, tokens: int) -> int:
        return -(-tokens // self.block_size)

    def allocate(self, seq_id: int) -> int:
        """The slot of a new sequence."""
        if seq_id in self.slots:
            raise ValueError(f"sequence {seq_id} has a slot already")
        taken = set(self.slots.values())
        for slot in range(len(self.cached)):
            if slot not in taken:
                self.slots[seq_id] = slot
                return slot
        raise RuntimeError(f"all {len(self.cached)} slots are taken")

    def can_append(self, new: dict[int, int]) -> bool:
        """Whether ``new`` tokens by sequence id fit in the free blocks."""
        need = 0
        for seq_id, n in new.items():
            held = self.cached[self.slots[seq_id]]
            need += self._blocks(held + n) - self._blocks(held)
        return need <= self.free

    def begin_step(self, new: dict[int, int], *, num_tokens: int | None = None) -> BlockTables:
        """Blocks, slots and positions of a step that brings ``new[seq_id]``
        tokens of each named sequence (one or more each; the step's rows are the
        sequences' in the order of their slots), and the attention context of
        its forward: ``num_tokens`` rows, more than the tokens for a padded
        batch.  Raises, with nothing changed, if a sequence grows past
        max_model_len or the blocks do not suffice."""
        counts = [0] * len(self.cached)
        for seq_id, n in new.items():
            slot = self.slots[seq_id]
            if n < 1 or self.cached[slot] + n > self.max_model_len:
                raise ValueError(f"sequence {seq_id} cannot go from {self.cached[slot]} by {n} tokens "
                                 f"(max_model_len {self.max_model_len})")
            counts[slot] = n
        total = sum(counts)
        num_tokens = total if num_tokens is None else num_tokens
        if total < 1 or num_tokens < total:
            raise ValueError(f"a step of {total} tokens in {num_tokens} rows")
        if not self.can_append(new):
            raise RuntimeError(f"the step needs more than the {self.free} free blocks")
        lens = torch.tensor([self.cached, counts], dtype=torch.int32, pin_memory=self._pin)
        lens = lens.to(self.device, non_blocking=True)
        step = prepare_block_tables(lens[0], lens[1], self.block_tables, self.free_blocks, self.free_count,
                                    block_size=self.block_size, num_tokens=num_tokens)
        fresh = all(held == 0 or n == 0 for held, n in zip(self.cached, counts))
        self.free -= sum(self._blocks(c + n) - self._blocks(c) for c, n in zip(self.cached, counts))
        self.free_count = step.free_count
        self.cached = [c + n for c, n in zip(self.cached, counts)]
        # prompts that begin here attend to their own rows, before they are rounded to codes
        prefill = max(counts) > 1
        set_context(prefill, step.cu_seqlens, step.cu_seqlens, max(counts), max(self.cached),
                    slot_mapping=step.slot_mapping, context_lens=step.context_lens,
                    block_tables=None if prefill and fresh else self.block_tables)
        return step

    def end_step(self) -> None:
        reset_context()

    def release(self, seq_id: int) -> None:
        """Return a sequence's blocks to the stack and its slot."""
        slot = self.slots.pop(seq_id)
        n = self._blocks(self.cached[slot])
        if n:
            self.free_blocks[self.free:self.free + n].copy_(self.block_tables[slot, :n])
            self.free += n
            self.free_count = torch.full((1,), self.free, device=self.device, dtype=torch.int32)
            self.block_tables[slot, :n].fill_(-1)
        self.cached[slot] = 0
