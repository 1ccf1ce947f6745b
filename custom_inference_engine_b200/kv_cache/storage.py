"""Paged K/V pools with the reference KVStorage interface (kv_cache/storage.py:4-141).

Layout per layer: ``(n_pages, H_kv, page_size, head_dim)`` for K and for V,
``n_pages = ceil(max_cache_len / page_size)``; ``lens (n_slots,)`` int64,
``block_table (n_slots, n_pages)`` int64 (or int32, ``block_table_dtype``) and
``last_generated (n_slots,)``.
Slot 0 and page 0 are padding. ``decode_update`` / ``mixed_update`` are the
mutating ops ``inference::kv_decode_update`` / ``inference::kv_mixed_update``
(one CUDA launch each for K and V of every token and head); Dynamo sees them
as opaque in-place ops, so they can be captured in CUDA graphs.

``QuantizedKVStorage`` (not in the reference) is the same storage with its pages
in 8 bits, one scale per page, K or V, and kv head: half the bytes per token to
keep and to stream in a decode step.
"""
from __future__ import annotations

import math

import torch

from custom_inference_engine_b200 import native

native.load_ops()
_decode_update = torch.ops.inference.kv_decode_update.default
_mixed_update = torch.ops.inference.kv_mixed_update.default
_q8_decode_update = torch.ops.inference.kv_q8_decode_update.default
_q8_mixed_update = torch.ops.inference.kv_q8_mixed_update.default
_q8_read = torch.ops.inference.kv_q8_read.default


class KVStorage:

    quantized = False

    def __init__(self, config, max_cache_len, page_size, n_slots, device, dtype, *,
                 block_table_dtype=torch.int64):
        """``block_table_dtype`` (keyword only, not in the reference): int64, the
        reference's layout, or int32 (half the bytes per entry; every op of this
        package takes either)."""
        if block_table_dtype not in (torch.int64, torch.int32):
            raise ValueError(f"block_table_dtype must be int64 or int32, not {block_table_dtype}")
        self.config = config
        self.max_cache_len = max_cache_len
        self.page_size = page_size
        self.n_slots = n_slots
        self.device = device
        self.dtype = dtype

        self.n_pages = math.ceil(max_cache_len / page_size)
        self.unused_idx = 0

        self.num_layers = config.num_hidden_layers
        self.num_q_heads = config.num_attention_heads
        self.num_kv_heads = config.num_key_value_heads
        self.head_dim = getattr(config, "head_dim",
                                config.hidden_size // config.num_attention_heads)

        self._allocate_pools()
        self.lens = torch.zeros((n_slots,), dtype=torch.long, device=device)
        self.block_table = torch.zeros((n_slots, self.n_pages), dtype=block_table_dtype,
                                       device=device)
        self.last_generated = torch.zeros((n_slots,), dtype=torch.long, device=device)

    def _allocate_pools(self) -> None:
        shape = (self.n_pages, self.num_kv_heads, self.page_size, self.head_dim)
        self.keys = [torch.zeros(shape, device=self.device, dtype=self.dtype)
                     for _ in range(self.num_layers)]
        self.values = [torch.zeros(shape, device=self.device, dtype=self.dtype)
                       for _ in range(self.num_layers)]

    def mixed_update(self, layer_num: int, pages: torch.Tensor, offsets: torch.Tensor,
                     k_proj: torch.Tensor, v_proj: torch.Tensor) -> None:
        """Token t's K/V rows -> (pages[t], :, offsets[t]) of layer ``layer_num``."""
        _mixed_update(self.keys[layer_num], self.values[layer_num], pages, offsets,
                      k_proj, v_proj)

    def decode_update(self, layer_num: int, slot_ids: torch.Tensor, k_proj: torch.Tensor,
                      v_proj: torch.Tensor) -> None:
        """Each slot's new token -> page block_table[slot, lens//16], offset lens%16."""
        _decode_update(self.keys[layer_num], self.values[layer_num], self.lens, slot_ids,
                       self.block_table, k_proj, v_proj)

    # The padding slot's length is reset with an in-place fill of a one-element
    # slice rather than ``lens[0] = 0``: the latter copies a host scalar, which a
    # CUDA graph capture rejects.
    def decode_advance(self, slot_ids: torch.Tensor) -> None:
        self.lens[slot_ids] += 1
        self.lens[self.unused_idx:self.unused_idx + 1].zero_()

    def mixed_advance(self, slot_ids: torch.Tensor, lens: torch.Tensor) -> None:
        self.lens[slot_ids] += lens
        self.lens[self.unused_idx:self.unused_idx + 1].zero_()

    def reset(self, slot_ids) -> None:
        self.lens[slot_ids] = 0
        self.block_table[slot_ids] = 0


class QuantizedKVStorage(KVStorage):
    """KVStorage with int8 pages (``keys`` / ``values``) and their fp32 ``scales``
    (n_pages, 2, H_kv) per layer. Writes quantise (``include/cie_kv_q8.h`` says how),
    decode attention reads the codes, and mixed passes read the histories they attend
    to back into one fp16 pool of the same page ids, which the layers share
    (``read``). ``dtype`` is that pool's, float16; pages of 16 rows of 64."""

    quantized = True

    def _allocate_pools(self) -> None:
        if self.dtype != torch.float16 or self.page_size != 16 or self.head_dim != 64:
            raise ValueError("8-bit pages need dtype float16, page_size 16 and head_dim 64")
        shape = (self.n_pages, self.num_kv_heads, self.page_size, self.head_dim)

        def zeros(dtype, size=shape):
            return torch.zeros(size, device=self.device, dtype=dtype)

        layers = range(self.num_layers)
        self.keys = [zeros(torch.int8) for _ in layers]
        self.values = [zeros(torch.int8) for _ in layers]
        self.scales = [zeros(torch.float32, (self.n_pages, 2, self.num_kv_heads)) for _ in layers]
        self.read_keys, self.read_values = zeros(self.dtype), zeros(self.dtype)

    def pool(self, layer_num: int):
        """(keys, values, scales) of layer ``layer_num``."""
        return self.keys[layer_num], self.values[layer_num], self.scales[layer_num]

    def mixed_update(self, layer_num: int, pages: torch.Tensor, offsets: torch.Tensor,
                     k_proj: torch.Tensor, v_proj: torch.Tensor) -> None:
        raise RuntimeError("8-bit pages are written by sequence (mixed_update_sequences): the "
                           "rows of a page are quantised together")

    def mixed_update_sequences(self, layer_num: int, cu_seqlens: torch.Tensor,
                               kv_lens: torch.Tensor, slot_ids: torch.Tensor,
                               k_proj: torch.Tensor, v_proj: torch.Tensor) -> None:
        """Rows cu_seqlens[b] .. cu_seqlens[b + 1] -> positions kv_lens[b] onward of slot
        slot_ids[b]."""
        _q8_mixed_update(*self.pool(layer_num), cu_seqlens, kv_lens, slot_ids, self.block_table,
                         k_proj, v_proj)

    def decode_update(self, layer_num: int, slot_ids: torch.Tensor, k_proj: torch.Tensor,
                      v_proj: torch.Tensor) -> None:
        _q8_decode_update(*self.pool(layer_num), self.lens, slot_ids, self.block_table, k_proj,
                          v_proj)

    def read(self, layer_num: int, slot_ids: torch.Tensor, lens: torch.Tensor, starts=None):
        """Positions [starts[b], lens[b]) (from 0 without ``starts``) of every slot as fp16,
        in the pools (``read_keys``, ``read_values``) that all layers share: valid until the
        next layer's read."""
        _q8_read(*self.pool(layer_num), starts, lens, slot_ids, self.block_table, self.read_keys,
                 self.read_values)
        return self.read_keys, self.read_values
