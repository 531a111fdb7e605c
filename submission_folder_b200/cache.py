"""Decode-side KV caches: each KV head once, in the model's dtype (``DistinctKVCache``) or in
8 bits in blocks of a shared pool (``PagedKVCache``).

After ``CircuitKVCluster.update_kv`` the reference's attention forward hands the
compressed K / V to ``past_key_value.update(key, value, layer_idx, cache_kwargs)``
(KVCache-Factory/pyramidkv/llama_model.py:2918-2928) and, at every decode step, the new
token's K / V the same way (llama_model.py:2931).  Its forward calls ``repeat_kv`` before
the cache, so an HF ``DynamicCache`` there stores every KV head ``num_key_value_groups``
times (4 times for Llama-3-8B).

``DistinctKVCache`` has the same ``update`` / ``get_seq_length`` / ``get_usable_length``
surface but keeps ``[B, Hkv, T, D]``: inputs that carry all query heads (the repeat_kv
layout, whose heads ``g * groups .. g * groups + groups - 1`` are equal) are reduced to
their distinct heads as they come in, and prefill outputs made with
``CircuitKVCluster(distinct_kv_heads=True)`` arrive that way already.  ``update`` returns
the layer's whole cache in the distinct layout for a GQA-aware attention (e.g.
``flash_attn_func`` with ``num_heads_k = Hkv``), or repeated to all query heads with
``repeat=True`` for one that is not.  Memory and decode reads: 1 / groups of the
repeated cache.

``PagedKVCache`` serves many requests from one pool of blocks, holds codes of 8 bits with a
scale for each (block, KV head), and runs a decode step on the device: block tables, rotary
positions, cache write and attention are sm_100a kernels (``ops.block_tables`` and those after
it), with no host synchronisation, so a step can be captured in a CUDA graph.
"""

from __future__ import annotations

from typing import Dict, List, NamedTuple, Optional, Sequence, Tuple

import torch

from . import ops


class DistinctKVCache:
    def __init__(self, num_key_value_heads: int, num_key_value_groups: int, repeat: bool = False):
        if num_key_value_groups < 1 or num_key_value_heads < 1:
            raise ValueError("num_key_value_heads and num_key_value_groups must be >= 1")
        self.kv_heads = int(num_key_value_heads)
        self.groups = int(num_key_value_groups)
        self.repeat = bool(repeat)
        self.key_cache: List[torch.Tensor] = []
        self.value_cache: List[torch.Tensor] = []
        self._seen_tokens = 0

    def _distinct(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() != 4:
            raise ValueError("expected [batch, heads, tokens, head_dim]")
        if x.shape[1] == self.kv_heads:
            return x
        if x.shape[1] == self.kv_heads * self.groups:
            return x[:, :: self.groups]   # the repeat_kv layout: equal heads in groups
        raise ValueError(f"expected {self.kv_heads} or {self.kv_heads * self.groups} heads, got {x.shape[1]}")

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
               cache_kwargs: Optional[Dict] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Appends this call's tokens to layer ``layer_idx`` and returns its whole cache."""
        k = self._distinct(key_states)
        v = self._distinct(value_states)
        if layer_idx == 0:
            self._seen_tokens += key_states.shape[-2]
        if layer_idx < len(self.key_cache):
            self.key_cache[layer_idx] = torch.cat([self.key_cache[layer_idx], k], dim=-2)
            self.value_cache[layer_idx] = torch.cat([self.value_cache[layer_idx], v], dim=-2)
        else:
            while len(self.key_cache) < layer_idx:   # layers this rank does not hold stay empty
                self.key_cache.append(torch.empty(0))
                self.value_cache.append(torch.empty(0))
            self.key_cache.append(k.contiguous())
            self.value_cache.append(v.contiguous())
        return self.layer(layer_idx)

    def layer(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor]:
        k, v = self.key_cache[layer_idx], self.value_cache[layer_idx]
        if self.repeat and self.groups > 1:
            return (k.repeat_interleave(self.groups, dim=1), v.repeat_interleave(self.groups, dim=1))
        return k, v

    def get_seq_length(self, layer_idx: int = 0) -> int:
        if layer_idx >= len(self.key_cache) or self.key_cache[layer_idx].dim() != 4:
            return 0
        return self.key_cache[layer_idx].shape[-2]

    def get_usable_length(self, new_seq_length: int, layer_idx: int = 0) -> int:
        return self.get_seq_length(layer_idx)

    def __len__(self) -> int:
        return len(self.key_cache)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.key_cache + self.value_cache)


class CacheStep(NamedTuple):
    """A step of a ``PagedKVCache``: its block tables (``ops.TableStep``) and the most query
    tokens of a request."""

    tables: ops.TableStep
    max_q: int


class PagedKVCache:
    """An 8-bit decode cache for ``max_requests`` requests of up to ``max_tokens`` cached tokens
    each, over one pool of ``num_blocks`` blocks shared by all of them (and by all layers: a block
    id stands for the same block of every layer).

    A decode step is ``step`` once, then ``decode`` (rotary positions, write, attention) or its
    parts once per layer::

        step = cache.step(new)                       # new: int32 [max_requests] on the device
        for layer in range(num_layers):
            out = cache.decode(layer, q, k, v, step)   # q [T, H, D], k / v [T, Hkv, D]

    A prompt whose layers were compressed by ``CircuitKVCluster.update_kv`` enters with ``admit``.
    ``inv_freq`` / ``factor`` / ``interleaved``: rotary positions of ``decode`` (``ops.rotary``); without
    ``inv_freq``, ``decode`` takes queries and keys that are rotated already.
    """

    def __init__(self, num_layers: int, num_blocks: int, max_requests: int, max_tokens: int, num_key_value_heads: int,
                 head_dim: int = 128, block_size: int = 32, dtype: torch.dtype = torch.float8_e4m3fn,
                 inv_freq: Optional[torch.Tensor] = None, factor: float = 1.0, interleaved: bool = False,
                 device="cuda"):
        if min(num_layers, num_blocks, max_requests, max_tokens, num_key_value_heads) < 1:
            raise ValueError("layers, blocks, requests, tokens and heads must be >= 1")
        if block_size not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise ValueError("block_size must be 16, 32, 64 or 128 and head_dim 64 or 128")
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise ValueError("dtype must be float8_e4m3fn or int8")
        self.block_size, self.kv_heads = int(block_size), int(num_key_value_heads)
        shape = (num_layers, num_blocks, num_key_value_heads)
        self.k = torch.zeros(*shape, block_size, head_dim, dtype=torch.int8, device=device).view(dtype)
        self.v = torch.zeros(*shape, block_size, head_dim, dtype=torch.int8, device=device).view(dtype)
        self.k_scale = torch.zeros(shape, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros(shape, dtype=torch.float32, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.tables = torch.zeros(max_requests, -(-max_tokens // block_size), **i32)
        self.lens = torch.zeros(max_requests, **i32)
        self.shift = torch.zeros(max_requests, **i32)      # evicted tokens: position = place in the cache + shift
        self.free_list = torch.arange(num_blocks, **i32).flip(0).contiguous()
        self.free_count = torch.full((1,), num_blocks, **i32)
        self.inv_freq = None if inv_freq is None else inv_freq.to(self.lens.device)
        self.factor, self.interleaved = float(factor), bool(interleaved)

    def __len__(self) -> int:
        return self.k.shape[0]

    def layer(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """``(k_cache, v_cache, k_scale, v_scale)`` of a layer, as the ``ops.cache_*`` calls take them."""
        return self.k[layer_idx], self.v[layer_idx], self.k_scale[layer_idx], self.v_scale[layer_idx]

    def step(self, new: torch.Tensor, total: Optional[int] = None, max_q: int = 1) -> CacheStep:
        """Blocks, slots and positions for ``new`` int32 ``[max_requests]`` tokens per request (0: none,
        negative: the request ends and frees its blocks).  ``total``: token rows of this step's
        tensors (default ``max_requests * max_q``, rows past the sum of ``new`` are padding);
        ``max_q``: the most tokens of one request (the attention of a request with more is NaN).  A request
        that does not fit gets none (``step.tables.granted``)."""
        total = self.lens.shape[0] * max_q if total is None else int(total)
        t = ops.block_tables(self.lens, new, self.tables, self.free_list, self.free_count, self.block_size, total,
                             shift=self.shift)
        self.shift.mul_(new >= 0)       # the row's next request begins at position 0
        return CacheStep(t, int(max_q))

    def write(self, layer_idx: int, key_states: torch.Tensor, value_states: torch.Tensor, step: CacheStep) -> None:
        """This step's keys and values ``[T, Hkv, D]`` into layer ``layer_idx``."""
        ops.cache_write(key_states, value_states, *self.layer(layer_idx), step.tables.slots)

    def attend(self, layer_idx: int, query_states: torch.Tensor, step: CacheStep, scale: Optional[float] = None,
               want_lse: bool = False):
        """Attention of this step's queries ``[T, H, D]`` over layer ``layer_idx``; rows of padding and of
        requests that did not fit are zeros."""
        return ops.cache_attention(query_states, *self.layer(layer_idx), self.tables, step.tables.seen, cu=step.tables.cu,
                                   max_q=step.max_q, scale=scale, want_lse=want_lse,
                                   out=torch.zeros_like(query_states, memory_format=torch.contiguous_format))

    def decode(self, layer_idx: int, query_states: torch.Tensor, key_states: torch.Tensor, value_states: torch.Tensor,
               step: CacheStep, scale: Optional[float] = None) -> torch.Tensor:
        """One layer of a decode step: rotary positions, write, attention; ``[T, H, D]``."""
        if self.inv_freq is not None:
            query_states, key_states = ops.rotary(query_states, key_states, step.tables.positions, self.inv_freq,
                                                  interleaved=self.interleaved, factor=self.factor)
        self.write(layer_idx, key_states, value_states, step)
        return self.attend(layer_idx, query_states, step, scale)

    def admit(self, request: int, layers: Sequence[Tuple[torch.Tensor, torch.Tensor]], seen: int) -> CacheStep:
        """Put a prompt into the free row ``request``: ``layers`` are each layer's ``(key_states,
        value_states)`` ``[1, heads, B, D]`` as ``CircuitKVCluster.update_kv`` returns them (each KV head
        once, or in the repeat_kv layout), with the same B in every layer; ``seen``: the prompt's
        length, so that the next token stands at position ``seen``.  A row that is not free, or has no room,
        gets nothing (``step.tables.granted``)."""
        if len(layers) != len(self):
            raise ValueError(f"expected {len(self)} layers, got {len(layers)}")
        kept = layers[0][0].shape[-2]
        rows = []
        for k, v in layers:
            if k.dim() != 4 or k.shape[0] != 1 or k.shape != v.shape or k.shape[-2] != kept:
                raise ValueError("expected [1, heads, tokens, head_dim] with the same tokens in every layer")
            if k.shape[1] % self.kv_heads:
                raise ValueError(f"expected a multiple of {self.kv_heads} heads, got {k.shape[1]}")
            groups = k.shape[1] // self.kv_heads
            rows.append((k[0, ::groups].transpose(0, 1), v[0, ::groups].transpose(0, 1)))
        if seen < kept:
            raise ValueError("seen counts the kept tokens too")
        for i, (k, v) in enumerate(rows):      # what ``write`` would refuse, before any block is taken
            ops.check_rows(k, v, *self.layer(i))
        new = torch.zeros_like(self.lens)
        free = self.lens[request] == 0
        new[request] = torch.where(free, kept, 0)
        step = self.step(new, total=kept, max_q=kept)
        self.shift[request] = torch.where(free & (step.tables.granted[request] == kept), seen - kept, self.shift[request])
        for i, (k, v) in enumerate(rows):
            self.write(i, k, v, step)
        return step

    def slots(self, request: int, tokens: int) -> torch.Tensor:
        """Slots of the first ``tokens`` tokens of a request (int64 ``[tokens]``)."""
        if not 0 <= tokens <= self.tables.shape[1] * self.block_size:
            raise ValueError(f"a request holds at most {self.tables.shape[1] * self.block_size} tokens, got {tokens}")
        at = torch.arange(tokens, device=self.lens.device)
        return self.tables[request].long()[at // self.block_size] * self.block_size + at % self.block_size

    def read(self, layer_idx: int, request: int, tokens: int, dtype: torch.dtype = torch.bfloat16):
        """The first ``tokens`` keys and values of a request as ``[1, Hkv, tokens, D]`` of ``dtype``, for
        another round of ``update_kv``."""
        k, v = ops.cache_read(*self.layer(layer_idx), self.slots(request, tokens), dtype)
        return k.transpose(0, 1).unsqueeze(0), v.transpose(0, 1).unsqueeze(0)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))
