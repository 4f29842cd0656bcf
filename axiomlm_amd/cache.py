"""StaticKVCache for the MI355X decode path (axiomlm/engine/paged_cache.py:122-462).

Same constructor, tensor layout and counters as the reference:
  cache  (L, 2, B, Hkv, S, hd)      fp16, or uint8 (FP8 E4M3FN) / uint8 hd/2 (INT4)
  scales (L, 2, B, Hkv, S, hd/64)   fp16 for the quantized caches
``k_caches[i]`` / ``v_caches[i]`` are views of ``cache[i, 0]`` / ``cache[i, 1]``.
Writes of new rows (``update``) quantize on the GPU with the reference CPU
quantizer semantics; ``compact_tree_path`` moves accepted tree slots of every
layer with one HIP kernel per call.

``PagedKVCache`` is the cache of several sequences of different lengths: pages of a common pool, handed out as sequences
grow (the role of the reference's PagedKVCache, axiomlm/engine/paged_cache.py:4-120).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Sequence

import torch

from . import _lib
from .kernels.ops import KV_CODES, compact_tree_kv, dequantize_kv_fp8, dequantize_kv_int4
from .kernels.paged import evict_paged_kv, gqa_paged_decode, rope_paged_kv_cache_write


class StaticKVCache:
    def __init__(
        self,
        max_batch_size: int,
        max_seq_len: int,
        n_layer: int,
        n_kv_head: int,
        head_dim: int,
        dtype: torch.dtype = torch.float16,
        device: torch.device | str | None = None,
        ring_buffer: bool = False,
        cache_dtype: str = "fp16",
    ):
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        elif isinstance(device, str):
            device = torch.device(device)
        self.max_batch_size = max_batch_size
        self.max_seq_len = max_seq_len
        self.n_layer = n_layer
        self.n_kv_head = n_kv_head
        self.head_dim = head_dim
        self.ring_buffer = ring_buffer
        self.cache_dtype = cache_dtype.lower()
        if self.cache_dtype not in KV_CODES:
            raise ValueError(f"unsupported cache_dtype {cache_dtype!r}")
        self.num_groups = max(1, head_dim // 64)
        shape5 = (n_layer, 2, max_batch_size, n_kv_head, max_seq_len)
        if self.cache_dtype == "fp8":
            self.cache = torch.zeros((*shape5, head_dim), dtype=torch.uint8, device=device)
        elif self.cache_dtype == "int4":
            self.cache = torch.zeros((*shape5, head_dim // 2), dtype=torch.uint8, device=device)
        else:
            self.cache = torch.empty((*shape5, head_dim), dtype=dtype, device=device)
        if self.cache_dtype == "fp16":
            self.scales = None
            self.k_scales = None
            self.v_scales = None
        else:
            self.scales = torch.zeros((*shape5, self.num_groups), dtype=torch.float16, device=device)
            self.k_scales = [self.scales[i, 0] for i in range(n_layer)]
            self.v_scales = [self.scales[i, 1] for i in range(n_layer)]
        self.k_caches = [self.cache[i, 0] for i in range(n_layer)]
        self.v_caches = [self.cache[i, 1] for i in range(n_layer)]
        self.layer_seq_lens = [0] * n_layer
        self.total_seen_tokens = [0] * n_layer

    @property
    def kv_code(self) -> int:
        return KV_CODES[self.cache_dtype]

    def get_memory_bytes(self) -> int:
        total = self.cache.numel() * self.cache.element_size()
        if self.scales is not None:
            total += self.scales.numel() * self.scales.element_size()
        return total

    @property
    def seq_len(self) -> int:
        return self.total_seen_tokens[0]

    def reset(self):
        for i in range(self.n_layer):
            self.layer_seq_lens[i] = 0
            self.total_seen_tokens[i] = 0

    # ---- writes ---------------------------------------------------------------
    def _write_rows(self, layer: int, k: torch.Tensor, v: torch.Tensor, write_pos: int) -> None:
        """Store k, v (1, Hkv, T, hd) at slots (write_pos + t) % S of batch 0."""
        T = k.shape[2]
        hd = self.head_dim
        kr = k[0].transpose(0, 1).reshape(T, self.n_kv_head * hd).to(torch.float16).contiguous()
        vr = v[0].transpose(0, 1).reshape(T, self.n_kv_head * hd).to(torch.float16).contiguous()
        ks = self.k_scales[layer] if self.scales is not None else None
        vs = self.v_scales[layer] if self.scales is not None else None
        _lib.check(
            _lib.lib().axm_kv_cache_write(
                _lib.ptr(kr), _lib.ptr(vr), self.n_kv_head * hd, T, _lib.ptr(self.k_caches[layer]),
                _lib.ptr(self.v_caches[layer]), _lib.ptr(ks), _lib.ptr(vs), self.kv_code, self.n_kv_head, hd,
                self.max_seq_len, int(write_pos) % self.max_seq_len, _lib.stream_of(self.cache.device)),
            "StaticKVCache.update",
        )

    def _active_views(self, layer: int, n: int):
        kb, vb = self.k_caches[layer][:1, :, :n], self.v_caches[layer][:1, :, :n]
        if self.cache_dtype == "fp8":
            return (dequantize_kv_fp8(kb, self.k_scales[layer][:1, :, :n], self.head_dim),
                    dequantize_kv_fp8(vb, self.v_scales[layer][:1, :, :n], self.head_dim))
        if self.cache_dtype == "int4":
            return (dequantize_kv_int4(kb, self.k_scales[layer][:1, :, :n], self.head_dim),
                    dequantize_kv_int4(vb, self.v_scales[layer][:1, :, :n], self.head_dim))
        return kb, vb

    def update(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor):
        """In-place write of (1, Hkv, T, hd) rows; returns the active (dequantized) views.

        Monotonic and ring-buffer semantics of paged_cache.py:218-361 (batch 1)."""
        if k.shape[0] != 1:
            raise ValueError("the MI355X StaticKVCache path supports batch 1 writes")
        T = k.shape[2]
        seen = self.total_seen_tokens[layer_idx]
        S = self.max_seq_len
        if not self.ring_buffer and seen + T <= S:
            self._write_rows(layer_idx, k, v, seen)
            self.layer_seq_lens[layer_idx] = self.total_seen_tokens[layer_idx] = seen + T
            return self._active_views(layer_idx, seen + T)
        if T >= S:
            self._write_rows(layer_idx, k[:, :, -S:], v[:, :, -S:], 0)
        else:
            self._write_rows(layer_idx, k, v, seen % S)
        active = min(seen + T, S)
        self.layer_seq_lens[layer_idx] = active
        self.total_seen_tokens[layer_idx] = seen + T
        return self._active_views(layer_idx, active)

    def get_quantized_views(self, layer_idx: int):
        k_s = self.k_scales[layer_idx] if self.scales is not None else None
        v_s = self.v_scales[layer_idx] if self.scales is not None else None
        return self.k_caches[layer_idx], self.v_caches[layer_idx], k_s, v_s

    def compact_tree_path(self, write_pos: int, accepted_indices: list[int], new_total_seen: int | None = None):
        """Move accepted tree slots (write_pos + a[m]) % S to (write_pos + m) % S in every layer
        with one race-free HIP pass (paged_cache.py:376-462)."""
        if self.scales is not None and not self.scales.is_contiguous():
            raise RuntimeError("compact_tree_path: cache and scales must be contiguous")
        compact_tree_kv(self.cache, self.scales, write_pos, accepted_indices)
        if new_total_seen is not None:
            active = min(new_total_seen, self.max_seq_len)
            self.total_seen_tokens[:] = [new_total_seen] * self.n_layer
            self.layer_seq_lens[:] = [active] * self.n_layer


class StepTokens(NamedTuple):
    """New tokens of one step, sequence by sequence (int32, on the device)."""

    seq_ids: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


class PagedKVCache:
    """Keys and values of up to ``max_batch_size`` sequences in pages of a common pool.

    cache  (L, 2, P, Hkv, page_size, width)  as StaticKVCache's, a page in the place of a batch entry's slots
    scales (L, 2, P, Hkv, page_size, hd/64)  fp16 for the quantized caches
    block_table (B, max_pages), seq_lens (B,) int32; mass (L, B, Hkv, max_pages * page_size) fp32 with ``account``

    A step: ``tokens = begin_step(counts)`` takes pages for the new tokens; per layer ``write`` stores their keys and
    values and ``attend`` lets one new token per sequence see them.  ``evict`` cuts long sequences to a budget by the
    account that ``attend`` keeps, ``free`` gives a sequence's pages back.  The device tensors keep their addresses, so
    a captured ``write`` / ``attend`` replays after later ``begin_step``s; host bookkeeping is done between steps."""

    def __init__(self, max_batch_size: int, max_seq_len: int, n_layer: int, n_kv_head: int, head_dim: int,
                 n_pages: int | None = None, page_size: int = 64, device: torch.device | str | None = None,
                 cache_dtype: str = "fp16", account: bool = False):
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.cache_dtype = cache_dtype.lower()
        if self.cache_dtype not in KV_CODES:
            raise ValueError(f"unsupported cache_dtype {cache_dtype!r}")
        if head_dim not in (64, 128):
            raise ValueError(f"PagedKVCache requires head_dim 64 or 128, got {head_dim}")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} must be a power of two between 16 and 1024")
        if min(max_batch_size, max_seq_len, n_layer, n_kv_head) < 1:
            raise ValueError("PagedKVCache of an empty shape")
        self.max_batch_size = max_batch_size
        self.n_layer, self.n_kv_head, self.head_dim, self.page_size = n_layer, n_kv_head, head_dim, page_size
        self.max_pages = -(-max_seq_len // page_size)
        self.max_seq_len = self.max_pages * page_size
        self.n_pages = max_batch_size * self.max_pages if n_pages is None else int(n_pages)
        if self.n_pages < 1:
            raise ValueError(f"PagedKVCache of {n_pages} pages")
        shape5 = (n_layer, 2, self.n_pages, n_kv_head, page_size)
        width = head_dim // 2 if self.cache_dtype == "int4" else head_dim
        dtype = torch.float16 if self.cache_dtype == "fp16" else torch.uint8
        self.cache = torch.zeros((*shape5, width), dtype=dtype, device=device)
        self.scales = None if self.cache_dtype == "fp16" else torch.zeros((*shape5, head_dim // 64),
                                                                          dtype=torch.float16, device=device)
        self.k_caches = [self.cache[i, 0] for i in range(n_layer)]
        self.v_caches = [self.cache[i, 1] for i in range(n_layer)]
        self.k_scales = [None if self.scales is None else self.scales[i, 0] for i in range(n_layer)]
        self.v_scales = [None if self.scales is None else self.scales[i, 1] for i in range(n_layer)]
        self.block_table = torch.full((max_batch_size, self.max_pages), -1, dtype=torch.int32, device=device)
        # Rows: cached tokens; the same for sequences with a token in this step, 0 for the others.
        self._lens = torch.zeros((2, max_batch_size), dtype=torch.int32, device=device)
        self.seq_lens, self.step_lens = self._lens
        self.mass = torch.zeros((n_layer, max_batch_size, n_kv_head, self.max_seq_len), dtype=torch.float32,
                                device=device) if account else None
        self.lens = [0] * max_batch_size       # cached tokens
        self.positions = [0] * max_batch_size  # tokens seen, evicted ones too: the next token's position
        self._in_step = [False] * max_batch_size
        self._pages: list[list[int]] = [[] for _ in range(max_batch_size)]
        self._free = list(range(self.n_pages - 1, -1, -1))

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def get_memory_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.cache, self.scales, self.mass) if t is not None)

    def _upload(self, table: bool) -> None:
        if table:
            rows = [p + [-1] * (self.max_pages - len(p)) for p in self._pages]
            self.block_table.copy_(torch.tensor(rows, dtype=torch.int32))
        step = [n if s else 0 for n, s in zip(self.lens, self._in_step)]
        self._lens.copy_(torch.tensor([self.lens, step], dtype=torch.int32))

    def begin_step(self, counts: Sequence[int]) -> StepTokens:
        """Room for ``counts[b]`` new tokens of every sequence b (0: none); their sequences, positions and slots in
        order.  Nothing changes where the pool or a sequence's length does not suffice (RuntimeError)."""
        counts = [int(c) for c in counts]
        if len(counts) != self.max_batch_size or min(counts) < 0:
            raise ValueError(f"begin_step: {len(counts)} counts for {self.max_batch_size} sequences")
        need = [max(0, -(-(n + c) // self.page_size) - len(p)) for n, c, p in zip(self.lens, counts, self._pages)]
        for b, (n, c) in enumerate(zip(self.lens, counts)):
            if n + c > self.max_seq_len:
                raise RuntimeError(f"begin_step: sequence {b} of {n} + {c} tokens passes {self.max_seq_len}")
        if sum(need) > len(self._free):
            raise RuntimeError(f"begin_step: {sum(need)} pages needed, {len(self._free)} free")
        seq, pos, slot = [], [], []
        for b, c in enumerate(counts):
            self._pages[b] += [self._free.pop() for _ in range(need[b])]
            seq += [b] * c
            pos += range(self.positions[b], self.positions[b] + c)
            slot += range(self.lens[b], self.lens[b] + c)
            self.positions[b] += c
            self.lens[b] += c
        self._in_step = [c > 0 for c in counts]
        self._upload(sum(need) > 0)
        dev = self.cache.device
        return StepTokens(*torch.tensor([seq, pos, slot], dtype=torch.int32).to(dev))

    def write(self, layer: int, qkv: torch.Tensor, freqs_cis: torch.Tensor, tokens: StepTokens, q_dim: int,
              qkv_bias: torch.Tensor | None = None) -> None:
        """RoPE of the new tokens' qkv rows (queries in place) and their keys and values into the layer's pages."""
        rope_paged_kv_cache_write(qkv, freqs_cis, self.k_caches[layer], self.v_caches[layer], self.block_table,
                                  tokens.positions, q_dim, self.n_kv_head * self.head_dim, self.head_dim,
                                  slots=tokens.slots, seq_ids=tokens.seq_ids, qkv_bias=qkv_bias,
                                  k_scales=self.k_scales[layer], v_scales=self.v_scales[layer],
                                  kv_dtype=self.cache_dtype)

    def attend(self, layer: int, q: torch.Tensor) -> torch.Tensor:
        """Attention of q (B, Hq, hd), the step's last token of every sequence, over all that the layer holds of it; with
        ``account`` its weights join ``mass``.  Sequences without a token in this step give zeros."""
        return gqa_paged_decode(q, self.k_caches[layer], self.v_caches[layer], self.block_table, self.step_lens,
                                self.k_scales[layer], self.v_scales[layer], self.cache_dtype,
                                None if self.mass is None else self.mass[layer])

    def evict(self, budget: int, recent: int) -> torch.Tensor:
        """Cut every sequence over ``budget`` to it (``evict_paged_kv``) and take back the pages behind it; returns the
        slots that stayed, int32 (L, B, Hkv, budget)."""
        if self.mass is None:
            raise RuntimeError("evict: the cache keeps no account (account=True)")
        kept, _, mass = evict_paged_kv(self.cache, self.scales, self.block_table, self.seq_lens, self.mass, budget,
                                       recent)
        self.mass.copy_(mass)
        for b, n in enumerate(self.lens):
            self._keep(b, min(n, budget))
        self._upload(True)
        return kept

    def _keep(self, seq: int, n: int) -> None:
        self.lens[seq] = n
        pages = -(-n // self.page_size)
        self._free += reversed(self._pages[seq][pages:])
        del self._pages[seq][pages:]

    def free(self, seq: int) -> None:
        """End sequence ``seq``: its pages go back to the pool."""
        self._keep(seq, 0)
        self.positions[seq] = 0
        self._in_step[seq] = False
        if self.mass is not None:
            self.mass[:, seq].zero_()
        self._upload(True)

    def reset(self) -> None:
        for b in range(self.max_batch_size):
            self._keep(b, 0)
            self.positions[b] = 0
            self._in_step[b] = False
        if self.mass is not None:
            self.mass.zero_()
        self._upload(True)
