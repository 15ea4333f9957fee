"""The paged KV cache as it is, bf16 or fp16: what an engine holds for the layers that it does not compress, and
what a prompt lies in before it is compressed (`CompressedKVStore.append_from_paged` walks the same pages).

Beside `CompressedPagedKVCache`, with its calls: `write` takes the engine's slot mapping, `decode` its block tables and
lengths.  Beyond them a cache here can be made shorter by what the model attends to:

* an `AttentionLedger` holds, for every cached token and kv head, the softmax weight that the token has received so far:
  `decode` adds a step's, `observe` those of a prompt's last queries;
* `evict` brings every sequence down to a budget: the latest tokens stay, then those that received most.

No counterpart in the reference, which leaves exact pages to its engine.
"""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import _engine as E
from . import _lib

HEAD_DIMS = (64, 128, 256)
DTYPES = (torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class ExactCacheSpec:
    """Page geometry of one layer's exact cache (the role of vLLM's AttentionSpec)."""

    head_dim: int
    num_kv_heads: int
    block_size: int = 16
    dtype: torch.dtype = torch.bfloat16

    def __post_init__(self):
        if self.head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {self.head_dim}: compiled are {HEAD_DIMS}")
        if self.dtype not in DTYPES:
            raise TypeError(f"exact pages hold bfloat16 or float16, not {self.dtype}")
        if self.num_kv_heads < 1 or self.block_size < 1:
            raise ValueError("num_kv_heads and block_size are at least 1")

    @property
    def bytes_per_token(self) -> int:
        """Per kv head: a key row and a value row."""
        return 4 * self.head_dim

    @property
    def page_size_bytes(self) -> int:
        return self.block_size * self.num_kv_heads * self.bytes_per_token

    def num_blocks_for(self, memory_bytes: int) -> int:
        return memory_bytes // self.page_size_bytes

    def max_memory_usage_bytes(self, max_model_len: int) -> int:
        return -(-max_model_len // self.block_size) * self.page_size_bytes


class AttentionLedger:
    """What the cached tokens of `batch` sequences have received: row b belongs to sequence b of the calls.

    mass       (batch, num_kv_heads, max_tokens) fp32, the sum of the softmax weights received, by slot
    positions  (batch, num_kv_heads, max_tokens) int32, the position in the sequence of the tokens in slots below `held`
    held       (batch,) int32, tokens that the last eviction left (0 before the first)
    seen       (batch,) int32, tokens of the sequence up to that eviction; slots from `held` on were filled after it, in
               order, from position `seen` on
    """

    def __init__(self, batch: int, num_kv_heads: int, max_tokens: int, device):
        if min(batch, num_kv_heads, max_tokens) < 1:
            raise ValueError("batch, num_kv_heads and max_tokens are at least 1")
        shape, dev = (batch, num_kv_heads, max_tokens), torch.device(device)
        self._take(torch.zeros(shape, dtype=torch.float32, device=dev), torch.full(shape, -1, dtype=torch.int32, device=dev),
                   torch.zeros(batch, dtype=torch.int32, device=dev), torch.zeros(batch, dtype=torch.int32, device=dev))

    def _take(self, mass, positions, held, seen):
        if mass.dim() != 3 or mass.dtype != torch.float32 or not mass.is_contiguous():
            raise ValueError("mass must be a contiguous (batch, num_kv_heads, max_tokens) float32 tensor")
        if positions.shape != mass.shape or positions.dtype != torch.int32 or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32 tensor of the shape of mass")
        for name, t in (("held", held), ("seen", seen)):
            if t.shape != mass.shape[:1] or t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous (batch,) int32 tensor")
        if len({t.device for t in (mass, positions, held, seen)}) != 1:
            raise ValueError("the tensors of a ledger are on one device")
        self.mass, self.positions, self.held, self.seen = mass, positions, held, seen

    @property
    def _tensors(self):
        return self.mass, self.positions, self.held, self.seen

    @classmethod
    def over(cls, mass: torch.Tensor, positions: torch.Tensor, held: torch.Tensor, seen: torch.Tensor) -> "AttentionLedger":
        """A ledger laid over tensors somebody else allocated; nothing is copied."""
        ledger = cls.__new__(cls)
        ledger._take(mass, positions, held, seen)
        return ledger

    @property
    def batch(self) -> int:
        return self.mass.shape[0]

    @property
    def max_tokens(self) -> int:
        return self.mass.shape[2]

    def reset(self, rows=None) -> None:
        """Forget the sequences `rows` (an index into the batch; None: all): others take their places."""
        at = slice(None) if rows is None else rows
        self.mass[at] = 0.0
        self.positions[at] = -1
        self.held[at] = 0
        self.seen[at] = 0


class PagedKVCache:
    """One layer's exact paged cache over an engine's planes.

    key_cache / value_cache: (num_blocks, block_size, num_kv_heads, head_dim) tensors or views of one layout (for vLLM's
    (2, num_blocks, block_size, H, D) tensor its two halves), head_dim contiguous, rows 16-byte aligned.

    The calls launch on the current stream of the cache's device and synchronise nothing; each has scratch memory of its own,
    so that calls on several streams, and captured ones, do not meet (two that touch the same pages are the caller's to order,
    and so is a stream's first call behind the making of the object, as for any tensor).
    An index that would lead outside the pages is skipped, its token taken for absent, and `status` reports it.
    """

    def __init__(self, spec: ExactCacheSpec, key_cache: torch.Tensor, value_cache: torch.Tensor):
        for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
            E.require_cuda(t, name)
            if t.dtype != spec.dtype:
                raise TypeError(f"{name} must be {spec.dtype} like the spec, not {t.dtype}")
            if t.dim() != 4 or tuple(t.shape[1:]) != (spec.block_size, spec.num_kv_heads, spec.head_dim) or t.shape[0] < 1:
                raise ValueError(f"{name} must be (num_blocks, {spec.block_size}, {spec.num_kv_heads}, {spec.head_dim})")
        # a dimension of one may have any stride
        strides, of_value = ([s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape)] for t in (key_cache, value_cache))
        if key_cache.shape != value_cache.shape or strides != of_value or key_cache.device != value_cache.device:
            raise ValueError("key_cache and value_cache must be of one layout on one device")
        if key_cache.stride(3) != 1 or value_cache.stride(3) != 1 or any(s % 8 for s in strides) or \
                any(t.data_ptr() % 16 for t in (key_cache, value_cache)):
            raise ValueError("rows of the planes must be contiguous and 16-byte aligned")
        self.spec, self.key_cache, self.value_cache = spec, key_cache, value_cache
        self.device = key_cache.device
        self.c = _lib.tq_pages(key_cache.data_ptr(), value_cache.data_ptr(), E.dtype_code(spec.dtype), spec.block_size,
                               key_cache.shape[0], spec.num_kv_heads, spec.head_dim, *strides)
        self.addr = C.addressof(self.c)
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._tickets: dict = {}        # by stream

    @classmethod
    def allocate(cls, spec: ExactCacheSpec, num_blocks: int, device) -> "PagedKVCache":
        """Stand-in for the engine's allocation (tests, stand-alone use)."""
        planes = torch.zeros(2, num_blocks, spec.block_size, spec.num_kv_heads, spec.head_dim, dtype=spec.dtype, device=device)
        return cls(spec, planes[0], planes[1])

    @property
    def num_blocks(self) -> int:
        return self.key_cache.shape[0]

    def status(self) -> int:
        """0, or the first device-side error since the last call (a `tq_status`: an index or a length out of range); reading
        clears it.  Waits for the current stream; calls on others are the caller's to wait for first."""
        code = int(self._status.item())
        if code:
            self._status.zero_()
        return code

    # -- checks of what the native calls do not take ---------------------------
    def _on_device(self, **tensors) -> None:
        for name, t in tensors.items():
            E.require_cuda(t, name)
            if t.device != self.device:
                raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")

    def _batch(self, batch: int, block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int):
        """Block tables and lengths as the kernels take them; raises for what they cannot be."""
        self._on_device(block_tables=block_tables, seq_lens=seq_lens)
        if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] < batch:
            raise ValueError(f"block_tables must be int32 (batch, max_blocks) with at least {batch} rows")
        if seq_lens.dtype != torch.int32 or seq_lens.dim() != 1 or seq_lens.shape[0] < batch:
            raise ValueError(f"seq_lens must be int32 (batch,) with at least {batch} entries")
        if not 0 <= max_seq_len < 2 ** 30:
            raise ValueError(f"max_seq_len {max_seq_len} is out of range")
        if block_tables.shape[1] * self.spec.block_size < max_seq_len:
            raise ValueError(f"block_tables of {block_tables.shape[1]} pages do not hold {max_seq_len} tokens")
        if (block_tables.shape[1] > 1 and block_tables.stride(1) != 1) or (block_tables.shape[0] > 1 and block_tables.stride(0) < block_tables.shape[1]):
            block_tables = block_tables.contiguous()
        return block_tables, seq_lens.contiguous()

    def _ledger(self, ledger: AttentionLedger, batch: int, max_seq_len: int, name: str = "ledger") -> None:
        if not isinstance(ledger, AttentionLedger):
            raise TypeError(f"{name} must be an AttentionLedger")
        if ledger.mass.device != self.device:
            raise ValueError(f"{name} is on {ledger.mass.device}, the cache on {self.device}")
        if ledger.batch < batch or ledger.mass.shape[1] != self.spec.num_kv_heads or ledger.max_tokens < max_seq_len:
            raise ValueError(f"{name} of {tuple(ledger.mass.shape)} does not hold {batch} sequences of {self.spec.num_kv_heads} kv heads "
                             f"and {max_seq_len} tokens")

    def _no_tokens(self, seq_lens: torch.Tensor) -> torch.Tensor:
        """The lengths under a bound of no tokens at all: zeros; any other is out of range and reported, as a kernel would."""
        wrong = (seq_lens != 0).any() & (self._status == 0)
        self._status.masked_fill_(wrong, _lib.TQ_ERR_RANGE)
        return torch.zeros_like(seq_lens)

    def _rows(self, t: torch.Tensor) -> torch.Tensor:
        """`t` as a contiguous tensor on a 16-byte boundary."""
        t = t.contiguous()
        return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)

    # -- the calls ----------------------------------------------------------------
    def write(self, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        """Copy `key` / `value` (T, H, D) into the slots the engine chose: slot = block * block_size + offset, negative =
        padding token to skip (the contract of vLLM's reshape_and_cache).  Slots are distinct."""
        rc = E.host().pages_write(self.addr, self._status, key, value, slot_mapping)
        if rc is None:
            self._on_device(key=key, value=value, slot_mapping=slot_mapping)
            if key.dtype != self.spec.dtype or value.dtype != self.spec.dtype:
                raise TypeError(f"key and value must be {self.spec.dtype} like the cache")
            if key.dim() != 3 or key.shape != value.shape or tuple(key.shape[1:]) != (self.spec.num_kv_heads, self.spec.head_dim):
                raise ValueError(f"expected (T, {self.spec.num_kv_heads}, {self.spec.head_dim}) key and value, got "
                                 f"{tuple(key.shape)} / {tuple(value.shape)}")
            if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.shape[0] < key.shape[0]:
                raise ValueError("slot_mapping must hold one int64 slot per token")
            if key.shape[0] == 0:
                return
            rc = E.host().pages_write(self.addr, self._status, self._rows(key), self._rows(value), slot_mapping.contiguous())
        E.check(_lib.TQ_ERR_SHAPE if rc is None else rc, "tq_pages_write")

    def decode(self, query: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               ledger: Optional[AttentionLedger] = None) -> torch.Tensor:
        """One decode token per sequence, already written as the last of its `seq_lens` tokens: query (B, Qh, D),
        block_tables (B, max_blocks) int32, seq_lens (B,) int32 -> (B, Qh, D); an empty sequence's rows are zero.  Every
        sequence of the step in one launch.  With a ledger the weight every cached token received, summed over the query heads
        of its kv head, is added to the ledger's mass; the call then takes 4 bytes a query head and token of `max_seq_len` for as
        many sequences as 512 MB hold (one at least), and a larger batch goes through in slices of that many."""
        if ledger is not None:
            self._ledger(ledger, 0, 0)
        args = (self.addr, self._status, self._tickets)
        mass = None if ledger is None else ledger.mass
        res = E.host().pages_decode(*args, query, block_tables, seq_lens, max_seq_len, scale, out, mass)
        if type(res) is torch.Tensor:
            return res
        if res is None:
            self._on_device(query=query)
            if query.dtype != self.spec.dtype:
                raise TypeError(f"query must be {self.spec.dtype} like the cache")
            if query.dim() != 3 or query.shape[2] != self.spec.head_dim or query.shape[1] < 1 or query.shape[1] % self.spec.num_kv_heads:
                raise ValueError(f"query {tuple(query.shape)} does not match {self.spec.num_kv_heads} kv heads x {self.spec.head_dim}")
            b = query.shape[0]
            if out is not None:
                self._on_device(out=out)
                if out.shape != query.shape or out.dtype != query.dtype or not out.is_contiguous() or out.data_ptr() % 16:
                    raise ValueError("out must be contiguous, 16-byte aligned and of the query's shape and dtype")
            block_tables, seq_lens = self._batch(b, block_tables, seq_lens, max_seq_len)
            if ledger is not None:
                self._ledger(ledger, b, max_seq_len)
            if b > 0 and max_seq_len == 0:
                self._no_tokens(seq_lens[:b])
            if b == 0 or max_seq_len == 0:
                return torch.zeros_like(query, memory_format=torch.contiguous_format) if out is None else out.zero_()
            res = E.host().pages_decode(*args, self._rows(query), block_tables, seq_lens, max_seq_len, scale, out, mass)
            if type(res) is torch.Tensor:
                return res
        E.check(_lib.TQ_ERR_SHAPE if res is None else res, "tq_pages_decode")

    def observe(self, query: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int,
                ledger: AttentionLedger, scale: Optional[float] = None) -> None:
        """Add to the ledger what the last `window` queries of every sequence give to its cached tokens: query (B, window, Qh,
        D), query i of a sequence of n tokens at position n - window + i, where it sees the tokens up to its own; a query before
        the first token gives nothing.  In a sequence that tokens have been evicted from, the window is one of the tokens that came
        after that (its slots are in order): a query further back gives nothing, and `status` reports it."""
        self._ledger(ledger, 0, 0)
        args = (self.addr, self._status)
        rc = E.host().pages_observe(*args, query, block_tables, seq_lens, max_seq_len, scale, *ledger._tensors)
        if rc is None:
            self._on_device(query=query)
            if query.dtype != self.spec.dtype:
                raise TypeError(f"query must be {self.spec.dtype} like the cache")
            if query.dim() != 4 or query.shape[3] != self.spec.head_dim or query.shape[2] < 1 or query.shape[2] % self.spec.num_kv_heads:
                raise ValueError(f"query {tuple(query.shape)} does not match {self.spec.num_kv_heads} kv heads x {self.spec.head_dim}")
            b = query.shape[0]
            block_tables, seq_lens = self._batch(b, block_tables, seq_lens, max_seq_len)
            self._ledger(ledger, b, max_seq_len)
            if b > 0 and max_seq_len == 0:
                self._no_tokens(seq_lens[:b])
            if b == 0 or query.shape[1] == 0 or max_seq_len == 0:
                return
            rc = E.host().pages_observe(*args, self._rows(query), block_tables, seq_lens, max_seq_len, scale, *ledger._tensors)
        E.check(_lib.TQ_ERR_SHAPE if rc is None else rc, "tq_pages_observe")

    def evict(self, block_tables: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int, ledger: AttentionLedger, budget: int,
              recent: int = 0, out: Optional[AttentionLedger] = None) -> torch.Tensor:
        """Bring every sequence down to `budget` tokens, kv head by kv head, and return the new lengths (B,) int32.

        Of a sequence with more tokens the `recent` latest by position stay, then those with the largest mass (NaN above every
        number; of equal ones the lower slot).  Kept tokens in slots from `budget` on move, in ascending order, into the free
        slots before it, row, mass and position; the order of a cache's tokens means nothing to attention.  Pages behind
        the new length are the engine's to take back.  The ledger is brought up to date in place, or written to `out` (itself or
        another, not one half over it); slots behind the new length have mass 0 and position -1 there.  `seq_lens` is left as it
        is.  Sequences must not share pages (a common prefix would be rearranged for one under the other)."""
        self._ledger(ledger, 0, 0)
        out = ledger if out is None else out
        self._ledger(out, 0, 0, "out")
        if not 0 <= recent <= budget:
            raise ValueError(f"recent ({recent}) lies between 0 and the budget ({budget})")
        native = E.host().pages_evict
        tail = (max_seq_len, budget, recent, *ledger._tensors, *out._tensors)
        res = native(self.addr, self._status, block_tables, seq_lens, *tail)
        if type(res) is torch.Tensor:
            return res
        if res is None:
            b = seq_lens.shape[0] if seq_lens.dim() == 1 else 0
            block_tables, seq_lens = self._batch(b, block_tables, seq_lens, max_seq_len)
            self._ledger(ledger, b, max_seq_len)
            self._ledger(out, b, max_seq_len, "out")
            if budget >= 2 ** 31:
                raise ValueError(f"budget {budget} is out of range")
            if b == 0:
                return torch.zeros_like(seq_lens)
            if max_seq_len == 0:                    # every sequence is empty: the ledgers still agree afterwards
                tail = (1, *tail[1:])
                seq_lens, block_tables = self._no_tokens(seq_lens), block_tables.new_zeros(b, 1)
            res = native(self.addr, self._status, block_tables, seq_lens, *tail)
            if type(res) is torch.Tensor:
                return res
        E.check(_lib.TQ_ERR_SHAPE if res is None else res, "tq_pages_evict")
