"""Keys and values of decoder attention held in 8 bits, and the operators that write, read, attend to and evict them.

The cache is (N, H, capacity, E) codes, int8 or float8_e4m3fn, with one float32 scale for `block` consecutive tokens
of a head: a value is code * scale. A scale is the largest |value| of its block / 127 (int8) or / 448 (e4m3), rounded
up to the next bfloat16; a code is the exact quotient to nearest, ties to even. A block that a non-finite value
enters reads as NaN.

A cache is storage only. How many tokens each sequence holds is the caller's int32 tensor `lengths` (N,), on the cache's
device, and the operators read it there: nothing is copied to the host, and a decode step can be captured in a CUDA
graph and replayed while the lengths grow::

    cache = QuantizedKVCache(batch, kv_heads, capacity, head_dim, dtype=torch.int8, block=64, device="cuda")
    kv_cache_append(cache, k, v, lengths)             # behind what the sequences hold
    lengths += k.shape[2]
    out = kv_cache_attention(q, cache, lengths, weights=seen)   # q: the last tokens; seen: what each token got, added up
    cache, lengths, seen, _ = kv_cache_evict(cache, lengths, seen, budget=4096, recent=512)

Lengths below 0 count as 0 and those above the capacity as the capacity; slots behind a length are never read. The
operators run on the current stream of the cache's device, whichever device is current. They have no derivative:
tensors that require a gradient (outside torch.no_grad()) and forward-mode duals are refused. torch.compile breaks its
graph at them.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Tuple, Union

import torch

from . import _host
from .dtensor import DeviceMesh, DTensor, Placement, cuda_device_of


class QuantizedKVCache:
    """An 8-bit key/value cache of `batch` sequences, zero-filled. `capacity`, in tokens, is a multiple of `block` (32, 64
    or 128 tokens that share a scale); `head_dim` a multiple of 16 up to 256; `dtype` torch.int8 or
    torch.float8_e4m3fn. Attributes: key, value, key_scale, value_scale (the tensors), batch, kv_heads, capacity,
    head_dim, block, dtype, device."""

    __slots__ = ("_c", "key", "value", "key_scale", "value_scale", "batch", "kv_heads", "capacity", "head_dim", "block",
                 "dtype", "device")

    def __init__(self, batch: int, kv_heads: int, capacity: int, head_dim: int, dtype: torch.dtype = torch.int8,
                 block: int = 64, device: Union[str, torch.device] = "cuda"):
        self._adopt(_host.QuantizedKVCache.empty(batch, kv_heads, capacity, head_dim, dtype, block, torch.device(device)))

    @classmethod
    def from_tensors(cls, key: torch.Tensor, value: torch.Tensor, key_scale: torch.Tensor,
                     value_scale: torch.Tensor) -> "QuantizedKVCache":
        """A cache over existing contiguous tensors, which it shares: codes (N, H, capacity, E) and scales
        (N, H, capacity / block). Codes are taken as the operators write them (no float8 NaN below a length)."""
        c = cls.__new__(cls)
        c._adopt(_host.QuantizedKVCache(key, value, key_scale, value_scale))
        return c

    def _adopt(self, c) -> None:
        self._c = c
        for name in ("key", "value", "key_scale", "value_scale", "batch", "kv_heads", "capacity", "head_dim", "block"):
            setattr(self, name, getattr(c, name))
        self.dtype, self.device = self.key.dtype, self.key.device

    def __repr__(self) -> str:
        return (f"QuantizedKVCache(batch={self.batch}, kv_heads={self.kv_heads}, capacity={self.capacity}, "
                f"head_dim={self.head_dim}, dtype={self.dtype}, block={self.block}, device={str(self.device)!r})")


def kv_cache_append(cache: QuantizedKVCache, key: torch.Tensor, value: torch.Tensor, lengths: torch.Tensor,
                    counts: Optional[torch.Tensor] = None) -> None:
    """Write new keys and values (N, H, T, E), bfloat16 or float16, behind the lengths[n] tokens that each sequence holds
    (the first counts[n] <= T of them where `counts` is given: a padded batch). The scale of a block that is still
    filling grows with its tokens; when it does, the codes of its earlier tokens are rounded again to the new scale.
    Tokens that would fall behind the capacity are not written. `lengths` is left to the caller, who advances it."""
    _host.kv_cache_append(cache._c, key, value, lengths, counts)


def kv_cache_read(cache: QuantizedKVCache, lengths: torch.Tensor, first: Union[int, torch.Tensor] = 0,
                  count: Optional[int] = None, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(key, value) of the tokens first .. first + count of every sequence as values, (N, H, count, E); zeros outside
    0 .. lengths[n]. `first` is a number or an int32 tensor (N,); `count` defaults to the rest of the capacity (for a
    tensor `first`: to the capacity). float32 is exact, bfloat16 and float16 are rounded once."""
    if isinstance(first, torch.Tensor):
        return _host.kv_cache_read(cache._c, lengths, first, 0, cache.capacity if count is None else count, dtype)
    if first < 0:
        raise ValueError("kv_cache_read: first must not be negative")
    if count is None:
        count = max(cache.capacity - first, 0)
    return _host.kv_cache_read(cache._c, lengths, None, first, count, dtype)


def kv_cache_attention(query: torch.Tensor, cache: QuantizedKVCache, lengths: torch.Tensor,
                       counts: Optional[torch.Tensor] = None, is_causal: bool = True, scale: Optional[float] = None,
                       weights: Optional[torch.Tensor] = None, accumulate: bool = True, return_lse: bool = False):
    """Softmax attention of query (N, Hq, T, E), bfloat16 or float16, over the lengths[n] cached tokens of each sequence:
    (N, Hq, T, E) in query's type. Hq is a multiple of the cache's heads, and head j reads key head
    j // (Hq // H). The queries are the last T (counts[n] where `counts` is given) of the lengths[n] tokens, which
    were appended before: with `is_causal` query i sees the first lengths[n] - T + i + 1. Queries that see nothing, and
    those behind counts[n], give zeros. `scale` defaults to 1 / sqrt(E).

    `weights`, a float32 tensor (N, H, capacity), takes the sum of each cached token's softmax weights over the
    queries and the query heads of its key head, for the tokens below lengths[n] (what kv_cache_evict goes by): added,
    or written where `accumulate` is False. A slot that a new token takes keeps what it had: set it to 0 first, or
    start from zeros. With `return_lse` also the log-sum-exp of the scaled scores, float32 (N, Hq, T), -inf for a
    query that sees nothing. The same inputs give the same bits.

    Scores, sums and outputs are fp32. A softmax weight is rounded to fp16 for the product with the values: 11 significant
    bits down to 2^-24 of the largest among the 32 tokens that share its step (up to 32 queries a key head, or heads above
    128 elements) or, times its value scale, among all that the query sees (more queries). Weights below 2^-110 of the
    largest may count as 0. NaN in a block (a non-finite value was appended) reaches the queries that see the block and no
    others; a query with an infinity or NaN gives NaN, and so do the weights of what it sees.

    Workspace: up to 1 GiB for weights of up to 16 queries a key head, by the cache's capacity; for those of more a copy of
    the queries in fp16."""
    s = 1.0 / math.sqrt(cache.head_dim) if scale is None else scale
    out, lse = _host.kv_cache_attention(query, cache._c, lengths, counts, is_causal, s, weights, accumulate, return_lse)
    return (out, lse) if return_lse else out


def kv_cache_evict(cache: QuantizedKVCache, lengths: torch.Tensor, weights: torch.Tensor, budget: int, recent: int = 0,
                   out: Optional[QuantizedKVCache] = None):
    """Cut every sequence back to at most `budget` tokens: in each head the last `recent` stay, and of the others those
    with the largest `weights` (N, H, capacity), ties to the lowest position and NaN above all; they keep their order. The
    kept tokens go to the front of `out`, a cache that shares no memory with `cache` (default: a new one of the budget rounded up to
    blocks), in blocks that are scaled anew. Returns (out, lengths, weights, kept): the new cache's lengths (N,) and
    weights (N, H, out.capacity), 0 behind the kept tokens, and the kept positions (N, H, budget), -1 behind the last."""
    if out is None:
        most = max(-(-budget // cache.block), 1) * cache.block
        out = QuantizedKVCache(cache.batch, cache.kv_heads, most, cache.head_dim, cache.dtype, cache.block, cache.device)
    new_lengths, new_weights, kept = _host.kv_cache_evict(cache._c, lengths, weights, budget, recent, out._c)
    return out, new_lengths, new_weights, kept


class DistributedKVCache:
    """The 8-bit cache of a decoder on a device mesh: every device holds a QuantizedKVCache of its part of (batch,
    kv_heads, capacity, head_dim) under `placements`, where a mesh dim may shard the batch (Shard(0)) or the heads
    (Shard(1): the placement after the Ulysses swap), evenly, or replicate. Every append adds as many tokens to all
    sequences: a ragged batch uses a QuantizedKVCache and counts. It keeps the lengths and, with
    `track_weights`, what evict goes by. scaled_dot_product_attention_with_cp(..., kv_cache=cache) appends and attends.

    Attributes: locals (QuantizedKVCache of each device id), lengths and weights (tensors of each device id),
    max_length (no sequence holds more tokens; known without asking the devices).

    A step of single tokens can be captured in a CUDA graph. max_length counts calls: add a step's tokens to it for each
    replay, and replay no step for which the capacity has no room (its tokens would not be written). Eviction moves the
    cache to new tensors, so it is not captured, and graphs captured before it are of the old ones."""

    def __init__(self, device_mesh: DeviceMesh, placements: Sequence[Placement], batch: int, kv_heads: int, capacity: int,
                 head_dim: int, dtype: torch.dtype = torch.int8, block: int = 64, track_weights: bool = False):
        self.device_mesh = device_mesh
        shape, ids = list(device_mesh.shape), device_mesh.ids
        names = _host.normalize([repr(p) for p in placements], shape, ids, 4)
        self.placements = [Placement(p) for p in names]
        self.shape = (batch, kv_heads, capacity, head_dim)
        parts = [1, 1]
        for size, p in zip(shape, self.placements):
            if p.is_shard() and not p.has_sub_split_coordinates() and p.get_shard_index() in (0, 1):
                parts[p.get_shard_index()] *= size
            elif not p.is_replicate():
                raise ValueError(f"DistributedKVCache: a mesh dim shards the batch or the heads or replicates, not {p}")
        if batch % parts[0] or kv_heads % parts[1]:
            raise ValueError(f"DistributedKVCache: batch {batch} and heads {kv_heads} do not divide evenly into "
                             f"{parts[0]} and {parts[1]} parts")
        self.max_length = 0
        self.locals: Dict[int, QuantizedKVCache] = {}
        self.lengths: Dict[int, torch.Tensor] = {}
        self.weights: Dict[int, torch.Tensor] = {}
        for gid, s in _host.compute_local_shapes(list(self.shape), shape, ids, names).items():
            dev = torch.device("cuda", cuda_device_of(gid))
            self.locals[gid] = QuantizedKVCache(s[0], s[1], capacity, head_dim, dtype, block, dev)
            self.lengths[gid] = torch.zeros(s[0], dtype=torch.int32, device=dev)
            if track_weights:
                self.weights[gid] = torch.zeros(s[:3], dtype=torch.float32, device=dev)

    def _check(self, t: DTensor, name: str, placements: Sequence[Placement]) -> None:
        """That `t`, which will come with `placements`, fits the cache on every device."""
        if (t.device_mesh is not self.device_mesh and t.device_mesh != self.device_mesh) or \
                list(placements) != self.placements:
            raise ValueError(f"DistributedKVCache: {name} is {list(placements)} on {t.device_mesh}, the cache "
                             f"{self.placements} on {self.device_mesh}")
        if len(t.shape) != 4 or t.shape[0] != self.shape[0] or t.shape[3] != self.shape[3]:
            raise ValueError(f"DistributedKVCache: {name} {t.shape} does not fit {self.shape}")
        if t.placements == self.placements:  # as it comes: every part in its cache's proportion
            shapes = [(c.batch, t.shape[1] * c.kv_heads // self.shape[1], t.shape[2], t.shape[3])
                      for c in self.locals.values()]
        else:
            of = _host.compute_local_shapes(list(t.shape), list(self.device_mesh.shape), self.device_mesh.ids,
                                            [repr(p) for p in t.placements])
            shapes = [of[gid] for gid in self.locals]
        parts = t.locals
        _host.kv_cache_check_rows([c._c for c in self.locals.values()], [parts[gid] for gid in self.locals], shapes,
                                  "DistributedKVCache", name)

    def _check_new(self, key: DTensor, value: DTensor, placements: Sequence[Placement]) -> None:
        self._check(key, "key", placements)
        self._check(value, "value", placements)
        if key.shape != value.shape or key.shape[1] != self.shape[1]:
            raise ValueError(f"DistributedKVCache: key {key.shape} and value {value.shape} do not fit {self.shape}")
        keys, values = key.locals, value.locals
        if any(keys[gid].dtype != values[gid].dtype for gid in self.locals):
            raise TypeError("DistributedKVCache: key and value differ in type")
        if self.max_length + key.shape[2] > self.shape[2]:
            raise ValueError(f"DistributedKVCache: {key.shape[2]} more tokens than {self.max_length} do not fit the "
                             f"capacity of {self.shape[2]}; evict first")

    def _check_query(self, query: DTensor, scale: Optional[float], placements: Sequence[Placement]) -> None:
        self._check(query, "query", placements)
        if query.shape[1] == 0 or query.shape[1] % self.shape[1]:
            raise ValueError(f"DistributedKVCache: query {query.shape} does not fit {self.shape}")
        if scale is not None and not math.fabs(scale) <= torch.finfo(torch.float32).max:
            raise ValueError("DistributedKVCache: scale must be finite")

    def _append(self, key: DTensor, value: DTensor) -> None:
        for gid, cache in self.locals.items():
            kv_cache_append(cache, key.local(gid), value.local(gid), self.lengths[gid])
            with torch.cuda.device(cache.device):
                self.lengths[gid] += key.shape[2]
        self.max_length += key.shape[2]

    def _attend(self, query: DTensor, is_causal: bool, scale: Optional[float]) -> DTensor:
        out = {gid: kv_cache_attention(query.local(gid), cache, self.lengths[gid], is_causal=bool(is_causal), scale=scale,
                                       weights=self.weights.get(gid)) for gid, cache in self.locals.items()}
        return DTensor(out, self.device_mesh, query.placements, query.shape)

    def append(self, key: DTensor, value: DTensor) -> None:
        """Append T tokens (batch, kv_heads, T, head_dim) to every sequence. What is refused is refused before anything
        is written on any device."""
        self._check_new(key, value, key.placements)
        self._append(key, value)

    def attend(self, query: DTensor, is_causal: bool = True, scale: Optional[float] = None) -> DTensor:
        """Attention of the last T tokens' queries (batch, query_heads, T, head_dim), as kv_cache_attention; adds to the
        weights where they are tracked."""
        self._check_query(query, scale, query.placements)
        return self._attend(query, is_causal, scale)

    def evict(self, budget: int, recent: int = 0) -> None:
        """kv_cache_evict on every device, by the tracked weights; the capacity stays."""
        if not self.weights:
            raise ValueError("DistributedKVCache: evict needs track_weights=True")
        if not 0 <= recent <= budget <= self.shape[2]:
            raise ValueError("DistributedKVCache: 0 <= recent <= budget <= capacity")
        for cache in self.locals.values():
            with torch.cuda.device(cache.device):
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("DistributedKVCache: evict moves the cache to new tensors and cannot be captured; "
                                       "capture kv_cache_evict")
        done = {}
        for gid, cache in self.locals.items():
            into = QuantizedKVCache(cache.batch, cache.kv_heads, cache.capacity, cache.head_dim, cache.dtype, cache.block,
                                    cache.device)
            done[gid] = kv_cache_evict(cache, self.lengths[gid], self.weights[gid], budget, recent, out=into)
        for gid, (cache, lengths, weights, _) in done.items():  # of all devices or, where one fails, of none
            self.locals[gid], self.lengths[gid], self.weights[gid] = cache, lengths, weights
        self.max_length = min(self.max_length, budget)
