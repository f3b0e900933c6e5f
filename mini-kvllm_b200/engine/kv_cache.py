"""Host side of the paged KV cache around the kernels: the cache allocation and
per-layer binding of ModelRunner.allocate_kv_cache, the per-step decode metadata of
ModelRunner.prepare_decode, and the tensor-parallel KV-head split.

Reference (heart1128/mini-kvllm, src/myvllm/engine/model_runner.py):
  allocate_kv_cache   204-395  one zeros(2, L, NB, BS, KVH/world, D) tensor; fp8 caches are
                               float8_e4m3fn and int8 caches int8 (247-252); per-tensor
                               scales ones(2, L, 1) fp32 (324-329); per-(token, head) scales
                               ones(2, L, NB, BS, KVH/world) fp32 (330-338); layer l gets
                               views [0, l] / [1, l] (376-395)
  prepare_decode      631-671  context_lens = len(seq) (includes the new token),
                               (decode_metadata restates it; DecodeMetadataBuilder
                               computes it with one copy and one kernel per step)
                               slot = block_table[-1] * BS + last_block_num_tokens - 1,
                               block_tables padded with -1 to the longest table; int64
                               slots and lengths, int32 tables
  KV-head sharding    215      each rank holds num_kv_heads // world_size heads, and the
                               matching num_heads // world_size query heads
                               (models/qwen3.py:27-33)

Not in the reference: decode steps over trees of drafted tokens (tree_metadata, tree_accept,
move_kv_rows around paged_attention_tree) and copies of whole pages (copy_kv_pages), for a
block manager that forks sequences or compacts the cache. Which pages are shared or free
stays the block manager's to know.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Iterable, Optional, Sequence

import torch

from .. import _lib
from ..layers.attention import _INDEX, _DTYPES, _call_packed, _device_index

PER_TOKEN_HEAD = ("fp8_per_token_head", "int8_per_token_head")
QUANTIZED = ("fp8_per_tensor",) + PER_TOKEN_HEAD
KV_CACHE_DTYPES = ("auto",) + QUANTIZED


@dataclass
class KVCache:
    kv: torch.Tensor                      # (2, L, NB, BS, KVH, D)
    k_scale: Optional[torch.Tensor]       # (L, 1) or (L, NB, BS, KVH) fp32 views, or None
    v_scale: Optional[torch.Tensor]
    kv_cache_dtype: str
    block_size: int

    def layer(self, l: int):
        """(k_cache, v_cache, k_scale, v_scale) of layer l."""
        ks = self.k_scale[l] if self.k_scale is not None else None
        vs = self.v_scale[l] if self.v_scale is not None else None
        return self.kv[0, l], self.kv[1, l], ks, vs


def allocate_kv_cache(num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int,
                      head_dim: int, kv_cache_dtype: str = "auto",
                      default_dtype: torch.dtype = torch.bfloat16,
                      device: torch.device | str = "cuda") -> KVCache:
    """One zero-initialised (2, L, NB, BS, KVH, D) cache (model_runner.py:311-314).
    'fp8_per_tensor': float8_e4m3fn pages and (2, L, 1) float32 scales at the calibration
    sentinel 1.0 (324-329). 'fp8_per_token_head' / 'int8_per_token_head': float8_e4m3fn /
    int8 pages and one float32 scale per (page, row, kv head), (2, L, NB, BS, KVH), set to
    1.0 (330-338); the append writes each row's scale."""
    if kv_cache_dtype not in KV_CACHE_DTYPES:
        raise NotImplementedError(f"kv_cache_dtype {kv_cache_dtype!r} is not implemented")
    if kv_cache_dtype == "int8_per_token_head":
        data_dtype = torch.int8
    elif kv_cache_dtype in QUANTIZED:
        data_dtype = torch.float8_e4m3fn
    else:
        data_dtype = default_dtype
    kv = torch.zeros(2, num_layers, num_blocks, block_size, num_kv_heads, head_dim,
                     dtype=data_dtype, device=device)
    ks = vs = None
    if kv_cache_dtype == "fp8_per_tensor":
        buf = torch.ones(2, num_layers, 1, dtype=torch.float32, device=device)
        ks, vs = buf[0], buf[1]
    elif kv_cache_dtype in PER_TOKEN_HEAD:
        buf = torch.ones(2, num_layers, num_blocks, block_size, num_kv_heads, dtype=torch.float32,
                         device=device)
        ks, vs = buf[0], buf[1]
    return KVCache(kv, ks, vs, kv_cache_dtype, block_size)


def bind_kv_cache(modules: Iterable[torch.nn.Module], cache: KVCache) -> int:
    """Injects per-layer cache views (and scales) into every module that has k_cache and
    v_cache attributes, in module order (model_runner.py:376-395). Returns the count."""
    layer = 0
    for m in modules:
        if hasattr(m, "k_cache") and hasattr(m, "v_cache"):
            k, v, ks, vs = cache.layer(layer)
            m.k_cache, m.v_cache = k, v
            m.kv_cache_dtype = cache.kv_cache_dtype
            if ks is not None:
                m.k_scale, m.v_scale = ks, vs
            layer += 1
    return layer


@dataclass
class DecodeMetadata:
    slot_mapping: torch.Tensor   # (B,) int64
    context_lens: torch.Tensor   # (B,) int64
    block_tables: torch.Tensor   # (B, max_blocks) int32, -1 padded


def decode_metadata(block_tables: Sequence[Sequence[int]], seq_lens: Sequence[int],
                    block_size: int, device: torch.device | str = "cuda",
                    pin_memory: bool = False) -> DecodeMetadata:
    """Per-step decode metadata of prepare_decode (model_runner.py:631-671): seq_lens are
    the sequence lengths including the token being decoded; each slot is the last
    token's position inside the last block of the sequence's table."""
    if len(block_tables) != len(seq_lens):
        raise ValueError("one block table per sequence is required")
    slots, lens = [], []
    for bt, n in zip(block_tables, seq_lens):
        if n <= 0 or len(bt) < (n + block_size - 1) // block_size:
            raise ValueError(f"sequence of length {n} needs {(n + block_size - 1) // block_size} blocks, has {len(bt)}")
        last_block_tokens = n - (len(bt) - 1) * block_size
        slots.append(bt[-1] * block_size + last_block_tokens - 1)
        lens.append(n)
    width = max((len(bt) for bt in block_tables), default=0)
    padded = [list(bt) + [-1] * (width - len(bt)) for bt in block_tables]
    pin = pin_memory and torch.cuda.is_available()
    def to(t):
        return t.pin_memory().to(device, non_blocking=True) if pin else t.to(device)
    return DecodeMetadata(
        slot_mapping=to(torch.tensor(slots, dtype=torch.int64)),
        context_lens=to(torch.tensor(lens, dtype=torch.int64)),
        block_tables=to(torch.tensor(padded, dtype=torch.int32).reshape(len(padded), width)))


class DecodeMetadataBuilder:
    """Decode metadata with one host-to-device copy and one kernel per step, instead of
    prepare_decode's per-sequence Python loops and three host tensors
    (model_runner.py:631-671).

    Block tables live in a host mirror indexed by a persistent sequence slot. The block
    manager reports only their changes: `set_table` when a sequence takes a slot,
    `append` when it takes a block. Each step then packs [lengths | tables] into a pinned
    buffer, copies it once, and `mkv_decode_metadata` derives the int64 slot mapping and
    context lengths on the device. The table width is max_blocks, fixed, so every step
    has the same shapes (capturable decode graphs). Two pinned buffers alternate, each
    reused only after its previous copy has completed. The returned tensors are
    overwritten by the next step."""

    def __init__(self, max_seqs: int, max_blocks: int, block_size: int,
                 device: torch.device | str = "cuda"):
        import numpy as np
        from .. import _lib
        self._np, self._lib_mod = np, _lib
        self._lib = _lib.load()
        self.max_seqs, self.max_blocks, self.block_size = max_seqs, max_blocks, block_size
        self.device = torch.device(device)
        n = max_seqs * (1 + max_blocks)
        self._host = [torch.empty(n, dtype=torch.int32, pin_memory=True) for _ in range(2)]
        self._host_np = [h.numpy() for h in self._host]
        self._copied = [None, None]
        self._k = 0
        self._tables = np.full((max_seqs, max_blocks), -1, dtype=np.int32)
        self._nblocks = np.zeros(max_seqs, dtype=np.int64)
        self._packed = torch.empty(n, dtype=torch.int32, device=self.device)
        self._slots = torch.empty(max_seqs, dtype=torch.int64, device=self.device)
        self._lens = torch.empty(max_seqs, dtype=torch.int64, device=self.device)

    def set_table(self, seq: int, table: Sequence[int]) -> None:
        if len(table) > self.max_blocks:
            raise ValueError(f"a table of {len(table)} blocks exceeds max_blocks {self.max_blocks}")
        row = self._tables[seq]
        row[:] = -1
        row[:len(table)] = table
        self._nblocks[seq] = len(table)

    def append(self, seq: int, block: int) -> None:
        n = int(self._nblocks[seq])
        if n >= self.max_blocks:
            raise ValueError(f"sequence slot {seq} already holds max_blocks {self.max_blocks}")
        self._tables[seq, n] = block
        self._nblocks[seq] = n + 1

    def step(self, seqs: Sequence[int], seq_lens: Sequence[int]) -> DecodeMetadata:
        """Metadata of one decode step over sequence slots `seqs` (batch order), with
        lengths including the token being decoded."""
        np = self._np
        B, W = len(seqs), self.max_blocks
        if B > self.max_seqs or len(seq_lens) != B:
            raise ValueError("one length per sequence, at most max_seqs sequences")
        k = self._k
        if self._copied[k] is not None:
            self._copied[k].synchronize()  # the copy that last read this buffer is done
        hv = self._host_np[k]
        idx = np.asarray(seqs, dtype=np.int64)
        hv[:B] = seq_lens
        hv[B:B + B * W].reshape(B, W)[:] = self._tables[idx]
        stream = torch.cuda.current_stream(self.device)
        self._packed[:B * (1 + W)].copy_(self._host[k][:B * (1 + W)], non_blocking=True)
        ev = torch.cuda.Event()
        ev.record(stream)
        self._copied[k] = ev
        self._k ^= 1
        st = self._lib.mkv_decode_metadata(self._packed.data_ptr(), B, W, self.block_size,
                                           self._slots.data_ptr(), self._lens.data_ptr(),
                                           stream.cuda_stream)
        self._lib_mod.check("mkv_decode_metadata", st)
        return DecodeMetadata(slot_mapping=self._slots[:B], context_lens=self._lens[:B],
                              block_tables=self._packed[B:B + B * W].view(B, W))


# ------------------------------------------------------------------ trees of drafted tokens
@dataclass
class TreeMetadata:
    slot_mapping: torch.Tensor   # (total_q,) int64
    context_lens: torch.Tensor   # (B,) int64, the drafted nodes included
    positions: torch.Tensor      # (total_q,) int64
    tree_mask: torch.Tensor      # (total_q, words) int64


@dataclass
class TreeAcceptance:
    num_accepted: torch.Tensor   # (B,) int32
    accepted_nodes: torch.Tensor  # (B, max_path) int32, -1 padded
    tokens: torch.Tensor         # (B, max_path) int64, -1 padded
    context_lens: torch.Tensor   # (B,) int64, cached tokens to keep
    src_slots: torch.Tensor      # (B, max_path) int64, -1: no move
    dst_slots: torch.Tensor      # (B, max_path) int64


def _indices(fn: str, what: str, t: torch.Tensor, dim: int) -> torch.Tensor:
    if t.dtype not in _INDEX or t.dim() != dim:
        raise ValueError(f"{fn}: {what} must be an int32 or int64 tensor of {dim} dimension(s), got "
                         f"{t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _count(fn: str, t: Optional[torch.Tensor], idx: int) -> int:
    """The address of a caller's count of skipped entries (0: none is kept)."""
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.numel() != 1 or t.get_device() != idx:
        raise ValueError(f"{fn}: invalid_count must be one int32 on the same device, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _tree_args(fn: str, parents, cu_seqlens_q, prefix_lens, block_tables, block_size):
    """(checked tensors, the argument list that the tree entry points share)"""
    parents = _indices(fn, "parents", parents, 1)
    cu = _indices(fn, "cu_seqlens_q", cu_seqlens_q, 1)
    prefix = _indices(fn, "prefix_lens", prefix_lens, 1)
    tables = block_tables
    tt = _INDEX.get(tables.dtype)
    if tt is None or tables.dim() != 2:
        raise ValueError(f"{fn}: block_tables must be a two-dimensional int32 or int64 tensor")
    stride = tables.stride()
    if stride[1] != 1:
        tables = tables.contiguous()
        stride = tables.stride()
    rows, width = tables.shape
    B = prefix.numel()
    if cu.numel() != B + 1 or rows < B:
        raise ValueError(f"{fn}: cu_seqlens_q/block_tables do not match {B} sequences")
    if not 0 < block_size < 1 << 31:  # (32 bits in the C call)
        raise ValueError(f"{fn}: block_size must be positive and below 2^31 (got {block_size})")
    return (parents, cu, prefix, tables), (
        parents.data_ptr(), _INDEX[parents.dtype], cu.data_ptr(), _INDEX[cu.dtype], prefix.data_ptr(),
        _INDEX[prefix.dtype], tables.data_ptr(), tt, stride[0], width, block_size, B, parents.numel())


def tree_metadata(parents: torch.Tensor, cu_seqlens_q: torch.Tensor, prefix_lens: torch.Tensor,
                  block_tables: torch.Tensor, block_size: int, max_nodes: int,
                  invalid_count: Optional[torch.Tensor] = None) -> TreeMetadata:
    """Metadata of a decode step over trees of drafted tokens, in one kernel. parents
    (total_q,) holds each node's parent within its own tree (a lower index, -1 for a root),
    sequence b's nodes being rows [cu_seqlens_q[b], cu_seqlens_q[b+1]); prefix_lens[b] tokens
    are cached before them. Node i is cached at position prefix_lens[b] + i
    (slot_mapping, -1 without a page), sits at position prefix_lens[b] + its depth
    (positions) and sees itself and its ancestors (tree_mask). max_nodes bounds every tree
    (at most 1024). Rows of no sequence get slot -1, which the append skips.

    A tree that breaks these rules is not seen on the host. A parent that is no lower node
    counts as -1; a node past max_nodes (rounded up to 64) gets slot -1, so it is not cached,
    and sees nothing. The number of both is added to invalid_count (one int32 on the device)
    where that is given."""
    fn = "tree_metadata"
    if not 1 <= max_nodes <= 1024:
        raise ValueError(f"{fn}: max_nodes must be 1 to 1024 (got {max_nodes})")
    idx = _device_index(fn, parents, cu_seqlens_q, prefix_lens, block_tables)
    bad = _count(fn, invalid_count, idx)
    keep, args = _tree_args(fn, parents, cu_seqlens_q, prefix_lens, block_tables, block_size)
    B, total, words, dev = args[-2], args[-1], (max_nodes + 63) // 64, parents.device
    slots = torch.empty(total, dtype=torch.int64, device=dev)
    lens = torch.empty(B, dtype=torch.int64, device=dev)
    positions = torch.empty(total, dtype=torch.int64, device=dev)
    mask = torch.empty(total, words, dtype=torch.int64, device=dev)
    st = _call_packed(_lib.load(), idx, _lib.CALL_TREE_METADATA, _lib.PACK_TREE_METADATA, args + (
        words, slots.data_ptr(), lens.data_ptr(), positions.data_ptr(), mask.data_ptr(), bad))
    if st:
        _lib.check(fn, st)
    return TreeMetadata(slots, lens, positions, mask)


def tree_accept(draft_tokens: torch.Tensor, target_tokens: torch.Tensor, parents: torch.Tensor,
                cu_seqlens_q: torch.Tensor, prefix_lens: torch.Tensor, block_tables: torch.Tensor,
                block_size: int, max_path: int) -> TreeAcceptance:
    """The path of each tree that the target model agrees with: from node 0, on to the
    lowest-numbered child whose draft token is the target token of the node before it
    (target_tokens[row], e.g. the argmax or the sample of the row's logits), at most max_path
    nodes. Returns the path, its target tokens (the step's new tokens), the number of cached
    tokens to keep, and the moves that bring the accepted rows there (move_kv_rows). The
    other arguments as for tree_metadata, whose rules hold for the trees (a node that it did
    not cache must not be accepted: its count tells)."""
    fn = "tree_accept"
    if not 1 <= max_path < 1 << 31:  # (32 bits in the C call)
        raise ValueError(f"{fn}: max_path must be at least 1 and below 2^31 (got {max_path})")
    idx = _device_index(fn, draft_tokens, target_tokens, parents, cu_seqlens_q, prefix_lens, block_tables)
    draft, target = _indices(fn, "draft_tokens", draft_tokens, 1), _indices(fn, "target_tokens", target_tokens, 1)
    keep, args = _tree_args(fn, parents, cu_seqlens_q, prefix_lens, block_tables, block_size)
    B, total = args[-2], args[-1]
    if draft.numel() != total or target.numel() != total or draft.dtype != target.dtype:
        raise ValueError(f"{fn}: draft_tokens and target_tokens must be {total} tokens each, of one dtype")
    dev = parents.device
    tokens = torch.empty(B, max_path, dtype=torch.int64, device=dev)
    src, dst = torch.empty_like(tokens), torch.empty_like(tokens)
    nodes = torch.empty(B, max_path, dtype=torch.int32, device=dev)
    count = torch.empty(B, dtype=torch.int32, device=dev)
    lens = torch.empty(B, dtype=torch.int64, device=dev)
    st = _call_packed(_lib.load(), idx, _lib.CALL_TREE_ACCEPT, _lib.PACK_TREE_ACCEPT, (
        draft.data_ptr(), target.data_ptr(), _INDEX[draft.dtype]) + args + (
        max_path, count.data_ptr(), nodes.data_ptr(), tokens.data_ptr(), lens.data_ptr(), src.data_ptr(),
        dst.data_ptr()))
    if st:
        _lib.check(fn, st)
    return TreeAcceptance(count, nodes, tokens, lens, src, dst)


# ------------------------------------------------------------------ copies inside the cache
def _cache_args(fn: str, cache: KVCache):
    kv = cache.kv
    if kv.dim() != 6 or kv.shape[0] != 2 or not kv.is_contiguous():
        raise ValueError(f"{fn}: the cache must be one contiguous (2, L, NB, BS, KVH, D) tensor")
    if kv.dtype not in _DTYPES:
        raise ValueError(f"{fn}: unsupported cache dtype {kv.dtype}")
    _, L, NB, BS, KVH, D = kv.shape
    ks = vs = stride = 0
    if cache.kv_cache_dtype in PER_TOKEN_HEAD:
        for t in (cache.k_scale, cache.v_scale):
            if t is None or t.dtype != torch.float32 or t.shape != (L, NB, BS, KVH) or not t.is_contiguous():
                raise ValueError(f"{fn}: {cache.kv_cache_dtype} needs contiguous float32 scales "
                                 f"({L}, {NB}, {BS}, {KVH})")
        ks, vs, stride = cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), NB * BS * KVH
    k = kv.data_ptr()
    v = k + kv.numel() // 2 * kv.element_size()
    return (k, v, _DTYPES[kv.dtype], L, NB * BS * KVH * D, NB, BS, KVH, D, ks, vs, stride)


def _pairs(fn: str, cache: KVCache, src: torch.Tensor, dst: torch.Tensor, dim: int):
    scales = cache.kv_cache_dtype in PER_TOKEN_HEAD
    idx = _device_index(fn, cache.kv, src, dst, cache.k_scale if scales else None,
                        cache.v_scale if scales else None)
    src, dst = _indices(fn, "the source", src, dim), _indices(fn, "the destination", dst, dim)
    if src.shape != dst.shape or src.dtype != dst.dtype:
        raise ValueError(f"{fn}: source and destination must have one shape and dtype")
    return idx, src, dst


def copy_kv_pages(cache: KVCache, src_pages: torch.Tensor, dst_pages: torch.Tensor,
                  invalid_count: Optional[torch.Tensor] = None) -> None:
    """Copies page src_pages[i] to page dst_pages[i] of every layer, K and V and the
    per-(token, head) scales, in one call: a forked sequence's own copy of a shared page,
    or the moves of a compaction. The copies are made in order, so one that reads a page
    written by an earlier one sees what was written; an entry below 0 is no copy, one past
    the cache is skipped, and counted in invalid_count (one int32 on the device, added to)
    where that is given."""
    fn = "copy_kv_pages"
    idx, src, dst = _pairs(fn, cache, src_pages, dst_pages, 1)
    st = _call_packed(_lib.load(), idx, _lib.CALL_COPY_KV_PAGES, _lib.PACK_COPY_PAGES, _cache_args(fn, cache) + (
        src.data_ptr(), dst.data_ptr(), _INDEX[src.dtype], src.numel(), _count(fn, invalid_count, idx)))
    if st:
        _lib.check(fn, st)


def move_kv_rows(cache: KVCache, src_slots: torch.Tensor, dst_slots: torch.Tensor,
                 invalid_count: Optional[torch.Tensor] = None) -> None:
    """Copies the cached row of slot src_slots[g, i] to slot dst_slots[g, i] in every layer,
    K and V and the per-(token, head) scales, in one call: the accepted rows of a tree,
    moved to the end of the cached prefix (tree_accept gives the slots). Moves are made in
    order within a group g (a sequence); the groups run side by side, so what one of them
    writes no other may read or write. An entry below 0 is no move, one past the cache is
    skipped, and counted in invalid_count as by copy_kv_pages."""
    fn = "move_kv_rows"
    idx, src, dst = _pairs(fn, cache, src_slots, dst_slots, 2)
    st = _call_packed(_lib.load(), idx, _lib.CALL_MOVE_KV_ROWS, _lib.PACK_MOVE_ROWS, _cache_args(fn, cache) + (
        src.data_ptr(), dst.data_ptr(), _INDEX[src.dtype], src.shape[0], src.shape[1],
        _count(fn, invalid_count, idx)))
    if st:
        _lib.check(fn, st)


def kv_head_shard(num_heads: int, num_kv_heads: int, rank: int, world_size: int):
    """(query-head range, kv-head range) owned by `rank` under tensor parallelism: KV heads
    split evenly (model_runner.py:215) with their GQA query heads (qwen3.py:27-33)."""
    if num_kv_heads % world_size or num_heads % world_size or num_heads % num_kv_heads:
        raise ValueError(f"cannot split {num_heads} query / {num_kv_heads} kv heads over {world_size} ranks")
    kvh = num_kv_heads // world_size
    h = num_heads // world_size
    return range(rank * h, (rank + 1) * h), range(rank * kvh, (rank + 1) * kvh)
