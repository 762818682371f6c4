"""A cache of keys and values in 8 bits: append, read back, and the attention of a few queries over it.

No counterpart in the reference.  Blocks of 64 tokens, int8 codes ``[num_blocks, kv_heads, 64, 128]`` and one fp32 scale per
block and head ``[num_blocks, kv_heads]`` for each of K and V; ``table`` int32 ``[sequences, max_blocks]`` names the block
that holds tokens ``64 b .. 64 b + 63`` of a sequence, ``lengths`` int32 ``[sequences]`` how many tokens it has.
"""

from __future__ import annotations

import ctypes
import dataclasses
from typing import Literal, NamedTuple

from pydantic import Field

from nano_omni_b200 import _lib
from nano_omni_b200.core import Arguments, Config, DType, Kernel, MmaType, TensorDesc, Workload, require_tensor
from nano_omni_b200.kernels.masked import DEFAULT_SCALE, check_masks, share_workspace_bytes

BLOCK = 64  # tokens of a block


def _cache_shape(arguments) -> tuple[int, int, int, int]:
    """(blocks, key heads, sequences, blocks of a sequence) of the cache tensors, checked against one another."""
    a = arguments
    assert len(a.key_codes.shape) == 4 and len(a.table.shape) == 2, "codes have rank 4, the table rank 2"
    num_blocks, kv_heads = a.key_codes.shape[:2]
    sequences, max_blocks = a.table.shape
    for what, codes, scales in (("key", a.key_codes, a.key_scales), ("value", a.value_codes, a.value_scales)):
        require_tensor(codes, DType.I8, (num_blocks, kv_heads, BLOCK, 128), f"{what} codes")
        require_tensor(scales, DType.F32, (num_blocks, kv_heads), f"{what} scales")
    require_tensor(a.table, DType.I32, (sequences, max_blocks), "table")
    require_tensor(a.lengths, DType.I32, (sequences,), "lengths")
    return num_blocks, kv_heads, sequences, max_blocks


def _empty_cache(w) -> tuple[TensorDesc, ...]:
    """key codes, value codes, key scales, value scales, table, lengths"""
    codes = TensorDesc.empty(DType.I8, (w.num_blocks, w.kv_heads, BLOCK, 128))
    scales = TensorDesc.empty(DType.F32, (w.num_blocks, w.kv_heads))
    table = TensorDesc.empty(DType.I32, (w.sequences, w.max_blocks))
    return codes, codes, scales, scales, table, TensorDesc.empty(DType.I32, (w.sequences,))


def _full_cache(arguments) -> dict[str, list]:
    """A table of distinct blocks, as far as there are any, and sequences that fill theirs."""
    num_blocks, _, sequences, max_blocks = _cache_shape(arguments)
    table = [[(s * max_blocks + b) % num_blocks for b in range(max_blocks)] for s in range(sequences)]
    return {"table": table, "lengths": [max_blocks * BLOCK] * sequences}


class CacheWorkload(Workload):
    sequences: int = Field(gt=0)
    max_blocks: int = Field(gt=0)
    num_blocks: int = Field(gt=0)
    kv_heads: int = Field(gt=0)


class CacheConfig(Config):
    pass


# ------------------------------------------------------------------ append
class CacheAppendWorkload(CacheWorkload):
    num_rows: int = Field(gt=0)


@dataclasses.dataclass(frozen=True, slots=True)
class CacheAppendArguments(Arguments):
    key: TensorDesc
    value: TensorDesc
    bounds: TensorDesc
    table: TensorDesc
    lengths: TensorDesc
    key_codes: TensorDesc
    key_scales: TensorDesc
    value_codes: TensorDesc
    value_scales: TensorDesc

    def dynamic_parameters(self) -> tuple[tuple[str, int], ...]:
        return (("num_rows", self.key.shape[0]),)

    def index_values(self) -> dict[str, list]:
        rows, sequences = self.key.shape[0], self.bounds.shape[0] - 1
        return _full_cache(self) | {"bounds": [rows * s // sequences for s in range(sequences + 1)]}


class CacheAppendKernel(Kernel[CacheAppendArguments, CacheAppendWorkload, CacheConfig]):
    """``key`` and ``value`` bf16 ``[rows, kv_heads, 128]`` become the last tokens of their sequences; ``lengths`` counts them."""

    name = "int8_cache_append_d128"
    symbol = "nob200_int8_cache_append_d128"

    @classmethod
    def make_arguments(cls, workload: CacheAppendWorkload) -> CacheAppendArguments:
        key_codes, value_codes, key_scales, value_scales, table, lengths = _empty_cache(workload)
        rows = TensorDesc.empty(DType.BF16, (workload.num_rows, workload.kv_heads, 128))
        bounds = TensorDesc.empty(DType.I32, (workload.sequences + 1,))
        return CacheAppendArguments(rows, rows, bounds, table, lengths, key_codes, key_scales, value_codes, value_scales)

    @classmethod
    def make_config(cls, workload: CacheAppendWorkload) -> CacheConfig:
        return CacheConfig()

    @classmethod
    def make_workload(cls, arguments: CacheAppendArguments) -> CacheAppendWorkload:
        num_blocks, kv_heads, sequences, max_blocks = _cache_shape(arguments)
        rows = arguments.key.shape[0]
        require_tensor(arguments.key, DType.BF16, (rows, kv_heads, 128), "key")
        require_tensor(arguments.value, DType.BF16, (rows, kv_heads, 128), "value")
        require_tensor(arguments.bounds, DType.I32, (sequences + 1,), "bounds")
        return CacheAppendWorkload(
            num_rows=rows, sequences=sequences, max_blocks=max_blocks, num_blocks=num_blocks, kv_heads=kv_heads
        )

    def _launch(self, function, stream: int) -> int:
        a, w = self.arguments, self.workload
        return function(
            ctypes.c_int(w.num_rows), ctypes.c_int(w.sequences), ctypes.c_int(w.max_blocks), ctypes.c_int(w.num_blocks),
            _lib.ptr(a.key), _lib.ptr(a.value), _lib.ptr(a.bounds), _lib.ptr(a.table), _lib.ptr(a.lengths),
            _lib.ptr(a.key_codes), _lib.ptr(a.key_scales), _lib.ptr(a.value_codes), _lib.ptr(a.value_scales),
            ctypes.c_int(w.kv_heads), ctypes.c_void_p(stream),
        )  # fmt: skip


# ------------------------------------------------------------------ read
class CacheReadWorkload(CacheWorkload):
    capacity: int = Field(gt=0)


@dataclasses.dataclass(frozen=True, slots=True)
class CacheReadArguments(Arguments):
    key_codes: TensorDesc
    value_codes: TensorDesc
    key_scales: TensorDesc
    value_scales: TensorDesc
    table: TensorDesc
    lengths: TensorDesc
    key: TensorDesc
    value: TensorDesc
    bounds: TensorDesc

    def dynamic_parameters(self) -> tuple[tuple[str, int], ...]:
        return (("capacity", self.key.shape[0]),)

    def index_values(self) -> dict[str, list]:
        return _full_cache(self) | {"bounds": [0] * self.bounds.shape[0]}


class CacheReadKernel(Kernel[CacheReadArguments, CacheReadWorkload, CacheConfig]):
    """The sequences' tokens as bf16 rows ``[capacity, kv_heads, 128]``, one sequence behind the other, and their bounds."""

    name = "int8_cache_read_d128"
    symbol = "nob200_int8_cache_read_d128"

    @classmethod
    def make_arguments(cls, workload: CacheReadWorkload) -> CacheReadArguments:
        rows = TensorDesc.empty(DType.BF16, (workload.capacity, workload.kv_heads, 128))
        return CacheReadArguments(
            *_empty_cache(workload), rows, rows, TensorDesc.empty(DType.I32, (workload.sequences + 1,))
        )

    @classmethod
    def make_config(cls, workload: CacheReadWorkload) -> CacheConfig:
        return CacheConfig()

    @classmethod
    def make_workload(cls, arguments: CacheReadArguments) -> CacheReadWorkload:
        num_blocks, kv_heads, sequences, max_blocks = _cache_shape(arguments)
        capacity = arguments.key.shape[0]
        require_tensor(arguments.key, DType.BF16, (capacity, kv_heads, 128), "key")
        require_tensor(arguments.value, DType.BF16, (capacity, kv_heads, 128), "value")
        require_tensor(arguments.bounds, DType.I32, (sequences + 1,), "bounds")
        return CacheReadWorkload(
            capacity=capacity, sequences=sequences, max_blocks=max_blocks, num_blocks=num_blocks, kv_heads=kv_heads
        )

    def _launch(self, function, stream: int) -> int:
        a, w = self.arguments, self.workload
        return function(
            ctypes.c_int(w.capacity), ctypes.c_int(w.sequences), ctypes.c_int(w.max_blocks), ctypes.c_int(w.num_blocks),
            _lib.ptr(a.key_codes), _lib.ptr(a.value_codes), _lib.ptr(a.key_scales), _lib.ptr(a.value_scales),
            _lib.ptr(a.table), _lib.ptr(a.lengths), _lib.ptr(a.key), _lib.ptr(a.value), _lib.ptr(a.bounds),
            ctypes.c_int(w.kv_heads), ctypes.c_void_p(stream),
        )  # fmt: skip


# ------------------------------------------------------------------ attention
class CacheAttentionWorkload(CacheWorkload):
    num_rows: int = Field(gt=0)
    heads: int = Field(gt=0)
    total_heads: int = Field(gt=0)
    causal: bool = True
    use_prefix: bool = False
    use_slopes: bool = False
    cap: float = Field(default=0.0, ge=0, allow_inf_nan=False)
    scale: float = Field(default=DEFAULT_SCALE, gt=0, allow_inf_nan=False)


MAX_CLUSTER = 8  # up to so many shares need no workspace: their CTAs are a cluster and join them themselves


class CacheUnits(NamedTuple):
    """How a launch becomes CTAs: rows of a sequence and key head (new tokens x query heads) of one, shares of its keys, and
    whether the shares of a unit are a cluster."""

    columns: int
    kv_splits: int
    clusters: bool


def _tile_shares(units: int, sequences: int, tokens: int, sm_count: int) -> int:
    """In key tiles of 128: a CTA takes 8 tiles' time beside its own, the join 3.  One sequence's CTAs run in whole rounds; of
    several, the longest is taken to hold twice the average and to begin first, and the last CTAs to end unevenly (drafted
    tokens of 16 sequences up to 8192 keys long x 8 key heads: 119 us undivided, 60 in two shares, 67 in three)."""
    tiles = max(1, tokens // 128)

    def cost(n: int) -> float:
        several = max(units * (tiles + 8 * n) / sm_count, 2 * tiles / n + 8) + tiles / (2 * n)
        whole = -(-units * n // sm_count) * (tiles / n + 8)
        return (whole if sequences == 1 else several) + 3 * (n > 1)

    return min(range(1, max(1, min(64, tiles // 4)) + 1), key=cost)


def _column_shares(units: int, sequences: int, tokens: int, room: int) -> tuple[int, bool]:
    """As many as have room at once, with 128 keys each at least.  Several sequences are taken to be of unequal lengths, the
    longest of which begin first: up to eight shares 2.25 rounds' worth, more 1.25, with 512 keys each at least (ragged
    contexts x 8 key heads: 64 of up to 16384 keys 160 us in 3 shares, 166 in 2, 169 in 4, 276 undivided; 24 of 8192 43 in 6,
    45 in 4, 46 in 8, 58 in 2; 8 of 8192 23.5 in 12, 25.0 in 8, 25.7 in 16).  Clusters where eight shares do: 1021 keys x 14
    heads 8.9 us, 11.3 with the second launch; of several sequences where 128 keys each are the bound (16 of 1024 keys 12.8
    us, 13.6), as a cluster's CTAs wait for room and for one another (8 of 8192 30 us in clusters of eight, 25)."""
    shares = max(1, min(64, tokens // 128, room // units))
    if sequences > 1:
        rounds = (9 * room + 2 * units) // (4 * units)
        rounds = min(tokens // 512, rounds if rounds <= 8 else max(8, 5 * room // (4 * units)))
        shares = min(64, max(shares, rounds))
    in_clusters = 1 < shares < 12 and units * min(shares, MAX_CLUSTER) <= room and (sequences == 1 or shares == tokens // 128)
    return (min(shares, MAX_CLUSTER) if in_clusters else shares), in_clusters


def plan_cache_units(num_rows: int, sequences: int, cached_tokens: int, heads: int, kv_heads: int, sm_count: int = 148) -> CacheUnits:
    """Units of a launch whose sequences are taken to be of one length (the device alone knows).

    Up to sixteen rows of a sequence and key head are columns of the small kernel, eight where they do, of which an SM has room
    for four CTAs; of sixteen it has room for three and two are planned for (16 rows against 8192 x 4 x 16 sequences 34 us as
    columns, 37 in tiles, measured so).  More are eights
    of columns or take the kernel of 128-row tiles, whichever is estimated to be faster: a CTA of eight columns 7.6 us and
    0.018 a key, of tiles 11.5 and 0.0081, a second launch 3 (64 sequences x 14 key heads, 30 rows: 100 keys 53 us in eights, 75
    in tiles, 276 72 and 84, 1005 154 and 121; 24 rows of one sequence x 8 key heads: 1524 keys 11 and 16, 30000 39 and 34)."""
    each = -(-num_rows * (heads // kv_heads) // sequences)
    tokens = -(-cached_tokens // sequences)

    def in_columns(columns: int) -> CacheUnits:
        units = max(1, -(-each // columns) * sequences * kv_heads)
        return CacheUnits(columns, *_column_shares(units, sequences, tokens, 32 // columns * sm_count))

    if each <= 16:
        return in_columns(8 if each <= 8 else 16)
    groups = sequences * kv_heads
    tiles = -(-each // 128) * groups
    shares = _tile_shares(tiles, sequences, tokens, sm_count)
    if each <= 64:
        few = in_columns(8)
        rounds = max(1.0, -(-each // 8) * groups * few.kv_splits / (4 * sm_count))
        of_columns = rounds * (7.6 + 0.018 * tokens / few.kv_splits) + (0 if few.kv_splits == 1 or few.clusters else 3)
        of_tiles = max(1.0, tiles * shares / sm_count) * (11.5 + 0.0081 * tokens / shares) + (0 if shares == 1 else 3)
        if of_columns < of_tiles:
            return few
    return CacheUnits(128, shares, False)


class CacheAttentionConfig(Config):
    columns: Literal[8, 16, 128] = 16  # rows of a CTA
    kv_splits: int = Field(default=1, ge=1, le=64)  # > 1: a sequence's keys over so many CTAs, clusters of up to 8 without `workspace`


@dataclasses.dataclass(frozen=True, slots=True)
class CacheAttentionArguments(Arguments):
    query: TensorDesc
    key_codes: TensorDesc
    value_codes: TensorDesc
    key_scales: TensorDesc
    value_scales: TensorDesc
    table: TensorDesc
    lengths: TensorDesc
    bounds: TensorDesc
    prefix: TensorDesc | None
    slopes: TensorDesc | None
    output: TensorDesc
    head_offset: int
    causal: bool
    scale: float = DEFAULT_SCALE
    cap: float = 0.0
    workspace: TensorDesc | None = None

    def dynamic_parameters(self) -> tuple[tuple[str, int], ...]:
        return (("num_rows", self.query.shape[0]), ("head_offset", self.head_offset))

    def index_values(self) -> dict[str, list]:
        rows, sequences = self.query.shape[0], self.bounds.shape[0] - 1
        values = _full_cache(self) | {"bounds": [rows * s // sequences for s in range(sequences + 1)]}
        return values | ({"prefix": [0] * sequences} if self.prefix is not None else {})


class CacheAttentionKernel(Kernel[CacheAttentionArguments, CacheAttentionWorkload, CacheAttentionConfig]):
    name = "int8_cache_attention_d128"
    symbol = "nob200_int8_cache_attention_d128"

    @classmethod
    def make_arguments(cls, workload: CacheAttentionWorkload) -> CacheAttentionArguments:
        w = workload
        return CacheAttentionArguments(
            TensorDesc.empty(DType.BF16, (w.num_rows, w.heads, 128)), *_empty_cache(w),
            TensorDesc.empty(DType.I32, (w.sequences + 1,)),
            TensorDesc.empty(DType.I32, (w.sequences,)) if w.use_prefix else None,
            TensorDesc.empty(DType.F32, (w.heads,)) if w.use_slopes else None,
            TensorDesc.empty(DType.BF16, (w.num_rows, w.total_heads, 128)), 0, w.causal, w.scale, w.cap,
        )  # fmt: skip

    @classmethod
    def make_config(cls, workload: CacheAttentionWorkload) -> CacheAttentionConfig:
        return CacheAttentionConfig()

    @classmethod
    def make_workload(cls, arguments: CacheAttentionArguments) -> CacheAttentionWorkload:
        a = arguments
        num_blocks, kv_heads, sequences, max_blocks = _cache_shape(a)
        assert len(a.query.shape) == 3 and len(a.output.shape) == 3, "attention tensors have rank 3"
        num_rows, heads, _ = a.query.shape
        total_heads = a.output.shape[1]
        require_tensor(a.query, DType.BF16, (num_rows, heads, 128), "query")
        require_tensor(a.output, DType.BF16, (num_rows, total_heads, 128), "output")
        assert kv_heads > 0 and heads % kv_heads == 0, f"{heads} heads cannot share {kv_heads} key heads evenly"
        assert 0 <= a.head_offset <= total_heads - heads, "head slice ends past the output's heads"
        check_masks(a, sequences, heads)
        return CacheAttentionWorkload(
            num_rows=num_rows, heads=heads, total_heads=total_heads, sequences=sequences, max_blocks=max_blocks,
            num_blocks=num_blocks, kv_heads=kv_heads, causal=a.causal, use_prefix=a.prefix is not None,
            use_slopes=a.slopes is not None, cap=a.cap, scale=a.scale,
        )  # fmt: skip

    @classmethod
    def tops(cls, arguments: CacheAttentionArguments) -> dict[MmaType, int]:
        """Of full tables."""
        w = cls.make_workload(arguments)
        return {MmaType.F16F16F32: 4 * w.heads * 128 * w.num_rows * w.max_blocks * BLOCK}

    def _launch(self, function, stream: int) -> int:
        a, w, c = self.arguments, self.workload, self.config
        need = share_workspace_bytes(w.num_rows, w.heads, c.kv_splits) if a.workspace is not None else 0
        assert need or c.kv_splits <= MAX_CLUSTER, f"more than {MAX_CLUSTER} kv_splits need workspace"
        assert need == 0 or a.workspace.num_bytes >= need, "workspace too small"
        return function(
            ctypes.c_int(w.num_rows), ctypes.c_int(w.sequences), ctypes.c_int(w.max_blocks), ctypes.c_int(w.num_blocks),
            ctypes.c_int(a.head_offset), _lib.ptr(a.query), _lib.ptr(a.key_codes), _lib.ptr(a.value_codes),
            _lib.ptr(a.key_scales), _lib.ptr(a.value_scales), _lib.ptr(a.table), _lib.ptr(a.lengths), _lib.ptr(a.bounds),
            _lib.ptr(a.prefix), _lib.ptr(a.slopes), _lib.ptr(a.output), ctypes.c_int(w.heads), ctypes.c_int(w.kv_heads),
            ctypes.c_int(w.total_heads), ctypes.c_int(int(a.causal)), ctypes.c_float(a.scale), ctypes.c_float(a.cap),
            ctypes.c_int(c.columns), ctypes.c_int(c.kv_splits), _lib.ptr(a.workspace), ctypes.c_size_t(need),
            ctypes.c_void_p(stream),
        )  # fmt: skip
