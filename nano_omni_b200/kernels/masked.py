"""bf16 attention over packed documents, bound to ``nob200_masked_bf16_attention_d128``.

No counterpart in the reference, whose attention of this head width is dense and takes one sequence.  Document, causal
and prefix masks, capped scores, a bias by distance and shared key heads; see the C header for the definition.
"""

from __future__ import annotations

import ctypes
import dataclasses
import math
from typing import Literal, NamedTuple

from pydantic import Field

from nano_omni_b200 import _lib
from nano_omni_b200.core import Arguments, Config, DType, Kernel, MmaType, TensorDesc, Workload, require_tensor

DEFAULT_SCALE = 128**-0.5


class MaskedBf16AttentionWorkload(Workload):
    num_rows: int = Field(gt=0)
    num_key_rows: int = Field(gt=0)
    documents: int = Field(gt=0)
    heads: int = Field(gt=0)
    kv_heads: int = Field(gt=0)
    total_heads: int = Field(gt=0)
    causal: bool = False
    use_prefix: bool = False
    use_slopes: bool = False
    cap: float = Field(default=0.0, ge=0, allow_inf_nan=False)
    scale: float = Field(default=DEFAULT_SCALE, gt=0, allow_inf_nan=False)


class MaskedBf16AttentionConfig(Config):
    unit_rows: Literal[128, 256] = 256  # query rows of a CTA
    kv_splits: int = Field(default=1, ge=1, le=64)  # > 1: the keys of a unit over so many CTAs; needs `workspace`


@dataclasses.dataclass(frozen=True, slots=True)
class MaskedBf16AttentionArguments(Arguments):
    query: TensorDesc
    key: TensorDesc
    value: TensorDesc
    bounds: TensorDesc
    key_bounds: TensorDesc
    prefix: TensorDesc | None
    slopes: TensorDesc | None
    output: TensorDesc
    head_offset: int
    causal: bool
    scale: float = DEFAULT_SCALE
    cap: float = 0.0
    workspace: TensorDesc | None = None

    def dynamic_parameters(self) -> tuple[tuple[str, int], ...]:
        return (("num_rows", self.query.shape[0]), ("num_key_rows", self.key.shape[0]), ("head_offset", self.head_offset))

    def index_values(self) -> dict[str, list]:
        """Plain contents of the index tensors, for launches outside a program: documents of one length."""
        documents = self.bounds.shape[0] - 1
        spread = lambda rows: [rows * d // documents for d in range(documents + 1)]  # noqa: E731
        values = {"bounds": spread(self.query.shape[0]), "key_bounds": spread(self.key.shape[0])}
        return values | ({"prefix": [0] * documents} if self.prefix is not None else {})


class MaskedUnits(NamedTuple):
    """How a launch becomes units: query rows of a unit, CTAs over which its keys are divided."""

    unit_rows: int
    kv_splits: int


def plan_masked_units(
    num_rows: int, num_key_rows: int, documents: int, heads: int, causal: bool, capped: bool = False, sm_count: int = 148
) -> MaskedUnits:
    """Units of a launch whose documents are taken to be of one length (the device alone knows their bounds).

    Times are counted in key tiles of a 256-row unit (1.9 us); 128 rows alone on an SM take 0.72 of one per key tile, a CTA 2
    beside its tiles, capped scores 1.28 times as long; units of 128 rows that share SMs, as they do where there are more
    than SMs, 0.88 (capped 0.7) and 0.3 (592 documents of 4 rows 23 us, 38 one to an SM; 148 of 100 rows x 4 heads 44, 57; five
    capped documents, 2100 x 28 63 and 75; nine of 9461 x 14 134, 119 in 256-row units); the join of shares 2.5 and 0.025 per
    256-row share.  Units of one length (or within a quarter of it: a chunk behind a long causal context) run in whole rounds
    of the SMs, others fill the last round to about a half.  One unit of 256 rows stays unless the estimate falls by 2 %: 1024
    rows x 14 heads 18.9 us in 128-row units, 21.9 in 256; 1560 causal rows against 30000 keys x 14 heads 331 us in three
    shares, 441 in six, 420 whole; 8192 rows x 14 heads 475 us whole, 505 in two shares."""
    rows, keys = -(-num_rows // documents), -(-num_key_rows // documents)
    seen = keys - min(rows, keys) / 2 if causal else keys
    tiles = max(1.0, seen / 128)
    alike = documents == 1 and (not causal or 4 * rows <= keys)
    best, plan = None, MaskedUnits(256, 1)
    for unit_rows in (256, 128):
        units = -(-rows // unit_rows) * documents * heads
        for splits in range(1, 65):
            if splits > 1 and tiles / splits < 2:
                break
            pieces = units * splits
            rounds = -(-pieces // sm_count) if alike or pieces <= sm_count else pieces / sm_count + 0.5
            if unit_rows == 128 and pieces > sm_count:
                step, beside = 0.7 if capped else 0.88, 0.3
            else:  # a document's 256 rows, or fewer alone; of ragged documents on few SMs some have more
                step, beside = (1.0 if unit_rows == 256 and (rows > 128 or pieces <= sm_count) else 0.72) * (1.28 if capped else 1.0), 2
            cost = rounds * (tiles / splits * step + beside)
            if splits > 1:
                cost += 2.5 + 0.025 * pieces * unit_rows / 256
            if best is None:
                best = 0.98 * cost
            elif cost < best:
                best, plan = cost, MaskedUnits(unit_rows, splits)
    return plan


def share_workspace_bytes(num_rows: int, heads: int, kv_splits: int) -> int:
    """Scratch of divided keys: normalised fp32 rows and their log-sum-exp."""
    return 0 if kv_splits <= 1 else kv_splits * heads * num_rows * 516


def check_masks(arguments, documents: int, heads: int) -> None:
    """Checks shared with the attention over a cache."""
    require_tensor(arguments.bounds, DType.I32, (documents + 1,), "bounds")
    if arguments.prefix is not None:
        require_tensor(arguments.prefix, DType.I32, (documents,), "prefix")
    if arguments.slopes is not None:
        require_tensor(arguments.slopes, DType.F32, (heads,), "slopes")
    scale, cap = arguments.scale, arguments.cap
    if scale > 0 and 0 < cap < math.inf:
        assert 1e-35 <= scale / cap <= 1e35, f"scale / cap must lie between 1e-35 and 1e35, not {scale} / {cap}"


class MaskedBf16AttentionKernel(
    Kernel[MaskedBf16AttentionArguments, MaskedBf16AttentionWorkload, MaskedBf16AttentionConfig]
):
    name = "masked_bf16_attention_d128"
    symbol = "nob200_masked_bf16_attention_d128"

    @classmethod
    def make_arguments(cls, workload: MaskedBf16AttentionWorkload) -> MaskedBf16AttentionArguments:
        w = workload
        keys = TensorDesc.empty(DType.BF16, (w.num_key_rows, w.kv_heads, 128))
        bounds = TensorDesc.empty(DType.I32, (w.documents + 1,))
        return MaskedBf16AttentionArguments(
            TensorDesc.empty(DType.BF16, (w.num_rows, w.heads, 128)), keys, keys, bounds, bounds,
            TensorDesc.empty(DType.I32, (w.documents,)) if w.use_prefix else None,
            TensorDesc.empty(DType.F32, (w.heads,)) if w.use_slopes else None,
            TensorDesc.empty(DType.BF16, (w.num_rows, w.total_heads, 128)), 0, w.causal, w.scale, w.cap,
        )  # fmt: skip

    @classmethod
    def make_config(cls, workload: MaskedBf16AttentionWorkload) -> MaskedBf16AttentionConfig:
        return MaskedBf16AttentionConfig()

    @classmethod
    def make_workload(cls, arguments: MaskedBf16AttentionArguments) -> MaskedBf16AttentionWorkload:
        a = arguments
        for tensor in (a.query, a.key, a.output):
            assert len(tensor.shape) == 3, "attention tensors have rank 3"
        num_rows, heads, _ = a.query.shape
        num_key_rows, kv_heads, _ = a.key.shape
        total_heads = a.output.shape[1]
        require_tensor(a.query, DType.BF16, (num_rows, heads, 128), "query")
        require_tensor(a.key, DType.BF16, (num_key_rows, kv_heads, 128), "key")
        require_tensor(a.value, DType.BF16, (num_key_rows, kv_heads, 128), "value")
        require_tensor(a.output, DType.BF16, (num_rows, total_heads, 128), "output")
        assert kv_heads > 0 and heads % kv_heads == 0, f"{heads} heads cannot share {kv_heads} key heads evenly"
        assert 0 <= a.head_offset <= total_heads - heads, "head slice ends past the output's heads"
        documents = a.bounds.shape[0] - 1
        check_masks(a, documents, heads)
        require_tensor(a.key_bounds, DType.I32, (documents + 1,), "key_bounds")
        assert a.slopes is None or a.cap > 0 or not a.scale < 1e-12, f"slopes need a scale of 1e-12 or more, not {a.scale}"
        return MaskedBf16AttentionWorkload(
            num_rows=num_rows, num_key_rows=num_key_rows, documents=documents, heads=heads, kv_heads=kv_heads,
            total_heads=total_heads, causal=a.causal, use_prefix=a.prefix is not None, use_slopes=a.slopes is not None,
            cap=a.cap, scale=a.scale,
        )  # fmt: skip

    @classmethod
    def tops(cls, arguments: MaskedBf16AttentionArguments) -> dict[MmaType, int]:
        """Of documents of one length; half of the pairs under a causal mask."""
        w = cls.make_workload(arguments)
        return {MmaType.BF16BF16F32: 4 * w.heads * 128 * w.num_rows * w.num_key_rows // w.documents // (2 if w.causal else 1)}

    def _launch(self, function, stream: int) -> int:
        a, w, c = self.arguments, self.workload, self.config
        need = share_workspace_bytes(w.num_rows, w.heads, c.kv_splits)
        assert need == 0 or (a.workspace is not None and a.workspace.num_bytes >= need), "kv_splits > 1 needs workspace"
        return function(
            ctypes.c_int(w.num_rows), ctypes.c_int(w.num_key_rows), ctypes.c_int(w.documents), ctypes.c_int(a.head_offset),
            _lib.ptr(a.query), _lib.ptr(a.key), _lib.ptr(a.value), _lib.ptr(a.bounds), _lib.ptr(a.key_bounds),
            _lib.ptr(a.prefix), _lib.ptr(a.slopes), _lib.ptr(a.output), ctypes.c_int(w.heads), ctypes.c_int(w.kv_heads),
            ctypes.c_int(w.total_heads), ctypes.c_int(int(a.causal)), ctypes.c_float(a.scale), ctypes.c_float(a.cap),
            ctypes.c_int(c.unit_rows), ctypes.c_int(c.kv_splits), _lib.ptr(a.workspace), ctypes.c_size_t(need),
            ctypes.c_void_p(stream),
        )  # fmt: skip
