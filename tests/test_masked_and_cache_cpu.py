"""Planning and refusals of the masked attention and the 8-bit cache (no GPU)."""

import ctypes

import pytest

from nano_omni_b200 import kernels, ops
from nano_omni_b200.core import DType, TensorDesc


def at(dtype, *shape):
    at.next += 1 << 30
    return TensorDesc.from_pointer(at.next, dtype, shape)


at.next = 1 << 40


def cache(blocks=20, kv_heads=2, sequences=3, max_blocks=8):
    codes, scales = (blocks, kv_heads, 64, 128), (blocks, kv_heads)
    return ops.BlockCache(
        at(DType.I8, *codes), at(DType.I8, *codes), at(DType.F32, *scales), at(DType.F32, *scales),
        at(DType.I32, sequences, max_blocks), at(DType.I32, sequences),
    )  # fmt: skip


def masked(heads=4, kv_heads=2, rows=300, key_rows=300, documents=3, total_heads=6, **options):
    return ops.MaskedBf16Attention(
        at(DType.BF16, rows, heads * 128), at(DType.BF16, key_rows, kv_heads * 128), at(DType.BF16, key_rows, kv_heads * 128),
        at(DType.I32, documents + 1), total_heads=total_heads, **options,
    )  # fmt: skip


def test_masked_attention_plans_one_launch_of_its_kernel():
    op = masked(causal=True, prefix=at(DType.I32, 3), slopes=at(DType.F32, 4), cap=20.0, head_offset=2)
    op.to(at(DType.BF16, 300, 6, 128))
    call = op.prepare()[0][0]
    assert call.name == "masked_bf16_attention_d128"
    w = call.workload
    assert (w.heads, w.kv_heads, w.documents, w.causal, w.use_prefix, w.use_slopes, w.cap) == (4, 2, 3, True, True, True, 20.0)
    assert call.arguments.key_bounds is call.arguments.bounds


def test_rotation_comes_in_front():
    rotation = ops.Rotation(at(DType.BF16, 128), at(DType.BF16, 128), at(DType.F32, 300, 48), at(DType.F32, 300, 48))
    op = masked(rotation=rotation).to(at(DType.BF16, 300, 6, 128))
    assert [c.name for c in op.prepare()[0]] == ["h3_head_norm_rope", "h3_head_norm_rope", "masked_bf16_attention_d128"]


@pytest.mark.parametrize(
    "options",
    [
        {"kv_heads": 3},  # does not divide the heads
        {"head_offset": 3},
        {"key_rows": 200},  # fewer keys than queries need bounds of their own
        {"causal": True, "prefix": (DType.I32, 2)},
        {"causal": True, "prefix": (DType.F32, 3)},
        {"slopes": (DType.F32, 2)},
        {"slopes": (DType.BF16, 4)},
        {"key_bounds": (DType.I32, 5)},
    ],
    ids=str,
)
def test_masked_attention_refuses(options):
    options = {n: at(x[0], *x[1:]) if isinstance(x, tuple) else x for n, x in options.items()}
    with pytest.raises(AssertionError):
        masked(**options).to(at(DType.BF16, 300, 6, 128)).prepare()


def test_masked_attention_refuses_slopes_with_next_to_no_scale():
    slopes, out = at(DType.F32, 4), at(DType.BF16, 300, 6, 128)
    with pytest.raises(AssertionError):
        masked(slopes=slopes, scale=1e-13).to(out).prepare()
    masked(slopes=slopes, scale=1e-13, cap=1.0).to(out).prepare()
    masked(scale=1e-13).to(out).prepare()


@pytest.mark.parametrize("options", [{"cap": -1.0}, {"cap": float("inf")}, {"scale": 0.0}, {"scale": float("nan")}], ids=str)
def test_masked_attention_refuses_numbers(options):
    with pytest.raises(ValueError):
        masked(**options).to(at(DType.BF16, 300, 6, 128)).prepare()
    op = ops.CacheAttention(at(DType.BF16, 3, 512), at(DType.I32, 4), cache(), total_heads=4, **options)
    with pytest.raises(ValueError):
        op.to(at(DType.BF16, 3, 4, 128)).prepare()


def test_cache_operators_plan_their_kernels():
    c = cache()
    append = ops.CacheAppend(at(DType.BF16, 9, 256), at(DType.BF16, 9, 256), at(DType.I32, 4), c)
    append.to(c.key, c.key_scales, c.value, c.value_scales)
    assert [k.name for k in append.prepare()[0]] == ["int8_cache_append_d128"]
    read = ops.CacheRead(c, 900).to(at(DType.BF16, 900, 256), at(DType.BF16, 900, 256), at(DType.I32, 4))
    assert [k.name for k in read.prepare()[0]] == ["int8_cache_read_d128"]
    attend = ops.CacheAttention(at(DType.BF16, 3, 512), at(DType.I32, 4), c, total_heads=4).to(at(DType.BF16, 3, 4, 128))
    assert [k.name for k in attend.prepare()[0]] == ["int8_cache_attention_d128"]
    assert c.capacity == 3 * 8 * 64


def test_cache_operators_refuse():
    c = cache()
    rows = at(DType.BF16, 9, 256)
    with pytest.raises(AssertionError):  # heads of the rows and of the cache
        ops.CacheAppend(at(DType.BF16, 9, 512), at(DType.BF16, 9, 512), at(DType.I32, 4), c)
    with pytest.raises(AssertionError):  # bounds of another number of sequences
        op = ops.CacheAppend(rows, rows, at(DType.I32, 5), c).to(c.key, c.key_scales, c.value, c.value_scales)
        op.prepare()
    with pytest.raises(AssertionError):  # outputs in another order
        ops.CacheAppend(rows, rows, at(DType.I32, 4), c).to(c.key, c.value, c.key_scales, c.value_scales)
    with pytest.raises(AssertionError):
        ops.CacheRead(c, 900).to(at(DType.BF16, 800, 256), at(DType.BF16, 900, 256), at(DType.I32, 4))
    with pytest.raises(AssertionError):  # heads that cannot share two key heads
        ops.CacheAttention(at(DType.BF16, 3, 384), at(DType.I32, 4), c, total_heads=3)
    with pytest.raises(AssertionError):  # a prefix for another number of sequences
        op = ops.CacheAttention(at(DType.BF16, 3, 512), at(DType.I32, 4), c, total_heads=4, prefix=at(DType.I32, 2))
        op.to(at(DType.BF16, 3, 4, 128)).prepare()
    for field, wrong in (("key_scales", (DType.F32, 20, 3)), ("table", (DType.F32, 3, 8)), ("lengths", (DType.I32, 2)),
                         ("value", (DType.I8, 20, 2, 32, 128))):  # fmt: skip
        fields = {n: getattr(c, n) for n in ("key", "value", "key_scales", "value_scales", "table", "lengths")}
        broken = ops.BlockCache(**fields | {field: at(wrong[0], *wrong[1:])})
        with pytest.raises(AssertionError):
            op = ops.CacheAttention(at(DType.BF16, 3, 512), at(DType.I32, 4), broken, total_heads=4)
            op.to(at(DType.BF16, 3, 4, 128)).prepare()


def test_workloads_survive_the_round_trip():
    from nano_omni_b200.kernels.cache import CacheAppendWorkload, CacheAttentionWorkload, CacheReadWorkload
    from nano_omni_b200.kernels.masked import MaskedBf16AttentionWorkload

    common = {"sequences": 3, "max_blocks": 5, "num_blocks": 11, "kv_heads": 2}
    for workload, name in (
        (MaskedBf16AttentionWorkload(num_rows=9, num_key_rows=70, documents=4, heads=6, kv_heads=2, total_heads=7, causal=True,
                                     use_prefix=True, use_slopes=True, cap=3.0), "masked_bf16_attention_d128"),
        (CacheAppendWorkload(num_rows=9, **common), "int8_cache_append_d128"),
        (CacheReadWorkload(capacity=90, **common), "int8_cache_read_d128"),
        (CacheAttentionWorkload(num_rows=9, heads=4, total_heads=4, use_slopes=True, **common), "int8_cache_attention_d128"),
    ):  # fmt: skip
        cls = kernels.classes()[name]
        arguments = cls.make_arguments(workload)
        assert cls.make_workload(arguments) == workload
        for field, values in arguments.index_values().items():
            shape = getattr(arguments, field).shape
            assert len(values) == shape[0] and (len(shape) == 1 or len(values[0]) == shape[1])


@pytest.fixture(scope="module")
def lib():
    from nano_omni_b200 import _lib, build

    build.build()
    lib = _lib.library()
    lib.nob200_last_error.restype = ctypes.c_char_p
    return lib


def test_c_entries_refuse_before_any_launch(lib):
    p, null, z = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0), ctypes.c_size_t(0)
    f = ctypes.c_float

    def refused(function, arguments, text):
        function.restype = ctypes.c_int
        assert function(*arguments) == -1 and text in lib.nob200_last_error(), lib.nob200_last_error()

    def attention(rows=9, heads=4, kv_heads=2, offset=0, query=p, output=p, scale=0.1, cap=0.0, unit=256, splits=1, workspace=null,
                  size=z, slopes=null):  # fmt: skip
        return (rows, 70, 3, offset, query, p, p, p, p, null, slopes, output, heads, kv_heads, 4, 1, f(scale), f(cap), unit, splits,
                workspace, size, null)  # fmt: skip

    fn = lib.nob200_masked_bf16_attention_d128
    refused(fn, attention(rows=0), b"positive")
    refused(fn, attention(kv_heads=3), b"cannot share 3 key heads")
    refused(fn, attention(offset=1), b"head_offset")
    refused(fn, attention(query=null), b"NULL")
    refused(fn, attention(output=ctypes.c_void_p(8)), b"16-byte aligned")
    refused(fn, attention(scale=float("nan")), b"scale")
    refused(fn, attention(cap=-1.0), b"cap")
    refused(fn, attention(unit=192), b"unit_rows")
    refused(fn, attention(scale=1e-13, slopes=p), b"slopes")
    refused(fn, attention(splits=65), b"kv_splits")
    refused(fn, attention(splits=2), b"workspace required")
    refused(fn, attention(rows=0x7FFFFFFF, heads=4, splits=64, workspace=p, size=ctypes.c_size_t(1 << 62)), b"grid limit")

    fn = lib.nob200_int8_cache_append_d128
    refused(fn, (0, 3, 5, 11, p, p, p, p, p, p, p, p, p, 2, null), b"positive")
    refused(fn, (9, 3, 5, 11, p, p, p, p, null, p, p, p, p, 2, null), b"NULL")
    refused(fn, (9, 3, 1 << 26, 11, p, p, p, p, p, p, p, p, p, 2, null), b"exceed the limit")
    refused(fn, (9, 3, 5, 11, ctypes.c_void_p(8), p, p, p, p, p, p, p, p, 2, null), b"aligned")
    fn = lib.nob200_int8_cache_read_d128
    refused(fn, (0, 3, 5, 11, p, p, p, p, p, p, p, p, p, 2, null), b"positive")
    refused(fn, (90, 3, 5, 11, p, p, p, p, p, p, p, p, null, 2, null), b"NULL")

    def cached(rows=3, blocks=11, kv_heads=2, splits=1, lengths=p, cap=0.0, columns=16):
        return (rows, 3, 5, blocks, 0, p, p, p, p, p, p, lengths, p, null, null, p, 4, kv_heads, 4, 1, f(0.1), f(cap), columns, splits, null, z,
                null)  # fmt: skip

    fn = lib.nob200_int8_cache_attention_d128
    refused(fn, cached(rows=0), b"positive")
    refused(fn, cached(kv_heads=3), b"cannot share")
    refused(fn, cached(lengths=null), b"NULL")
    refused(fn, cached(cap=float("inf")), b"cap")
    refused(fn, cached(blocks=1 << 28), b"exceed the limit")
    refused(fn, cached(splits=9), b"workspace required")
    refused(fn, cached(columns=12), b"columns")


def test_workspace_sizes_are_the_planned_ones(lib):
    from nano_omni_b200.kernels.masked import share_workspace_bytes

    for name in ("masked_bf16", "int8_cache"):
        fn = getattr(lib, f"nob200_{name}_attention_d128_workspace_bytes")
        fn.restype = ctypes.c_size_t
        for rows, heads, splits in ((1, 1, 1), (1, 14, 21), (32768, 28, 8), (100, 8, 9), (4096, 56, 64)):
            assert fn(rows, heads, splits) == share_workspace_bytes(rows, heads, splits)


def test_the_kernels_are_in_the_registry():
    from nano_omni_b200 import kernels

    names = {"masked_bf16_attention_d128", "int8_cache_append_d128", "int8_cache_read_d128", "int8_cache_attention_d128"}
    assert names <= set(kernels.classes())


def test_a_chunk_behind_a_long_context_runs_in_whole_rounds():
    from nano_omni_b200.kernels.masked import plan_masked_units

    for causal in (False, True):  # 7 units x 14 heads x 3 shares: 294 of the 296 places of two rounds
        assert plan_masked_units(1560, 30000, 1, 14, causal) == (256, 3)


def test_calls_without_rows_documents_or_tokens_are_refused():
    with pytest.raises(AssertionError):
        masked(documents=0)
    with pytest.raises(AssertionError):
        masked(rows=0, key_rows=0)
    for rows, tokens in ((0, None), (3, 0)):
        with pytest.raises(AssertionError):
            ops.CacheAttention(at(DType.BF16, rows, 512), at(DType.I32, 4), cache(), total_heads=4, cached_tokens=tokens)


@pytest.mark.parametrize("scale,cap", [(0.1, 1e-37), (1e-12, 1e26), (1e20, 1e-17)])
def test_a_scale_over_the_cap_outside_fp32_is_refused(lib, scale, cap):
    with pytest.raises(AssertionError):
        masked(scale=scale, cap=cap).to(at(DType.BF16, 300, 6, 128)).prepare()
    op = ops.CacheAttention(at(DType.BF16, 3, 512), at(DType.I32, 4), cache(), total_heads=4, scale=scale, cap=cap)
    with pytest.raises(AssertionError):
        op.to(at(DType.BF16, 3, 4, 128)).prepare()
    p, null, z, f = ctypes.c_void_p(1 << 20), ctypes.c_void_p(0), ctypes.c_size_t(0), ctypes.c_float
    calls = {
        "masked_bf16": (9, 70, 3, 0, p, p, p, p, p, null, null, p, 4, 2, 4, 1, f(scale), f(cap), 256, 1, null, z, null),
        "int8_cache": (3, 3, 5, 11, 0, p, p, p, p, p, p, p, p, null, null, p, 4, 2, 4, 1, f(scale), f(cap), 16, 1, null, z, null),
    }
    for name, arguments in calls.items():
        fn = getattr(lib, f"nob200_{name}_attention_d128")
        fn.restype = ctypes.c_int
        assert fn(*arguments) == -1 and b"scale / cap" in lib.nob200_last_error()


def test_masked_units_follow_the_options():
    """An option that is set later is planned for as if it had been given at construction; chosen units stay."""
    from nano_omni_b200.kernels.masked import MaskedUnits

    shape = {"heads": 28, "kv_heads": 28, "rows": 2100, "key_rows": 2100, "documents": 5, "total_heads": 28}
    late, out = masked(**shape).to(at(DType.BF16, 2100, 28, 128)), at(DType.BF16, 2100, 28, 128)
    plain = late.prepare()[0][-1].config
    late.cap = 30.0
    early = masked(**shape, cap=30.0).to(out)
    assert late.prepare()[0][-1].config == early.prepare()[0][-1].config != plain
    late.units = MaskedUnits(256, 2)
    late.causal = True
    call = late.prepare()[0][-1]
    assert (call.config.unit_rows, call.config.kv_splits) == (256, 2) and call.arguments.workspace is not None


@pytest.mark.parametrize("sequences", [1, 2, 7, 64, 300])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (14, 14), (32, 8), (56, 8), (16, 1)])
def test_cache_plans_can_be_launched(sequences, heads, kv_heads):
    """Whatever the plan: shares within their limits, clusters of what a cluster holds, workspace where there is none."""
    from nano_omni_b200.kernels.cache import MAX_CLUSTER, plan_cache_units
    from nano_omni_b200.kernels.masked import share_workspace_bytes

    for rows in (1, 2, 3, 8, 9, 16, 17, 24, 64, 65, 128, 129, 600, 4096):
        for blocks in (1, 2, 4, 16, 100, 2048):
            c = cache(blocks=sequences * blocks, kv_heads=kv_heads, sequences=sequences, max_blocks=blocks)
            for tokens in (1, 65, c.capacity):
                columns, splits, clusters = plan = plan_cache_units(rows, sequences, min(tokens, c.capacity), heads, kv_heads)
                assert columns in (8, 16, 128) and 1 <= splits <= 64, plan
                assert not clusters or (2 <= splits <= MAX_CLUSTER and columns < 128), plan
                query, bounds = at(DType.BF16, rows, heads * 128), at(DType.I32, sequences + 1)
                op = ops.CacheAttention(query, bounds, c, total_heads=heads, cached_tokens=tokens).to(at(DType.BF16, rows, heads, 128))
                (call,), scratch = op.prepare()
                assert (call.config.columns, call.config.kv_splits) == (columns, splits)
                need = 0 if clusters else share_workspace_bytes(rows, heads, splits)
                assert scratch == need == (call.arguments.workspace.num_bytes if call.arguments.workspace else 0)


@pytest.mark.parametrize(
    "call,plan",
    [
        # eight and nine, sixteen and seventeen rows of a sequence and key head
        ((64, 64, 64 * 1021, 8, 1), (8, 7, True)),
        ((64, 64, 64 * 1021, 9, 1), (16, 4, False)),
        ((64, 64, 64 * 1021, 16, 1), (16, 4, False)),
        ((64, 64, 64 * 1021, 17, 1), (8, 3, False)),
        # 64 and 65: from there on tiles alone
        ((64, 1, 300, 8, 8), (8, 2, True)),
        ((65, 1, 300, 8, 8), (128, 1, False)),
        # few rows against few keys and many: eights, tiles
        ((24, 1, 1524, 8, 8), (8, 8, True)),
        ((24, 1, 30000, 8, 8), (128, 18, False)),
        # a token against keys of one share, of a cluster's, of more
        ((1, 1, 128, 4, 4), (8, 1, False)),
        ((1, 1, 256, 4, 4), (8, 2, True)),
        ((1, 1, 1021, 14, 14), (8, 7, True)),
        ((1, 1, 131072, 14, 14), (8, 42, False)),
    ],
)
def test_cache_plans_on_both_sides_of_their_limits(call, plan):
    from nano_omni_b200.kernels.cache import plan_cache_units

    assert plan_cache_units(*call) == plan
