"""Masked attention over packed documents against 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0**-8  # half a step of bf16, relative


def tolerance(o, size, extra=0.0):
    """Probabilities and the result are rounded to bf16 once each: HALF of sum p |v| and of the result.  What fp32 leaves out
    (scores of magnitude up to 30, 128 products each: 30 * 128 * 2^-24 = 2.3e-4, twice that in a probability; sums and
    exponentials 1e-6) is under a fifth of a step: 0.2 * HALF covers it.  ``extra``: of the scores, absolute."""
    return HALF * (1.2 * size + o.abs()) + 2 * extra * size + 1e-30


def rows(seed, n, heads, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, 128, generator=g) * spread).bfloat16().cuda()


def ends(lengths):
    found = [0]
    for n in lengths:
        found.append(found[-1] + n)
    return found


def op_of(q, k, v, bounds, key_bounds=None, total_heads=None, head_offset=0, **options):
    from nano_omni_b200 import ops
    from tests.gpu_util import desc

    ints = {n: torch.tensor(options[n], dtype=torch.int32, device="cuda") for n in ("prefix",) if options.get(n) is not None}
    b = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    kb = torch.tensor(key_bounds, dtype=torch.int32, device="cuda") if key_bounds is not None else None
    options = {n: x for n, x in options.items() if x is not None and n not in ("prefix", "slopes")}
    flat = [desc(x.view(x.shape[0], -1)) for x in (q, k, v)]
    slopes = options.pop("slope_tensor", None)
    op = ops.MaskedBf16Attention(
        *flat, desc(b), total_heads=total_heads or q.shape[1], head_offset=head_offset, key_bounds=desc(kb) if kb is not None else None,
        prefix=desc(ints["prefix"]) if ints else None, slopes=desc(slopes) if slopes is not None else None, **options,
    )  # fmt: skip
    op.kept = (b, kb, ints, slopes)
    return op


def attend(q, k, v, bounds, key_bounds=None, total_heads=None, head_offset=0, fill=float("nan"), check=True, **options):
    from nano_omni_b200 import _lib
    from tests.gpu_util import desc

    total = total_heads or q.shape[1]
    out = torch.full((q.shape[0], total, 128), fill, dtype=torch.bfloat16, device="cuda")
    op = op_of(q, k, v, bounds, key_bounds, total, head_offset, **options).to(desc(out))
    scratch = torch.empty(op.prepare()[1] + 256, dtype=torch.uint8, device="cuda")
    op.run(scratch[(-scratch.data_ptr()) % 256 :])
    status = _lib.read_status()
    assert status == 0, f"{status:#x}"
    return out


def compare(q, k, v, bounds, key_bounds=None, extra=0.0, **options):
    from tests.attention64 import attend_documents

    out = attend(q, k, v, bounds, key_bounds, **options).double()
    slopes = options.pop("slope_tensor", None)
    want, size = attend_documents(q, k, v, bounds, key_bounds or bounds, slopes=slopes, **options)
    inside = slice(bounds[0], bounds[-1])
    off = (out - want).abs()[inside]
    allowed = tolerance(want, size, extra)[inside]
    assert torch.isfinite(out[inside]).all()
    assert (off <= allowed).all(), f"{(off / allowed).max().item():.3f} times the tolerance"
    outside = torch.ones(len(q), dtype=torch.bool)
    outside[inside] = False
    assert out[outside.cuda()].isnan().all(), "rows outside the documents were written"


LENGTHS = [[1], [2], [127], [128], [129], [255], [256], [257], [300], [385], [513, 1, 0, 128, 77], [0, 0, 5], [64] * 40, [640, 900]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_documents(lengths, causal):
    n = sum(lengths) + 7  # some rows behind the last document
    q, k, v = rows(1, n, 2), rows(2, n, 2), rows(3, n, 2)
    compare(q, k, v, ends(lengths), causal=causal)


@pytest.mark.parametrize("heads,kv_heads", [(6, 2), (8, 1), (4, 4), (14, 7)])
@pytest.mark.parametrize("queries,keys", [([5, 130, 1], [400, 131, 0]), ([300], [77]), ([129, 64], [1000, 64])])
@pytest.mark.parametrize("causal", [False, True])
def test_other_keys_than_queries(heads, kv_heads, queries, keys, causal):
    """Chunks of queries against longer (and shorter: rows that see nothing) documents, heads that share key heads."""
    q, k, v = rows(4, sum(queries), heads), rows(5, sum(keys) + 3, kv_heads), rows(6, sum(keys) + 3, kv_heads)
    compare(q, k, v, ends(queries), ends(keys), causal=causal)


@pytest.mark.parametrize("prefix", [[1, 0, 0], [200, 129, 5000], [128, 128, 300]])
@pytest.mark.parametrize("causal", [True, False])
def test_prefix(prefix, causal):
    """Without a causal mask a prefix changes nothing."""
    lengths = [390, 200, 300]
    q, k, v = rows(7, 890, 2), rows(8, 890, 2), rows(9, 890, 2)
    compare(q, k, v, ends(lengths), causal=causal, prefix=prefix)


@pytest.mark.parametrize("spread,cap", [(1.0, 50.0), (6.0, 20.0), (6.0, 1.0), (40.0, 30.0), (1.0, 0.05)])
@pytest.mark.parametrize("biased", [False, True])
def test_capped_scores(spread, cap, biased):
    """Scores well inside the cap (the polynomial), past it and far past it (the exponential).  Errors of a capped score: the
    tanh's 3e-7 times the cap, and the score's own in the linear part."""
    q, k, v = rows(10, 517, 4, spread), rows(11, 517, 2), rows(12, 517, 2)
    slopes = torch.tensor([0.5, 0.01, 0.0, 0.1], device="cuda") if biased else None
    compare(q, k, v, [0, 400, 517], causal=True, cap=cap, slope_tensor=slopes, extra=3e-7 * cap + 1e-4 * spread)


@pytest.mark.parametrize("causal,prefix", [(True, None), (True, [300, 0]), (False, None)])
@pytest.mark.parametrize("queries,keys", [([700, 130], [700, 130]), ([60, 130], [900, 20])])
def test_distance_bias(causal, prefix, queries, keys):
    """Keys behind, at and (prefix, no causal mask) ahead of the query.  The bias in fp32: 900 * 0.5 * 3 * 2^-24 absolute."""
    q, k, v = rows(13, sum(queries), 3), rows(14, sum(keys), 3), rows(15, sum(keys), 3)
    slopes = torch.tensor([0.5, 0.004, -0.02], device="cuda")
    compare(q, k, v, ends(queries), ends(keys), causal=causal, prefix=prefix, slope_tensor=slopes, extra=1e-4)


@pytest.mark.parametrize("where", ["behind", "other_document", "later_key"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_masked_places_may_hold_anything(where, value):
    """What a row does not see does not reach it, whatever it is; a value that is not finite shows where it is seen."""
    from tests.attention64 import attend_documents

    bounds, n = [0, 200, 333], 340
    q, k, v = rows(16, n, 2), rows(17, n, 2), rows(18, n, 2)
    want, size = attend_documents(q, k, v, bounds, bounds, causal=True)
    if where == "behind":
        k[333:], v[333:], q[333:], clean = value, value, value, slice(0, 333)
    elif where == "other_document":
        k[200:333], v[200:333], q[200:333], clean = value, value, value, slice(0, 200)
    else:
        k[150], v[150], clean = value, value, slice(0, 150)
    out = attend(q, k, v, bounds, causal=True, fill=0.0).double()
    assert ((out - want).abs() <= tolerance(want, size))[clean].all()
    if where == "later_key" and not math.isfinite(value):
        assert out[150:200].isnan().any(-1).all()


def test_a_value_that_is_not_finite_shows_in_rows_that_see_it():
    q, k, v = rows(19, 256, 1), rows(20, 256, 1), rows(21, 256, 1)
    v[130, 0, 77] = float("inf")
    out = attend(q, k, v, [0, 256], causal=True)
    assert torch.isfinite(out[:130]).all() and not torch.isfinite(out[130:, 0, 77]).any()
    whole = attend(q, k, v, [0, 256])
    assert not torch.isfinite(whole[:, 0, 77]).any()


def test_head_slice_scale_and_rotation():
    """A slice of a wider output, another scale, norm and rotary embedding in front as in the dense operators."""
    from nano_omni_b200 import ops
    from tests.gpu_util import desc

    t, h = 300, 3
    q, k, v = rows(22, t, h), rows(23, t, h), rows(24, t, h)
    weight = [(1 + 0.1 * torch.randn(128)).bfloat16().cuda() for _ in range(2)]
    angle = torch.rand(t, 48, device="cuda") * 6
    planes = angle.cos().contiguous(), angle.sin().contiguous()
    rotation = ops.Rotation(*(desc(x) for x in (*weight, *planes)))
    out = attend(q, k, v, [0, t], total_heads=8, head_offset=4, rotation=rotation, scale=0.05)
    assert out[:, :4].isnan().all() and out[:, 7:].isnan().all()

    from nano_omni_b200.kernels.norm_rope import H3HeadNormRopeArguments, H3HeadNormRopeKernel
    from tests.attention64 import attend as attend64

    turned = [torch.empty_like(x) for x in (q, k)]
    for x, y, w in zip((q, k), turned, weight):
        H3HeadNormRopeKernel(H3HeadNormRopeArguments(desc(x), desc(w), desc(planes[0]), desc(planes[1]), desc(y))).submit()
    want, size = attend64(*turned, v, scale=0.05)
    assert ((out[:, 4:7].double() - want).abs() <= tolerance(want, size)).all()


@pytest.mark.parametrize("unit_rows", [128, 256])
@pytest.mark.parametrize("splits", [1, 2, 7])
@pytest.mark.parametrize("causal", [False, True])
def test_units_and_key_shares(unit_rows, splits, causal):
    """Every division of the work, more shares than a unit has key tiles among them, gives the definition's result."""
    from nano_omni_b200.core import DType
    from nano_omni_b200.kernels.masked import (
        MaskedBf16AttentionArguments,
        MaskedBf16AttentionConfig,
        MaskedBf16AttentionKernel,
        share_workspace_bytes,
    )
    from tests.attention64 import attend_documents
    from tests.gpu_util import desc, run

    bounds = [0, 3, 600, 600, 1111]
    q, k, v = rows(25, 1130, 4), rows(26, 1130, 2), rows(27, 1130, 2)
    slopes = torch.tensor([0.1, 0.02, 0.0, 0.4], device="cuda")
    b = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, float("nan"))
    need = share_workspace_bytes(1130, 4, splits)
    workspace = desc(torch.empty(need, dtype=torch.uint8, device="cuda"), DType.U8) if need else None
    arguments = MaskedBf16AttentionArguments(
        desc(q), desc(k), desc(v), desc(b), desc(b), None, desc(slopes), desc(out), 0, causal, 128**-0.5, 30.0, workspace
    )
    run(MaskedBf16AttentionKernel(arguments, MaskedBf16AttentionConfig(unit_rows=unit_rows, kv_splits=splits)))
    want, size = attend_documents(q, k, v, bounds, bounds, causal=causal, cap=30.0, slopes=slopes)
    off = (out.double() - want).abs()[:1111]
    assert (off <= tolerance(want, size, 1e-4)[:1111]).all()
    assert out[1111:].isnan().all()


def test_bounds_outside_the_rows_touch_nothing_else():
    """Bounds are clamped to the tensors: a last document that claims more rows than there are ends with them."""
    q, k, v = rows(28, 200, 1), rows(29, 200, 1), rows(30, 200, 1)
    got = attend(q, k, v, [0, 90, 1 << 30], causal=True)
    want = attend(q, k, v, [0, 90, 200], causal=True)
    assert torch.equal(got, want)
    got = attend(q, k, v, [-5, 90, 200], causal=True)
    assert torch.equal(got, want)


def test_runs_again_with_other_bounds_streams_and_graphs():
    """The bounds are read when the operator runs: changed in place they count, in a replayed graph too."""
    from tests.gpu_util import desc

    q, k, v = rows(31, 500, 2), rows(32, 500, 2), rows(33, 500, 2)
    out = torch.zeros(500, 2, 128, dtype=torch.bfloat16, device="cuda")
    op = op_of(q, k, v, [0, 200, 500], causal=True).to(desc(out))
    scratch = torch.empty(op.prepare()[1] + 256, dtype=torch.uint8, device="cuda")
    scratch = scratch[(-scratch.data_ptr()) % 256 :]
    first, second = (attend(q, k, v, b, causal=True) for b in ([0, 200, 500], [0, 333, 500]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    op.run(scratch, side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run(scratch)
    op.kept[0].copy_(torch.tensor([0, 333, 500], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, second)


@pytest.mark.parametrize("documents", [2, 31, 384, 385, 900])  # a CTA orders up to 384 documents by their keys, more it does not
@pytest.mark.parametrize("causal", [False, True])
def test_many_documents(documents, causal):
    g = torch.Generator().manual_seed(documents)
    queries = torch.randint(0, 4, (documents,), generator=g)
    queries[documents // 2], queries[-1] = 300, 140
    keys = queries + torch.randint(0, 30, (documents,), generator=g)
    keys[0], keys[1] = 500, 0
    q, k, v = rows(34, int(queries.sum()) + 1, 2), rows(35, int(keys.sum()), 1), rows(36, int(keys.sum()), 1)
    compare(q, k, v, ends(queries.tolist()), ends(keys.tolist()), causal=causal)


@pytest.mark.parametrize("causal", [False, True])
def test_rows_in_front_of_the_first_document(causal):
    """Neither Q's nor K's documents need begin at row 0; several key shares write and join only what lies inside."""
    q, k, v = rows(37, 340, 2), rows(38, 3000, 2), rows(39, 3000, 2)
    compare(q, k, v, [7, 200, 333], [500, 700, 2990], causal=causal)
    compare(q, k, v, [339, 340], [11, 2999], causal=causal)


def test_two_calls_at_once():
    """The same operator twice, on two streams with scratch of their own, beside each other."""
    from nano_omni_b200 import _lib
    from tests.gpu_util import desc

    q, k, v = rows(40, 600, 4), rows(41, 20000, 2), rows(42, 20000, 2)
    want = attend(q, k, v, [0, 100, 600], [0, 9000, 20000], causal=True)
    outs, ops_, streams, scratches = [], [], [torch.cuda.Stream() for _ in range(2)], []
    for _ in streams:
        outs.append(torch.zeros_like(q))
        ops_.append(op_of(q, k, v, [0, 100, 600], [0, 9000, 20000], causal=True).to(desc(outs[-1])))
        scratch = torch.empty(ops_[-1].prepare()[1] + 256, dtype=torch.uint8, device="cuda")
        scratches.append(scratch[(-scratch.data_ptr()) % 256 :])
    torch.cuda.synchronize()
    for _ in range(5):
        for op, stream, scratch in zip(ops_, streams, scratches):
            op.run(scratch, stream.cuda_stream)
    torch.cuda.synchronize()
    assert _lib.read_status() == 0
    assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("causal,prefix", [(False, None), (True, None), (True, [300, 0, 40, 10])])
@pytest.mark.parametrize("cap,biased", [(0.0, False), (30.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("spoiled", [False, True])
def test_units_that_share_an_sm(causal, prefix, cap, biased, spoiled):
    """More units of 128 rows than SMs, from no key tile to eight; what lies behind a document's keys may be anything."""
    from nano_omni_b200.core import DType
    from nano_omni_b200.kernels.masked import MaskedBf16AttentionArguments, MaskedBf16AttentionConfig, MaskedBf16AttentionKernel
    from tests.attention64 import attend_documents
    from tests.gpu_util import desc, run

    bounds, key_bounds = [0, 3, 600, 601, 1111], [0, 130, 1130, 1130, 1200]
    q, k, v = rows(43, 1130, 16), rows(44, 1250, 4), rows(45, 1250, 4)
    slopes = torch.linspace(0.0, 0.4, 16, device="cuda") if biased else None
    want, size = attend_documents(q, k, v, bounds, key_bounds, causal=causal, prefix=prefix, cap=cap, slopes=slopes)
    if spoiled:
        k[1200:], v[1200:], q[1111:] = float("nan"), float("inf"), float("nan")
    b, kb = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (bounds, key_bounds))
    p = torch.tensor(prefix, dtype=torch.int32, device="cuda") if prefix else None
    out = torch.full_like(q, float("nan"))
    arguments = MaskedBf16AttentionArguments(
        desc(q), desc(k), desc(v), desc(b), desc(kb), None if p is None else desc(p), None if slopes is None else desc(slopes),
        desc(out), 0, causal, 128**-0.5, cap, None,
    )  # fmt: skip
    run(MaskedBf16AttentionKernel(arguments, MaskedBf16AttentionConfig(unit_rows=128)))
    off = (out.double() - want).abs()[:1111]
    assert (off <= tolerance(want, size, 1e-4)[:1111]).all()
    assert out[1111:].isnan().all()
