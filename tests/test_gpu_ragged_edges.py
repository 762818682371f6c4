"""Edges of the ragged operators: bounds and lengths that cannot be right, caps and scales of any size, weights far below
the largest."""

import math

import pytest
import torch

from tests.test_gpu_kv_cache import HALF, Cache, append_op, ints, random_rows, run_op

pytestmark = pytest.mark.gpu

MOST, LEAST = 2**31 - 1, -(2**31)
BAD = 64  # bit 6 of the status word


def cached(cache, q, bounds, columns, splits=1, status=0, total_heads=None, causal=True, cap=0.0, scale=128**-0.5):
    """The cache attention at a chosen division of the work; rows that it does not write stay NaN."""
    from nano_omni_b200 import _lib
    from nano_omni_b200.core import DType
    from nano_omni_b200.kernels.cache import CacheAttentionArguments, CacheAttentionConfig, CacheAttentionKernel
    from nano_omni_b200.kernels.masked import share_workspace_bytes
    from tests.gpu_util import desc

    c, out, b = cache.desc(), torch.full_like(q, float("nan")), ints(bounds)
    need = share_workspace_bytes(len(q), q.shape[1], splits)
    workspace = desc(torch.full((need,), 255, dtype=torch.uint8, device="cuda"), DType.U8) if need else None
    arguments = CacheAttentionArguments(
        desc(q), c.key, c.value, c.key_scales, c.value_scales, c.table, c.lengths, desc(b), None, None, desc(out), 0, causal, scale, cap,
        workspace,
    )  # fmt: skip
    CacheAttentionKernel(arguments, CacheAttentionConfig(columns=columns, kv_splits=splits)).submit()
    got = _lib.read_status()
    assert got == status, f"{got:#x}"
    return out


def allowed_of(want, size, keys, most, extra=0.0):
    """Of the cached attention: the result rounded to bf16, probabilities to f16 (2^-11 = HALF / 8, and HALF / 5 for what fp32
    leaves out), those below 2^-21 of the row's largest by 2^-32 of it; ``extra``: of the scores, absolute."""
    return HALF * (0.4 * size + want.abs()) + 2 * extra * size + keys * 2.0**-32 * most + 1e-30


# ------------------------------------------------------------------ append
@pytest.mark.parametrize(
    "bounds,good",
    [([0, 3, 10, 10], [0]), ([0, 3, MOST, MOST], [0]), ([-2, 3, 6, 8], [1, 2]), ([LEAST, 3, 6, 8], [1, 2]), ([0, 5, 3, 8], [0, 2]),
     ([0, 9, 9, 8], [])],
    ids=str,
)  # fmt: skip
def test_append_skips_sequences_whose_bounds_are_not_right(bounds, good):
    """Rows that the tensor does not have, or an end before its beginning: the sequence is left as it is, the others are appended."""
    from tests.attention64 import append

    cache = Cache([90, 75, 140], 2, seed=1)
    k, v = random_rows(2, 8, 2), random_rows(3, 8, 2)
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in good:
        for which, x in enumerate((k, v)):
            fresh = x[bounds[s] : bounds[s + 1]].float()
            append(want[0][which], want[1][which], fresh, cache.table[s], cache.plain[s] - len(fresh))
    run_op(append_op(cache, k, v, ints(bounds)), status=BAD)
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])


@pytest.mark.parametrize("length", [LEAST, LEAST + 1, -1, 2, 193, MOST])
def test_append_skips_lengths_that_are_not_right(length):
    """Of any size: fewer tokens than the new ones, or more than the table has room for."""
    from tests.attention64 import append

    cache = Cache([90, 75, 140], 2, seed=4)
    k, v = random_rows(5, 8, 2), random_rows(6, 8, 2)
    bounds = [0, 3, 6, 8]
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in (0, 2):
        for which, x in enumerate((k, v)):
            fresh = x[bounds[s] : bounds[s + 1]].float()
            append(want[0][which], want[1][which], fresh, cache.table[s], cache.plain[s] - len(fresh))
    cache.lengths[1] = length
    run_op(append_op(cache, k, v, ints(bounds)), status=BAD)
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])


@pytest.mark.parametrize("bounds", [(128, 300), (128, 100)])
def test_append_notes_bounds_behind_the_last_rows(bounds):
    """More sequences than a CTA looks up at once; those behind the first 128 have no rows, and no CTA to look for any."""
    from tests.attention64 import append

    cache = Cache([70] * 300, 1, seed=28)
    k, v = random_rows(29, 128, 1), random_rows(30, 128, 1)
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in range(128):
        for which, x in enumerate((k, v)):
            append(want[0][which], want[1][which], x[s : s + 1].float(), cache.table[s], 69)
    run_op(append_op(cache, k, v, ints([*range(129), *[128] * 170, *bounds])), status=BAD)
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])


@pytest.mark.parametrize("spread", [0.1, 30.0])
def test_append_behind_a_negative_scale(spread):
    """A block whose scale is negative, smaller or larger in magnitude than the new tokens need: its values stay, on a grid of
    the larger magnitude."""
    cache = Cache([50], 2, seed=38)
    k, v = random_rows(39, 7, 2, spread), random_rows(40, 7, 2, spread)
    block = cache.table[0, 0].long()
    want = []
    for which, x in enumerate((k, v)):
        cache.scales[which][block, 0] *= -1
        cache.codes[which][block, 0, 5, 7] = -128
        old = cache.scales[which][block].clone()
        scale = torch.maximum(old.abs(), x.float().abs().amax((0, 2)) * (1 / 127))
        codes = cache.codes[which][block].clone()
        held = torch.round(codes[:, :43].float() * (old / scale)[:, None, None]).clamp(-128, 127)
        codes[:, :43] = torch.where((scale == old)[:, None, None], codes[:, :43].float(), held).to(torch.int8)
        codes[:, 43:50] = torch.round(x.float().transpose(0, 1) / scale[:, None, None]).clamp(-127, 127).to(torch.int8)
        want.append((scale, codes))
    run_op(append_op(cache, k, v, ints([0, 7])))
    for which in range(2):
        assert torch.equal(cache.scales[which][block], want[which][0])
        assert torch.equal(cache.codes[which][block], want[which][1])


# ------------------------------------------------------------------ bounds of the attentions
@pytest.mark.parametrize("columns,splits", [(8, 1), (8, 3), (16, 1), (128, 1), (128, 2)])
@pytest.mark.parametrize("bounds", [[0, 30, 50], [-7, 20, 40], [0, 30, MOST], [LEAST, 25, 40], [0, 40, 41]], ids=str)
def test_cached_rows_keep_their_positions_under_bounds_outside_the_rows(columns, splits, bounds):
    """Rows that are there stand where the bounds put them, and the status word says that some are not there."""
    from tests.attention64 import attend

    cache = Cache([300, 170], 2, seed=7)
    q = random_rows(8, 40, 4)
    out = cached(cache, q, bounds, columns, splits, status=BAD)
    for s in range(2):
        k, v = cache.rows(0, s), cache.rows(1, s)
        for row in range(max(bounds[s], 0), min(bounds[s + 1], 40)):
            seen = min(len(k), max(0, len(k) - (bounds[s + 1] - row) + 1))
            want, size = attend(q[row : row + 1], k[:seen], v[:seen])
            off = (out[row : row + 1].double() - want).abs()
            assert (off <= allowed_of(want, size, seen, v.abs().amax())).all(), (s, row)


@pytest.mark.parametrize("columns,splits", [(8, 1), (16, 2), (128, 1), (128, 2)])
def test_cached_bounds_that_descend_show(columns, splits):
    """A sequence that ends before it begins has no rows; the others' are right where no two claim a row."""
    from tests.attention64 import attend

    cache = Cache([300, 170, 90], 2, seed=9)
    q, bounds = random_rows(10, 40, 4), [0, 20, 12, 40]
    out = cached(cache, q, bounds, columns, splits, status=BAD)
    for s, rows in ((0, slice(0, 12)), (2, slice(20, 40))):
        k, v = cache.rows(0, s), cache.rows(1, s)
        want, size = attend(q[bounds[s] : bounds[s + 1]], k, v, causal=True)
        here = slice(rows.start - bounds[s], rows.stop - bounds[s])
        off = (out[rows].double() - want[here]).abs()
        assert (off <= allowed_of(want, size, len(k), v.abs().amax())[here]).all(), s


@pytest.mark.parametrize("columns,first", [(8, 128), (128, 640)])
@pytest.mark.parametrize("last", [9999, 100])
def test_cached_bounds_behind_the_last_rows_show(columns, first, last):
    """More sequences than a CTA looks up at once; those behind the first have no rows, and no CTA to look for any."""
    from tests.attention64 import attend

    cache = Cache([70] * (2 * first + 20), 1, seed=31)
    q = random_rows(32, first, 1)
    out = cached(cache, q, [*range(first + 1), *[first] * (first + 19), last], columns, status=BAD)
    for s in (0, 1, first - 1):
        k, v = cache.rows(0, s), cache.rows(1, s)
        want, size = attend(q[s : s + 1], k, v)
        assert ((out[s : s + 1].double() - want).abs() <= allowed_of(want, size, 70, v.abs().amax())).all()


@pytest.mark.parametrize("unit_rows,splits", [(256, 1), (128, 1), (128, 2)])
@pytest.mark.parametrize("which", ["rows", "keys"])
def test_masked_bounds_that_descend_show(unit_rows, splits, which):
    from nano_omni_b200 import _lib
    from nano_omni_b200.core import DType
    from nano_omni_b200.kernels.masked import (
        MaskedBf16AttentionArguments,
        MaskedBf16AttentionConfig,
        MaskedBf16AttentionKernel,
        share_workspace_bytes,
    )
    from tests.attention64 import attend
    from tests.gpu_util import desc
    from tests.test_gpu_masked_attention import tolerance

    q, k, v = (random_rows(seed, 300, 2) for seed in (11, 12, 13))
    bounds = [0, 120, 90, 300] if which == "rows" else [0, 120, 200, 300]
    key_bounds = [0, 120, 90, 300] if which == "keys" else bounds
    out = torch.full_like(q, float("nan"))
    need = share_workspace_bytes(300, 2, splits)
    workspace = desc(torch.empty(need, dtype=torch.uint8, device="cuda"), DType.U8) if need else None
    b, kb = ints(bounds), ints(key_bounds)
    arguments = MaskedBf16AttentionArguments(desc(q), desc(k), desc(v), desc(b), desc(kb), None, None, desc(out), 0, False, workspace=workspace)
    MaskedBf16AttentionKernel(arguments, MaskedBf16AttentionConfig(unit_rows=unit_rows, kv_splits=splits)).submit()
    got = _lib.read_status()
    assert got == BAD, f"{got:#x}"
    want, size = attend(q[:120], k[:120], v[:120])
    assert ((out[:90].double() - want[:90]).abs() <= tolerance(want, size)[:90]).all()
    if which == "keys":
        assert (out[120:200] == 0).all()  # no keys
    want, size = attend(q[200:300], k[90:300], v[90:300])
    assert ((out[200:300].double() - want).abs() <= tolerance(want, size)).all()


@pytest.mark.parametrize("heads,last", [(1, 100), (4, 100), (4, 9999)])
def test_masked_bounds_behind_the_last_rows(heads, last):
    """More documents than a CTA looks up at once; those behind the first have no rows, and no CTA to look for any."""
    from nano_omni_b200 import _lib
    from tests.gpu_util import desc
    from tests.test_gpu_masked_attention import op_of

    q, k, v = (random_rows(seed, 384, heads) for seed in (33, 34, 35))
    out = torch.zeros_like(q)
    op = op_of(q, k, v, [*range(385), *[384] * 600, last]).to(desc(out))
    scratch = torch.empty(op.prepare()[1] + 256, dtype=torch.uint8, device="cuda")
    op.run(scratch[(-scratch.data_ptr()) % 256 :])
    got = _lib.read_status()
    assert got == (BAD if last < 384 else 0), f"{got:#x}"
    assert torch.equal(out, v)  # every document is a row that sees itself


# ------------------------------------------------------------------ caps
@pytest.mark.parametrize("columns", [8, 16, 128])
@pytest.mark.parametrize("cap", [1e3, 1e5, 1e6, 1e9, 1e30])
def test_cached_scores_far_below_the_cap(columns, cap):
    """Scores of up to some 10 under caps that are next to none: the tanh's polynomial is off by 4e-6 of a score."""
    from tests.attention64 import attend

    cache = Cache([900], 1, seed=14)
    q = random_rows(15, 9, 3)
    out = cached(cache, q, [0, 9], columns, cap=cap)
    k, v = cache.rows(0, 0), cache.rows(1, 0)
    want, size = attend(q, k, v, causal=True, cap=cap)
    most = (torch.einsum("nhd,md->nhm", q.double(), k[:, 0]) * 128**-0.5).abs().amax().item()
    assert ((out.double() - want).abs() <= allowed_of(want, size, 900, v.abs().amax(), extra=4e-6 * most)).all()


@pytest.mark.parametrize("columns", [8, 16, 128])
def test_small_scores_beside_capped_ones(columns):
    """Rows of one call whose scores differ by orders of magnitude: a large cap is as exact for the small ones."""
    from tests.attention64 import attend

    cache = Cache([700], 1, seed=16)
    q = random_rows(17, 8, 1)
    q[::2] *= 2.0**20
    out = cached(cache, q, [0, 8], columns, cap=1e6)[1::2]
    k, v = cache.rows(0, 0), cache.rows(1, 0)
    want, size = (x[1::2] for x in attend(q, k, v, causal=True, cap=1e6))
    assert ((out.double() - want).abs() <= allowed_of(want, size, 700, v.abs().amax(), extra=6e-5)).all()


@pytest.mark.parametrize("cap", [1e-9, 1e-12, 1e-20, 1e-30])
@pytest.mark.parametrize("zero", [True, False])
@pytest.mark.parametrize("form", ["masked", 8, 16, 128])
def test_caps_next_to_nothing(form, zero, cap):
    """All scores are within the cap of zero, so a row is the plain mean of what it sees."""
    from tests.attention64 import attend
    from tests.test_gpu_masked_attention import attend as masked_attend
    from tests.test_gpu_masked_attention import tolerance

    q = random_rows(18, 200, 2)
    if zero:
        q.zero_()
    if form == "masked":
        k, v = random_rows(19, 200, 2), random_rows(20, 200, 2)
        out = masked_attend(q, k, v, [0, 200], causal=True, cap=cap)
        want, size = attend(q, k, v, causal=True, cap=cap)
        allowed = tolerance(want, size)
    else:
        cache = Cache([300], 2, seed=21)
        out = cached(cache, q, [0, 200], form, cap=cap)
        k, v = cache.rows(0, 0), cache.rows(1, 0)
        want, size = attend(q, k, v, causal=True, cap=cap)
        allowed = allowed_of(want, size, 300, v.abs().amax())
    assert ((out.double() - want).abs() <= allowed).all()


def test_capped_scores_of_large_products():
    """Products of 2^50 under a scale that makes ordinary scores of them: the scale over the cap has no square in fp32's range."""
    from tests.attention64 import attend
    from tests.test_gpu_masked_attention import attend as masked_attend
    from tests.test_gpu_masked_attention import tolerance

    q, k, v = random_rows(22, 130, 1), random_rows(23, 130, 1), random_rows(24, 130, 1)
    scale = 128**-0.5 * 2.0**-50
    q, k = q * 2.0**25, k * 2.0**25
    out = masked_attend(q, k, v, [0, 130], cap=15.0, scale=scale)
    want, size = attend(q, k, v, cap=15.0, scale=scale)
    assert ((out.double() - want).abs() <= tolerance(want, size, extra=6e-5)).all()


# ------------------------------------------------------------------ scales of any sign
@pytest.mark.parametrize("columns,rows", [(8, 8), (16, 9), (128, 9), (128, 40), (128, 100)])
@pytest.mark.parametrize("others", [0.01, 0.0, -0.01, 1e-34])
def test_value_scales_of_any_sign(columns, rows, others):
    """Blocks whose values are negated, zero or next to it, beside ordinary ones and alone."""
    from tests.attention64 import attend

    cache = Cache([500], 1, seed=25)
    blocks = cache.table[0].long()
    cache.scales[1][blocks[::2]] = others
    cache.scales[1][blocks[1]] *= -1
    cache.scales[1][blocks[3]] = 0.0
    for alone in (False, True):
        if alone:
            cache.scales[1].fill_(others)
        q = random_rows(26, rows, 1)
        out = cached(cache, q, [0, rows], columns)
        k, v = cache.rows(0, 0), cache.rows(1, 0)
        want, size = attend(q, k, v, causal=True)
        assert ((out.double() - want).abs() <= allowed_of(want, size, 500, v.abs().amax())).all(), alone


@pytest.mark.parametrize("columns,rows", [(8, 8), (16, 9), (128, 9), (128, 40), (128, 100)])
@pytest.mark.parametrize("cap", [0.0, 2.0])
def test_key_scales_of_any_sign(columns, rows, cap):
    """Keys that are negated, with scores large enough that the largest and the lowest are not to be taken for one another."""
    from tests.attention64 import attend

    cache = Cache([500], 1, seed=36)
    blocks = cache.table[0].long()
    cache.scales[0][blocks[1:6]] *= -1
    q = random_rows(37, rows, 1, 6.0)
    out = cached(cache, q, [0, rows], columns, cap=cap)
    k, v = cache.rows(0, 0), cache.rows(1, 0)
    want, size = attend(q, k, v, causal=True, cap=cap)
    assert ((out.double() - want).abs() <= allowed_of(want, size, 500, v.abs().amax(), extra=1e-4)).all()


# ------------------------------------------------------------------ small weights
@pytest.mark.parametrize("columns,rows,splits", [(8, 1, 1), (8, 1, 8), (16, 9, 2), (128, 9, 1), (128, 40, 4), (128, 100, 1)])
def test_many_keys_of_little_weight_count(columns, rows, splits):
    """One key 18 above 131071 others, whose weights, 2^-26 each, make 0.2 % together: they are all of the result where the
    large one's value is zero."""
    from tests.attention64 import attend

    n = 131072
    cache = Cache([n], 1, seed=27)
    for which in range(2):
        cache.codes[which].zero_()
        cache.scales[which].fill_(1 / 128)
    first = cache.table[0, 0].long()
    cache.codes[0][first, 0, 0] = 64  # key 0: halves
    cache.codes[1].fill_(100)
    cache.codes[1][first, 0, 0] = 0
    q = torch.full((rows, 1, 128), 18 * 2 * 128**-0.5, dtype=torch.bfloat16, device="cuda")
    out = cached(cache, q, [0, rows], columns, splits)
    k, v = cache.rows(0, 0), cache.rows(1, 0)
    want, size = attend(q[-1:], k, v)
    assert want.amin() > 0.0005
    assert ((out[-1:].double() - want).abs() <= allowed_of(want, size, n, v.abs().amax())).all()


@pytest.mark.parametrize("columns,rows", [(8, 8), (16, 9), (128, 20), (128, 40), (128, 100)])
@pytest.mark.parametrize("size", [5e6, 1.8e7, 5e7, 1.1e8])
def test_large_scores_that_grow_slowly(columns, rows, size):
    """Scores of `size` in log2 units, where a step of fp32 is 0.5 to 8 units, that grow from block to block by up to 60 such
    steps: no probability leaves f16, so that equal values come back whatever the weights are."""
    cache = Cache([640], 1, seed=41)
    blocks = cache.table[0].long()
    for which in range(2):
        cache.scales[which].fill_(0.01)
    cache.codes[1].fill_(100)
    q = torch.zeros(rows, 1, 128, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0], q[:, :, 1:5] = 1.0, 2.0**-17  # 127 + code * 2^-17 is exact in fp32
    for step in (*range(1, 13), 15, 20, 30, 60):
        cache.codes[0].zero_()
        for b in range(10):
            cache.codes[0][blocks[b], 0, :, 0] = 127
            for channel in range(1, 5):
                cache.codes[0][blocks[b], 0, :, channel] = min(127, max(0, step * b - 127 * (channel - 1)))
        out = cached(cache, q, [0, rows], columns, causal=False, scale=size / (127 * 0.01 * 1.4426950408889634))
        off = (out.double() - 1.0).abs().amax().item()  # probabilities are rounded by 2^-11 beside their sum, the result by 2^-8
        assert off <= 2.0**-8 + 2.0**-11, (step, off)


# ------------------------------------------------------------------ arguments for timing
def test_addressing_arguments_leaves_given_tensors():
    """What a caller has put in place, index tensors among it, is not written."""
    import dataclasses

    from nano_omni_b200 import tune
    from nano_omni_b200.kernels.cache import CacheReadKernel, CacheReadWorkload
    from tests.gpu_util import desc

    empty = CacheReadKernel.make_arguments(CacheReadWorkload(capacity=90, sequences=2, max_blocks=3, num_blocks=9, kv_heads=1))
    table, lengths = ints([[5, 6, 7], [1, 2, 3]]), ints([40, 50])
    arguments = tune.address(dataclasses.replace(empty, table=desc(table), lengths=desc(lengths)))
    assert table.tolist() == [[5, 6, 7], [1, 2, 3]] and lengths.tolist() == [40, 50]
    assert arguments.bounds.as_torch().tolist() == [0, 0, 0] and arguments.table.as_torch() is table
    filled = tune.address(empty)
    assert filled.lengths.as_torch().tolist() == [192, 192] and filled.table.as_torch().tolist() == [[0, 1, 2], [3, 4, 5]]
    assert not math.isnan(filled.key_scales.as_torch().sum().item())
