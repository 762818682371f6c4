"""The 8-bit cache of keys and values: append, read back and attend, against 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = 2.0**-8  # half a step of bf16, relative


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def ends(lengths):
    found = [0]
    for n in lengths:
        found.append(found[-1] + n)
    return found


class Cache:
    """Random codes and scales in blocks that lie in any order."""

    def __init__(self, lengths, kv_heads, seed=0, room=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // 64) for n in lengths]
        self.blocks, self.kv_heads = sum(need) + 2, kv_heads
        self.max_blocks = max(1, max(need)) + room
        order = torch.randperm(self.blocks, generator=g).int()
        self.table = torch.full((len(lengths), self.max_blocks), -7, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at : at + n]
            at += n
        shape = (self.blocks, kv_heads, 64, 128)
        self.codes = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).cuda() for _ in range(2)]
        self.scales = [(0.005 + 0.02 * torch.rand(self.blocks, kv_heads, generator=g)).cuda() for _ in range(2)]
        self.table, self.lengths, self.plain = self.table.cuda(), ints(lengths), list(lengths)

    def desc(self):
        from nano_omni_b200 import ops
        from tests.gpu_util import desc

        (k, v), (ks, vs) = self.codes, self.scales
        return ops.BlockCache(desc(k), desc(v), desc(ks), desc(vs), desc(self.table), desc(self.lengths))

    def rows(self, which, s):
        from tests.attention64 import cached_rows

        return cached_rows(self.codes[which], self.scales[which], self.table[s], self.plain[s])


def run_op(op, status=0):
    from nano_omni_b200 import _lib

    scratch = torch.empty(op.prepare()[1] + 256, dtype=torch.uint8, device="cuda")
    op.run(scratch[(-scratch.data_ptr()) % 256 :])
    got = _lib.read_status()
    assert got == status, f"{got:#x}"


def random_rows(seed, n, heads, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, heads, 128, generator=g) * spread).bfloat16().cuda()


def append_op(cache, k, v, bounds):
    from nano_omni_b200 import ops
    from tests.gpu_util import desc

    c = cache.desc()
    op = ops.CacheAppend(desc(k.view(len(k), -1)), desc(v.view(len(v), -1)), desc(bounds), c)
    return op.to(c.key, c.key_scales, c.value, c.value_scales)


def attention_op(cache, q, bounds, **options):
    from nano_omni_b200 import ops
    from tests.gpu_util import desc

    options = {n: desc(x) if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    options.setdefault("total_heads", q.shape[1])
    return ops.CacheAttention(desc(q.view(len(q), -1)), desc(bounds), cache.desc(), **options)


@pytest.mark.parametrize(
    "before,new",
    [([0], [1]), ([63], [1]), ([64], [1]), ([1], [62]), ([0], [64]), ([10], [300]), ([0, 7, 130, 64], [5, 0, 200, 64]),
     ([3] * 40, [1] * 40), ([500, 0], [129, 1])],
    ids=str,
)  # fmt: skip
@pytest.mark.parametrize("spread", [0.02, 1.0, 30.0])  # scales that never grow, some that do, all that do
def test_append(before, new, spread):
    from tests.attention64 import append

    cache = Cache([b + n for b, n in zip(before, new)], 3, seed=1, room=1)
    rows = sum(new)
    k, v = random_rows(2, rows + 2, 3, spread), random_rows(3, rows + 2, 3, spread)
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    bounds = ends(new)
    for s, b in enumerate(before):
        for which, x in enumerate((k, v)):
            append(want[0][which], want[1][which], x[bounds[s] : bounds[s + 1]].float(), cache.table[s], b)
    run_op(append_op(cache, k, v, ints(bounds)))
    for which in range(2):  # the arithmetic is fixed: equal to the last bit, in the blocks that were not touched too
        assert torch.equal(cache.scales[which], want[1][which])
        assert torch.equal(cache.codes[which], want[0][which])
    again = [x.clone() for x in cache.codes]
    run_op(append_op(cache, k, v, ints(bounds)))  # the same call once more finds its own scales and changes nothing new
    assert all(torch.equal(a, b) for a, b in zip(again, cache.codes))


@pytest.mark.parametrize("bits", [0x3C7FFFFF, 0x3D7FFFFF, 0x3D000000, 0x3CFFFFFE, 0x3D2AAAAB])
def test_append_divides_as_ieee_does(bits):
    """Codes by scales that are there, one significand of all ones among them, for every bf16 value up to the largest code."""
    cache = Cache([1 + 63], 1, seed=33)
    scale = torch.tensor([bits], dtype=torch.int32, device="cuda").view(torch.float32)
    block = cache.table[0, 0].long()
    top = float(scale) * 127
    x = torch.arange(0x7F80, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.bfloat16)
    x = x[x.float() <= top]
    for part in x.split(63 * 128):
        rows = torch.zeros(63 * 128, dtype=torch.bfloat16, device="cuda")
        rows[: len(part)] = part * torch.where(torch.arange(len(part), device="cuda") % 2 == 0, 1, -1).bfloat16()
        rows = rows.view(63, 1, 128)
        for which in range(2):
            cache.scales[which][block] = scale
        run_op(append_op(cache, rows, rows, ints([0, 63])))
        want = torch.round(rows.float() / scale).to(torch.int8)[:, 0]
        for which in range(2):
            assert torch.equal(cache.scales[which][block], scale)
            assert torch.equal(cache.codes[which][block, 0, 1:], want)


def test_append_token_by_token_stays_near_the_values():
    """64 tokens appended one at a time: every raise of the scale rounds what is there once more, by half a step at most."""
    cache = Cache([64], 2, seed=4)
    k, v = random_rows(5, 64, 2), random_rows(6, 64, 2)
    for t in range(64):
        cache.lengths.fill_(t + 1)
        run_op(append_op(cache, k[t : t + 1].contiguous(), v[t : t + 1].contiguous(), ints([0, 1])))
    for which, x in enumerate((k, v)):
        top = x.float().abs().amax(-1)  # [64, heads]
        raises = (torch.cummax(top, 0).values.diff(dim=0) > 0).sum(0) + 1
        scale = cache.scales[which][cache.table[0, 0].long()]
        assert torch.equal(scale, top.amax(0) * (1 / 127))
        off = (cache.rows(which, 0) - x.double()).abs().amax((0, 2))
        assert (off <= scale * 0.5001 * raises).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_append_of_what_is_not_a_number_shows(value):
    cache = Cache([100], 2, seed=7)
    k, v = random_rows(8, 20, 2), random_rows(9, 20, 2)
    k[3, 1, 5] = value
    run_op(append_op(cache, k, v, ints([0, 20])))
    block = cache.table[0, 1].long()  # tokens 64 .. 99
    assert not torch.isfinite(cache.scales[0][block, 1]) and torch.isfinite(cache.scales[0][block, 0])
    assert torch.isfinite(cache.scales[1]).all()


def test_append_of_zeros_and_into_fresh_blocks():
    """A fresh block's scale does not look at what a block held before; zeros get the smallest scale."""
    cache = Cache([64 + 5], 1, seed=10)
    for x in cache.scales:
        x.fill_(float("nan"))
    k = torch.zeros(69, 1, 128, dtype=torch.bfloat16, device="cuda")
    run_op(append_op(cache, k, random_rows(11, 69, 1), ints([0, 69])))
    blocks = cache.table[0, :2].long()
    assert torch.equal(cache.scales[0][blocks], torch.full((2, 1), 1e-10, device="cuda"))
    assert torch.isfinite(cache.scales[1][blocks]).all() and (cache.rows(0, 0) == 0).all()


@pytest.mark.parametrize("lengths,extra", [([1], 0), ([64, 65, 63], 5), ([0, 300, 0, 1], 0), ([129] * 70, 3)])
def test_read(lengths, extra):
    from nano_omni_b200 import ops
    from tests.gpu_util import desc

    cache = Cache(lengths, 2, seed=12)
    total = sum(lengths)
    out = [torch.full((total + extra, 256), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    bounds = torch.full((len(lengths) + 1,), -1, dtype=torch.int32, device="cuda")
    run_op(ops.CacheRead(cache.desc(), total + extra).to(desc(out[0]), desc(out[1]), desc(bounds)))
    assert bounds.tolist() == ends(lengths)
    for which in range(2):
        want = torch.cat([cache.rows(which, s) for s in range(len(lengths))]).view(total, 256)
        # code * scale has 7 + 24 bits: one rounding to fp32, one to bf16
        assert torch.equal(out[which][:total], want.float().bfloat16())
        assert out[which][total:].isnan().all()


def test_read_past_the_capacity():
    from nano_omni_b200 import ops
    from tests.gpu_util import desc

    cache = Cache([100, 100, 100], 1, seed=13)
    out = [torch.full((130, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    bounds = torch.zeros(4, dtype=torch.int32, device="cuda")
    guard = [x.clone() for x in out]
    run_op(ops.CacheRead(cache.desc(), 120).to(desc(out[0][:120]), desc(out[1][:120]), desc(bounds)), status=64)
    assert bounds.tolist() == [0, 100, 120, 120]
    want = torch.cat([cache.rows(0, 0), cache.rows(0, 1)])[:120].view(120, 128)
    assert torch.equal(out[0][:120], want.float().bfloat16())
    assert all(torch.equal(x[120:].isnan(), g[120:].isnan()) for x, g in zip(out, guard))


def compare(cache, q, bounds, extra=0.0, prefix=None, slopes=None, **options):
    """The result is rounded to bf16 (HALF of it), probabilities to f16 (2^-11 = HALF / 8; below 2^-14 of the maximum by 2^-25
    absolute).  Codes and queries are exact; the scores in fp32 as in the masked attention: 0.2 HALF of sum p |v| covers them."""
    from tests.attention64 import attend

    out = torch.full((len(q), q.shape[1], 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    from tests.gpu_util import desc

    more = {} if prefix is None else {"prefix": ints(prefix)}
    more |= {} if slopes is None else {"slopes": slopes}
    run_op(attention_op(cache, q, ints(bounds), **more, **options).to(desc(out)))
    options.pop("cached_tokens", None)
    options.setdefault("causal", True)
    for s in range(len(bounds) - 1):
        rows = slice(bounds[s], bounds[s + 1])
        k, v = cache.rows(0, s), cache.rows(1, s)
        want, size = attend(q[rows], k, v, prefix=prefix[s] if prefix else 0, slopes=slopes, **options)
        most = v.abs().amax() if len(v) else 0.0
        allowed = HALF * (0.3 * size + want.abs()) + 2 * extra * size + len(k) * 2.0**-25 * most + 1e-30
        off = (out[rows].double() - want).abs()
        assert torch.isfinite(out[rows]).all()
        assert (off <= allowed).all(), f"sequence {s}: {(off / allowed).max().item():.3f} times the tolerance"
    assert out[bounds[-1] :].isnan().all() and out[: bounds[0]].isnan().all()


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (7, 1), (32, 1), (6, 3)])
@pytest.mark.parametrize("lengths", [[1], [64], [65, 63], [1021], [0, 2000, 1, 640]], ids=str)
def test_one_token(heads, kv_heads, lengths):
    cache = Cache(lengths, kv_heads, seed=14)
    compare(cache, random_rows(15, len(lengths) + 1, heads), ends([1] * len(lengths)))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lengths", [([3, 0, 5, 17], [3, 100, 700, 300]), ([40], [1500]), ([9, 2], [5, 2])], ids=str)
def test_a_few_tokens(new, lengths, causal):
    """Drafted tokens: causal among themselves; more tokens than the sequence holds see nothing where their place is negative."""
    cache = Cache(lengths, 2, seed=16)
    compare(cache, random_rows(17, sum(new) + 1, 6), ends(new), causal=causal)


@pytest.mark.parametrize("cap,biased,prefix", [(30.0, False, None), (0.5, True, [200, 0]), (0.0, True, None), (0.0, True, [9999, 65])])
def test_masks_cap_and_bias(cap, biased, prefix):
    cache = Cache([700, 130], 2, seed=18)
    slopes = torch.tensor([0.3, 0.01, 0.0, -0.002], device="cuda") if biased else None
    compare(cache, random_rows(19, 30, 4), [0, 20, 30], cap=cap, slopes=slopes, prefix=prefix, extra=1e-4)


def test_queries_of_any_size():
    """Rows from 2^-100 to 2^100 of the usual size: their f16 form is scaled by a power of two of its own."""
    cache = Cache([300], 1, seed=20)
    q = random_rows(21, 6, 1, 0.05)
    compare(cache, (q.float() * torch.tensor([2.0**-100, 2.0**-30, 1, 0, 16, 0.5], device="cuda")[:, None, None]).bfloat16(), [0, 6],
            causal=False)  # fmt: skip


@pytest.mark.parametrize("splits", [1, 2, 5, 8, 9, 17, 64])
@pytest.mark.parametrize("columns", [8, 16, 128])
@pytest.mark.parametrize("clusters", [False, True])
def test_shares(splits, columns, clusters):
    """Every division of the blocks, empty shares among them."""
    from nano_omni_b200.core import DType
    from nano_omni_b200.kernels.cache import CacheAttentionArguments, CacheAttentionConfig, CacheAttentionKernel
    from nano_omni_b200.kernels.masked import share_workspace_bytes
    from tests.attention64 import attend
    from tests.gpu_util import desc, run

    cache, c = (x := Cache([900, 0, 70], 2, seed=22)), x.desc()
    q = random_rows(23, 9, 4)
    out = torch.full_like(q, float("nan"))
    if clusters and (splits > 8 or (columns == 128 and splits > 1)):
        pytest.skip("no cluster holds so many shares")
    need = 0 if clusters else share_workspace_bytes(9, 4, splits)
    workspace = desc(torch.empty(need, dtype=torch.uint8, device="cuda"), DType.U8) if need else None
    bounds = ints([0, 4, 6, 9])
    arguments = CacheAttentionArguments(
        desc(q), c.key, c.value, c.key_scales, c.value_scales, c.table, c.lengths, desc(bounds), None, None, desc(out), 0, True,
        workspace=workspace,
    )  # fmt: skip
    run(CacheAttentionKernel(arguments, CacheAttentionConfig(columns=columns, kv_splits=splits)))
    for s, (a, b) in enumerate(((0, 4), (4, 6), (6, 9))):
        want, size = attend(q[a:b], cache.rows(0, s), cache.rows(1, s), causal=True)
        assert ((out[a:b].double() - want).abs() <= HALF * (0.3 * size + want.abs()) + 1e-3).all()


def test_blocks_that_are_not_there():
    """A block number outside the cache is not followed: its tokens count as masked and the status word says so."""
    from tests.attention64 import attend
    from tests.gpu_util import desc

    cache = Cache([200], 1, seed=24)
    q = random_rows(25, 1, 2)
    cache.table[0, 1] = 1 << 20
    out = torch.zeros_like(q)
    run_op(attention_op(cache, q, ints([0, 1])).to(desc(out)), status=64)
    keep = torch.ones(200, dtype=torch.bool)
    keep[64:128] = False
    cache.table[0, 1] = 0
    want, size = attend(q, cache.rows(0, 0)[keep.cuda()], cache.rows(1, 0)[keep.cuda()])
    assert ((out.double() - want).abs() <= HALF * (0.3 * size + want.abs()) + 1e-4).all()

    cache.table[0, 3] = -1
    before = [x.clone() for x in (*cache.codes, *cache.scales)]
    k = random_rows(26, 3, 1)
    run_op(append_op(cache, k, k, ints([0, 3])), status=64)
    assert all(torch.equal(a, b) for a, b in zip(before, (*cache.codes, *cache.scales)))
    cache.lengths.fill_(2)  # fewer than the new rows
    run_op(append_op(cache, k, k, ints([0, 3])), status=64)
    assert all(torch.equal(a, b) for a, b in zip(before, (*cache.codes, *cache.scales)))


def test_scales_that_are_not_finite_stay_in_their_block():
    """A block's scale that is not a number spoils the rows that see its tokens and no others."""
    from tests.gpu_util import desc

    cache = Cache([130], 1, seed=27)
    last = cache.table[0, 2].long()  # tokens 128 and 129
    q = random_rows(28, 130, 1)
    for which in range(2):
        cache.scales[which][last] = float("nan")
        out = torch.zeros_like(q)
        run_op(attention_op(cache, q, ints([0, 130])).to(desc(out)))
        assert torch.isfinite(out[:128]).all() and out[128:].isnan().all()
        cache.scales[which][last] = 0.01


def test_append_then_attend_then_read():
    """A generation's steps in one graph: append the step's tokens, attend, and the same tokens read back and attended at
    bf16; replayed with other lengths."""
    from nano_omni_b200 import ops
    from tests.attention64 import attend
    from tests.gpu_util import desc

    before, new = [70, 0, 200], [2, 3, 1]
    cache = Cache([b + n + 10 for b, n in zip(before, new)], 2, seed=29)
    cache.plain = [b + n for b, n in zip(before, new)]
    cache.lengths.copy_(ints(cache.plain))
    k, v, q = random_rows(30, 6, 2), random_rows(31, 6, 2), random_rows(32, 6, 4)
    bounds, out, again = ints(ends(new)), torch.zeros_like(q), torch.zeros_like(q)
    total = 400
    flat = [torch.zeros(total, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    key_bounds = torch.zeros(4, dtype=torch.int32, device="cuda")
    steps = [
        append_op(cache, k, v, bounds),
        attention_op(cache, q, bounds).to(desc(out)),
        ops.CacheRead(cache.desc(), total).to(desc(flat[0]), desc(flat[1]), desc(key_bounds)),
        ops.MaskedBf16Attention(desc(q.view(6, -1)), desc(flat[0]), desc(flat[1]), desc(bounds), total_heads=4,
                                key_bounds=desc(key_bounds), causal=True).to(desc(again)),
    ]  # fmt: skip
    arena = torch.empty(max(s.prepare()[1] for s in steps) + 256, dtype=torch.uint8, device="cuda")
    arena = arena[(-arena.data_ptr()) % 256 :]
    for step in steps:
        step.run(arena)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for step in steps:
            step.run(arena)
    for more in (0, 3):
        cache.plain = [b + n + more for b, n in zip(before, new)]
        cache.lengths.copy_(ints(cache.plain))
        out.zero_(), again.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s in range(3):
            rows = slice(sum(new[:s]), sum(new[: s + 1]))
            want, size = attend(q[rows], cache.rows(0, s), cache.rows(1, s), causal=True)
            assert ((out[rows].double() - want).abs() <= HALF * (0.3 * size + want.abs()) + 1e-4).all()
            # read back, K and V are rounded to bf16: a score by HALF of sum |q k| / sqrt(128), a value by HALF of itself
            near = HALF * (q[rows].double().abs().sum(-1).amax() * cache.rows(0, s).abs().amax() * 128**-0.5)
            assert ((again[rows].double() - want).abs() <= (2 * near + 3 * HALF) * size + HALF * want.abs()).all()


def run_attention_kernel(cache, q, bounds, columns, splits, causal=True, prefix=None, cap=0.0, slopes=None):
    """The kernel at a chosen division of the work, whatever the operator would choose."""
    from nano_omni_b200.core import DType
    from nano_omni_b200.kernels.cache import CacheAttentionArguments, CacheAttentionConfig, CacheAttentionKernel
    from nano_omni_b200.kernels.masked import share_workspace_bytes
    from tests.gpu_util import desc, run

    c, out, b = cache.desc(), torch.full_like(q, float("nan")), ints(bounds)
    need = share_workspace_bytes(len(q), q.shape[1], splits)
    workspace = desc(torch.empty(need, dtype=torch.uint8, device="cuda"), DType.U8) if need else None
    p = ints(prefix) if prefix else None
    arguments = CacheAttentionArguments(
        desc(q), c.key, c.value, c.key_scales, c.value_scales, c.table, c.lengths, desc(b), None if p is None else desc(p),
        None if slopes is None else desc(slopes), desc(out), 0, causal, cap=cap, workspace=workspace,
    )  # fmt: skip
    run(CacheAttentionKernel(arguments, CacheAttentionConfig(columns=columns, kv_splits=splits)))
    return out


def check(cache, out, q, bounds, extra=0.0, prefix=None, **options):
    """As in ``compare``; key shares are joined in fp32 and rounded once."""
    from tests.attention64 import attend

    for s in range(len(bounds) - 1):
        rows = slice(bounds[s], bounds[s + 1])
        if rows.start == rows.stop:
            continue
        k, v = cache.rows(0, s), cache.rows(1, s)
        want, size = attend(q[rows], k, v, prefix=prefix[s] if prefix else 0, **options)
        allowed = HALF * (0.3 * size + want.abs()) + 2 * extra * size + len(k) * 2.0**-25 * (v.abs().amax() if len(v) else 0) + 1e-30
        assert ((out[rows].double() - want).abs() <= allowed).all(), f"sequence {s}"
    assert out[bounds[-1] :].isnan().all()


@pytest.mark.parametrize("columns,sequences", [(8, 128), (8, 129), (16, 300), (128, 640), (128, 641)])
def test_many_sequences(columns, sequences):
    """As many sequences as a CTA orders by their lengths, and more, which it takes as they come."""
    g = torch.Generator().manual_seed(sequences)
    new = torch.randint(0, 3, (sequences,), generator=g)
    new[sequences // 2], new[-1] = 40, 0
    held = new + torch.randint(0, 90, (sequences,), generator=g)
    held[1], held[2] = 700, 0
    cache = Cache(held.tolist(), 2, seed=40)
    q, bounds = random_rows(41, int(new.sum()) + 2, 4), ends(new.tolist())
    for splits in (1, 3):
        check(cache, run_attention_kernel(cache, q, bounds, columns, splits), q, bounds, causal=True)


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("cap,prefix", [(0.0, None), (20.0, None), (0.0, [650, 0, 3]), (20.0, [650, 0, 3])])
def test_bias_and_cap_over_shares_of_tiles(splits, cap, prefix):
    """Several units of rows to a sequence, nearest tiles first, shares that a unit's rows do not reach."""
    cache = Cache([900, 290, 40], 2, seed=42)
    q, bounds = random_rows(43, 401, 4), [0, 120, 390, 400]
    slopes = torch.tensor([0.3, 0.01, 0.0, -0.002], device="cuda")
    options = {"causal": True, "prefix": prefix, "cap": cap, "slopes": slopes}
    for columns in (8, 128):
        check(cache, run_attention_kernel(cache, q, bounds, columns, splits, **options), q, bounds, extra=1e-4, **options)


@pytest.mark.parametrize("new", [1, 30])
def test_head_slice_and_scale(new):
    from tests.gpu_util import desc

    cache = Cache([400, 90], 1, seed=44)
    q, bounds = random_rows(45, 2 * new, 3), [0, new, 2 * new]
    out = torch.full((2 * new, 8, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    run_op(attention_op(cache, q, ints(bounds), total_heads=8, head_offset=4, scale=0.05).to(desc(out)))
    assert out[:, :4].isnan().all() and out[:, 7:].isnan().all()
    check(cache, out[:, 4:7], q, bounds, causal=True, scale=0.05)


@pytest.mark.parametrize("sequences", [256, 257, 600])
def test_append_and_read_of_many_sequences(sequences):
    from nano_omni_b200 import ops
    from tests.attention64 import append
    from tests.gpu_util import desc

    g = torch.Generator().manual_seed(sequences)
    new = torch.randint(0, 3, (sequences,), generator=g)
    new[5] = 100
    before = torch.randint(0, 70, (sequences,), generator=g)
    cache = Cache((before + new).tolist(), 1, seed=46)
    total, bounds = int(new.sum()), ends(new.tolist())
    k, v = random_rows(47, total, 1), random_rows(48, total, 1)
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s in range(sequences):
        for which, x in enumerate((k, v)):
            append(want[0][which], want[1][which], x[bounds[s] : bounds[s + 1]].float(), cache.table[s], int(before[s]))
    run_op(append_op(cache, k, v, ints(bounds)))
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])
    held = int((before + new).sum())
    out = [torch.full((held, 128), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    found = torch.full((sequences + 1,), -1, dtype=torch.int32, device="cuda")
    run_op(ops.CacheRead(cache.desc(), held).to(desc(out[0]), desc(out[1]), desc(found)))
    assert found.tolist() == ends((before + new).tolist())
    for which in range(2):
        rows = torch.cat([cache.rows(which, s) for s in range(sequences)]).view(held, 128)
        assert torch.equal(out[which], rows.float().bfloat16())


@pytest.mark.parametrize("new", [1, 20, 70])
def test_a_cache_past_32_bits(new):
    """Blocks whose codes lie further than 2^32 bytes behind the first; what lies between is never touched."""
    from nano_omni_b200 import ops
    from tests.attention64 import append
    from tests.gpu_util import desc

    cache, blocks = Cache([200], 8, seed=49), 66000  # x 8 heads x 8192 bytes = 4.3e9
    used = cache.table[0].long()
    far = torch.arange(blocks - len(used), blocks, device="cuda")
    for part, shape, kind in ((cache.codes, (blocks, 8, 64, 128), torch.int8), (cache.scales, (blocks, 8), torch.float32)):
        for which in range(2):
            whole = torch.empty(shape, dtype=kind, device="cuda")
            whole[far] = part[which][used]
            part[which] = whole
    cache.table[0] = far.int()
    k, v, q = random_rows(50, new, 8), random_rows(51, new, 8), random_rows(52, new, 16)
    want = [[part[which][far].clone() for which in range(2)] for part in (cache.codes, cache.scales)]
    local = torch.arange(len(far), device="cuda")
    for which, x in enumerate((k, v)):
        append(want[0][which], want[1][which], x.float(), local, 200 - new)
    run_op(append_op(cache, k, v, ints([0, new])))
    for which in range(2):
        assert torch.equal(cache.codes[which][far], want[0][which]) and torch.equal(cache.scales[which][far], want[1][which])
    compare(cache, q, [0, new])
    out = [torch.empty(200, 1024, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    run_op(ops.CacheRead(cache.desc(), 200).to(desc(out[0]), desc(out[1]), desc(ints([0, 0]))))
    for which in range(2):
        assert torch.equal(out[which], cache.rows(which, 0).view(200, 1024).float().bfloat16())


@pytest.mark.parametrize("new", [[1, 3], [40, 25]])
def test_rows_in_front_of_the_first_sequence(new):
    from tests.attention64 import append

    cache = Cache([300, 90], 2, seed=53)
    bounds = [5, 5 + new[0], 5 + sum(new)]
    k, v, q = (random_rows(seed, bounds[-1] + 3, heads) for seed, heads in ((54, 2), (55, 2), (56, 8)))
    want = [[x.clone() for x in part] for part in (cache.codes, cache.scales)]
    for s, n in enumerate(new):
        for which, x in enumerate((k, v)):
            append(want[0][which], want[1][which], x[bounds[s] : bounds[s + 1]].float(), cache.table[s], cache.plain[s] - n)
    run_op(append_op(cache, k, v, ints(bounds)))
    for which in range(2):
        assert torch.equal(cache.scales[which], want[1][which]) and torch.equal(cache.codes[which], want[0][which])
    compare(cache, q, bounds)


@pytest.mark.parametrize("new", [1, 20, 64])
def test_sequences_that_share_blocks(new):
    """The blocks of a common beginning stand in several rows of the table."""
    cache = Cache([200, 150, 128], 2, seed=57)
    cache.table[1, :2] = cache.table[0, :2]
    cache.table[2, :2] = cache.table[0, :2]
    compare(cache, random_rows(58, 3 * new, 4), [0, new, 2 * new, 3 * new])


def test_attention_on_two_streams_at_once():
    from nano_omni_b200 import _lib
    from tests.gpu_util import desc

    cache = Cache([5000, 40, 3000], 2, seed=59)
    for new in (1, 30):
        q, bounds = random_rows(60, 3 * new, 8), ints([0, new, 2 * new, 3 * new])
        want = torch.zeros_like(q)
        run_op(attention_op(cache, q, bounds).to(desc(want)))
        runs = []
        for _ in range(2):
            out = torch.zeros_like(q)
            op = attention_op(cache, q, bounds).to(desc(out))
            scratch = torch.empty(op.prepare()[1] + 256, dtype=torch.uint8, device="cuda")
            runs.append((op, out, scratch[(-scratch.data_ptr()) % 256 :], torch.cuda.Stream()))
        torch.cuda.synchronize()
        for _ in range(5):
            for op, _, scratch, stream in runs:
                op.run(scratch, stream.cuda_stream)
        torch.cuda.synchronize()
        assert _lib.read_status() == 0
        assert all(torch.equal(out, want) for _, out, _, _ in runs)
