"""Attention over packed and partly masked sequences, and the 8-bit cache of keys and values beside it, as timed cases.

Three kinds of case, each one pass of operators of ``nano_omni_b200.ops``:

* ``masked``  ``MaskedBf16Attention``: packed documents, causal with a prefix that every query sees, scores capped by a
              tanh, a bias that grows with distance, heads that share keys and values;
* ``append``  ``CacheAppend`` then ``CacheRead``: new keys and values quantised into the blocks of a cache (8 bits, one scale per
              block of 64 tokens and head), and the whole sequences read back as bf16 rows;
* ``cached``  ``CacheAttention``: a few queries per sequence (one, or a chunk) against such a cache.

Lengths are a function of the case, values of the seed.  A token's position counts from the start of its document; with
fewer queries than keys the last query stands at the last key.
"""

import math
import random

import torch

own = False

DIM = 128
BLOCK = 64  # tokens of a cache block


def listed():
    return [
        # a prompt with a system prefix in front, alone: the latency of one launch
        _masked("masked_prompt", rows=300, documents=1, heads=8, kv_heads=8, causal=True, prefix=77),
        # images and short clips of one batch packed into one sequence, each attending to itself; rows behind the last one
        _masked("masked_packed", rows=9461, documents=9, heads=14, kv_heads=14, padding=117),
        # a few text documents: capped scores, eight query heads to a key head
        _masked("masked_capped_groups", rows=4096, documents=3, heads=32, kv_heads=4, causal=True, cap=50.0),
        # one long document under a distance bias, odd length, a head slice of a wider output
        _masked("masked_distance", rows=15104, documents=1, heads=14, kv_heads=14, total_heads=28, causal=True, bias=True),
        # a video generated frame after frame behind 512 text tokens that see one another
        _masked("masked_clip", rows=32768, documents=1, heads=14, kv_heads=14, causal=True, prefix=512),
        # one decoding step of a batch: one token each, appended inside a block
        _append("append_step", sequences=64, rows=64, held=320, kv_heads=8),
        # the tokens of a clip appended behind what two sequences hold
        _append("append_clip", sequences=2, rows=15104, held=1021, kv_heads=14),
        # the smallest call: one token of one sequence
        _cached("cached_token", sequences=1, rows=1, held=1021, heads=14, kv_heads=14),
        # a decoding step of a batch with ragged contexts, four query heads to a key head
        _cached("cached_batch", sequences=64, rows=64, held=16384, heads=32, kv_heads=8),
        # one token against a very long context, distance bias: the keys divided over all SMs
        _cached("cached_long", sequences=1, rows=1, held=131072, heads=14, kv_heads=14, bias=True),
        # a few drafted tokens per sequence, some sequences without any, capped scores, seven heads to a key head
        _cached("cached_draft", sequences=16, rows=60, held=8192, heads=56, kv_heads=8, cap=30.0),
        # a frame of a clip against what was generated before; its tokens see one another
        _cached("cached_chunk", sequences=1, rows=1560, held=30000, heads=14, kv_heads=14, prefix=1 << 20),
    ]


def _masked(name, *, rows, documents, heads, kv_heads, total_heads=0, causal=False, prefix=0, cap=0.0, bias=False, padding=0, earlier=0):
    return {
        "name": name, "kind": "masked", "rows": rows, "documents": documents, "heads": heads, "kv_heads": kv_heads,
        "total_heads": total_heads or heads, "causal": causal, "prefix": prefix, "cap": cap, "bias": bias, "padding": padding,
        "earlier": earlier,
    }  # fmt: skip


def _append(name, *, sequences, rows, held, kv_heads):
    return {"name": name, "kind": "append", "sequences": sequences, "rows": rows, "held": held, "kv_heads": kv_heads}


def _cached(name, *, sequences, rows, held, heads, kv_heads, causal=True, prefix=0, cap=0.0, bias=False):
    return {
        "name": name, "kind": "cached", "sequences": sequences, "rows": rows, "held": held, "heads": heads,
        "kv_heads": kv_heads, "causal": causal, "prefix": prefix, "cap": cap, "bias": bias,
    }  # fmt: skip


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["masked", "masked", "append", "cached", "cached"])
    heads, kv_heads = rng.choice([(4, 4), (8, 8), (14, 14), (8, 2), (32, 4), (28, 14), (32, 8), (56, 8), (16, 1), (6, 2)])
    cap, bias = rng.choice([0.0, 0.0, 20.0, 50.0]), rng.random() < 0.3
    if kind == "append":
        sequences = rng.choice([1, 2, 7, 33, 64])
        rows = max(sequences, _log_between(rng, 1, 15104 * 14 // kv_heads // 2))
        held = _log_between(rng, 1, max(2, 65536 // sequences // kv_heads))
        case = _append("", sequences=sequences, rows=rows, held=held, kv_heads=kv_heads)
    elif kind == "cached":
        sequences = rng.choice([1, 1, 3, 16, 64])
        rows = sequences * (1 if rng.random() < 0.5 else _log_between(rng, 1, 1560 // sequences))
        held = _log_between(rng, 1, 131072)
        while sequences * held * kv_heads > 4_000_000 or rows * held * heads > 6e8:
            held //= 2
        prefix = rng.choice([0, 0, held // 3, 1 << 20])
        case = _cached("", sequences=sequences, rows=rows, held=max(1, held), heads=heads, kv_heads=kv_heads,
                       causal=rng.random() < 0.8, prefix=prefix, cap=cap, bias=bias)  # fmt: skip
    else:
        rows = _log_between(rng, 2, 32768)
        documents = min(rows, rng.choice([1, 1, 2, 5, 40]))
        earlier = rng.choice([0, 0, 130, 1000])
        while rows * (rows + documents * earlier) * heads > 1.5e10:
            rows = rows * 3 // 4
        case = _masked("", rows=rows, documents=min(documents, rows), heads=heads, kv_heads=kv_heads,
                       total_heads=heads * rng.choice([1, 2]), causal=rng.random() < 0.6, prefix=rng.choice([0, 0, 33, 512]),
                       cap=cap, bias=bias, padding=rng.choice([0, 0, 5, rows // 8]), earlier=earlier)  # fmt: skip
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- lengths
def _shares(total, count, seed):
    """``count`` ragged parts of ``total``; from three parts on one of them is empty."""
    rng = random.Random(seed)
    weights = [0.2 + rng.random() for _ in range(count)]
    if count >= 3:
        weights[rng.randrange(count)] = 0.0
    scale = total / sum(weights)
    ends = [0]
    for w in weights:
        ends.append(ends[-1] + w * scale)
    ends = [min(total, int(round(e))) for e in ends[:-1]] + [total]
    return [b - a for a, b in zip(ends, ends[1:])]


def _lengths(case):
    """(new tokens, tokens seen) of every document or sequence."""
    if case["kind"] == "masked":
        new = _shares(case["rows"] - case["padding"], case["documents"], case["rows"])
        return new, [n + case["earlier"] for n in new]
    count, rows, held = case["sequences"], case["rows"], case["held"]
    if rows == count:
        new = [1] * count
    else:
        new = _shares(rows, count, rows + held)
    rng = random.Random(held + count)
    # from an eighth of the longest on, over the logarithm; one sequence holds the longest
    before = [held] + [_log_between(rng, max(1, held // 8), held) for _ in range(count - 1)]
    return new, [b + n for b, n in zip(before, new)]


def _ends(lengths):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return ends


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(generator, *shape, std=1.0):
    return torch.randn(*shape, generator=generator, device="cuda", dtype=torch.float32) * std


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _slopes(heads):
    """Slopes of the distance bias: a geometric row from 1/2 down to 1/256."""
    return torch.logspace(-1, -8, heads, base=2.0, device="cuda", dtype=torch.float32)


def _rows(generator, tokens, heads, outlier=False):
    """bf16 [tokens, heads * 128]: unit noise, neighbouring tokens alike, one outlier channel per head of K."""
    x = _normal(generator, tokens, heads, DIM)
    x += _normal(generator, -(-tokens // 64), heads, DIM, std=0.3).repeat_interleave(64, 0)[:tokens]
    if outlier:
        channel = torch.randint(0, DIM, (heads,), generator=generator, device="cuda")
        x[:, torch.arange(heads, device="cuda"), channel] *= 6.0
    return x.bfloat16().view(tokens, heads * DIM)


def _cache(generator, lengths, kv_heads):
    """A cache whose blocks lie in any order, with some to spare: codes with their largest near 127, scales of unit data."""
    need = [-(-n // BLOCK) for n in lengths]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=generator, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    ends = _ends(need)
    for s, n in enumerate(need):
        table[s, :n] = order[ends[s] : ends[s] + n]
    shape = (blocks, kv_heads, BLOCK, DIM)
    codes = [(_normal(generator, *shape, std=32.0)).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [0.03 + 0.01 * torch.rand(blocks, kv_heads, generator=generator, device="cuda") for _ in range(2)]
    return {"key": codes[0], "value": codes[1], "key_scales": scales[0], "value_scales": scales[1], "table": table, "lengths": _ints(lengths)}


def _arena(num_bytes):
    buffer = torch.empty(num_bytes + 256, dtype=torch.uint8, device="cuda")
    return buffer[(-buffer.data_ptr()) % 256 :]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    new, seen = _lengths(case)
    state = {"case": case, "bounds": _ints(_ends(new)), "most": max(new)}
    kv_heads = case["kv_heads"]
    if case["kind"] == "append":
        state |= {name: _rows(generator, case["rows"], kv_heads, name == "k") for name in ("k", "v")}
        state["cache"] = _cache(generator, seen, kv_heads)
        tokens = sum(seen)
        state["read"] = [torch.zeros(tokens, kv_heads * DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        state["read_bounds"] = torch.zeros(len(seen) + 1, dtype=torch.int32, device="cuda")
    else:
        heads, total = case["heads"], case.get("total_heads", case["heads"])
        state["q"] = _rows(generator, case["rows"], heads)
        state["slopes"] = _slopes(heads) if case["bias"] else None
        state["prefix"] = _ints([min(case["prefix"], n) for n in seen]) if case["prefix"] else None
        state["out"] = torch.zeros(case["rows"], total, DIM, dtype=torch.bfloat16, device="cuda")
        if case["kind"] == "cached":
            state["cache"] = _cache(generator, seen, kv_heads)
        else:
            tokens = sum(seen) + case["padding"]
            state["k"], state["v"] = _rows(generator, tokens, kv_heads, True), _rows(generator, tokens, kv_heads)
            state["key_bounds"] = _ints(_ends(seen))
    if own:
        state["steps"], state["scratch"] = _steps(case, state)
    return state


def _steps(case, state):
    """The planned operators, as a program keeps them, and the scratch that they share."""
    from nano_omni_b200 import ops
    from nano_omni_b200.core import TensorDesc

    def desc(tensor):
        return None if tensor is None else TensorDesc.from_torch(tensor)

    cache = state.get("cache")
    if cache is not None:
        cache = ops.BlockCache(**{name: desc(tensor) for name, tensor in cache.items()})
    if case["kind"] == "append":
        read = state["read"]
        steps = [
            ops.CacheAppend(desc(state["k"]), desc(state["v"]), desc(state["bounds"]), cache).to(
                cache.key, cache.key_scales, cache.value, cache.value_scales
            ),
            ops.CacheRead(cache, read[0].shape[0]).to(desc(read[0]), desc(read[1]), desc(state["read_bounds"])),
        ]
    else:
        options = {
            "total_heads": case.get("total_heads", case["heads"]), "causal": case["causal"], "cap": case["cap"],
            "prefix": desc(state["prefix"]), "slopes": desc(state["slopes"]),
        }  # fmt: skip
        query, bounds = desc(state["q"]), desc(state["bounds"])
        if case["kind"] == "masked":
            options["head_offset"] = options["total_heads"] - case["heads"]
            options["key_bounds"] = desc(state["key_bounds"]) if case["earlier"] else None
            op = ops.MaskedBf16Attention(query, desc(state["k"]), desc(state["v"]), bounds, **options)
        else:
            options["cached_tokens"] = sum(_lengths(case)[1])
            op = ops.CacheAttention(query, bounds, cache, **options)
        steps = [op.to(desc(state["out"]))]
    return steps, _arena(max(step.prepare()[1] for step in steps))


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        for step in state["steps"]:
            step.run(state["scratch"])
    elif kind == "masked":
        _plain_masked(state)
    elif kind == "append":
        _plain_append(state)
        _plain_read(state)
    else:
        _plain_cached(state)
    if kind == "append":
        cache = state["cache"]
        return [*state["read"], state["read_bounds"], cache["key_scales"], cache["value_scales"]]
    return state["out"]


def _places(bounds, count):
    """Document and place in it of rows 0 .. count - 1; document len(bounds) - 1 behind the last bound."""
    row = torch.arange(count, device=bounds.device, dtype=torch.int32)
    document = torch.bucketize(row, bounds[1:], right=True)
    return document, row - torch.cat([bounds[:-1], bounds[-1:]])[document]


def _weights(scores, position, index, visible, case, slopes):
    """Softmax numerators and sums of scores [..., rows, keys] of heads in dimension -3; nothing visible gives zeros."""
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    if slopes is not None:
        scores = scores - slopes[:, None, None] * (position[..., :, None] - index).abs().float()
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    return p, p.sum(-1, keepdim=True)


def _plain_masked(state):
    case, bounds, key_bounds = state["case"], state["bounds"], state["key_bounds"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    tokens = state["k"].shape[0]
    q = state["q"].view(-1, heads, DIM).float().transpose(0, 1) / math.sqrt(DIM)
    k, v = (state[n].view(tokens, kv_heads, DIM).float().transpose(0, 1).repeat_interleave(heads // kv_heads, 0) for n in "kv")
    document, place = _places(bounds, case["rows"])
    key_document, index = _places(key_bounds, tokens)
    ahead = torch.cat([key_bounds.diff() - bounds.diff(), bounds[:1]])
    position = place + ahead[document]
    documents = len(bounds) - 1
    free = torch.cat([state["prefix"], bounds[:1]])[document] if state["prefix"] is not None else torch.zeros_like(position)
    first = case.get("total_heads", heads) - heads
    step = max(1, (1 << 28) // (heads * tokens))
    for a in range(0, case["rows"], step):  # a few rows at a time: the scores of all do not fit
        rows = slice(a, a + step)
        visible = (document[rows, None] == key_document) & (document[rows, None] < documents)
        if case["causal"]:
            visible &= (index <= position[rows, None]) | (index < free[rows, None])
        p, total = _weights(q[:, rows] @ k.transpose(1, 2), position[rows], index, visible, case, state["slopes"])
        out = (p @ v) / total.masked_fill(total == 0, 1.0)
        state["out"][rows, first : first + heads] = out.transpose(0, 1).bfloat16()


def _plain_append(state):
    cache, bounds = state["cache"], state["bounds"]
    kv_heads = state["case"]["kv_heads"]
    rows = state["k"].shape[0]
    sequence, place = _places(bounds, rows)
    before = cache["lengths"] - bounds.diff()
    position = before[sequence] + place
    block = cache["table"][sequence, position // BLOCK].long()
    kept = (before[sequence] - position // BLOCK * BLOCK).clamp(0, BLOCK)  # tokens that the block held before
    for name in ("key", "value"):
        codes, scales = cache[name], cache[name + "_scales"]
        x = state[name[0]].view(rows, kv_heads, DIM).float()
        most = torch.zeros_like(scales).scatter_reduce(0, block[:, None].expand(rows, kv_heads), x.abs().amax(-1), "amax")
        touched = torch.zeros(len(scales), dtype=torch.bool, device=x.device).index_fill(0, block, True)
        holds = torch.zeros(len(scales), dtype=torch.int32, device=x.device).index_put((block,), kept)
        old = scales.masked_fill((holds == 0)[:, None], 0.0)
        scale = torch.maximum(old, (most / 127.0).clamp(min=1e-10))
        again = torch.round(codes.float() * (old / scale)[..., None, None]).to(torch.int8)
        older = touched[:, None] & (torch.arange(BLOCK, device=x.device) < holds[:, None])
        codes.copy_(torch.where(older[:, None, :, None], again, codes))
        scales.copy_(torch.where(touched[:, None], scale, scales))
        codes[block, :, (position % BLOCK).long()] = torch.round(x / scale[block][..., None]).clamp(-127, 127).to(torch.int8)


def _plain_read(state):
    cache, (key, value) = state["cache"], state["read"]
    bounds = torch.cat([torch.zeros_like(cache["lengths"][:1]), cache["lengths"].cumsum(0, dtype=torch.int32)])
    sequence, place = _places(bounds, key.shape[0])
    block, slot = cache["table"][sequence, place // BLOCK].long(), (place % BLOCK).long()
    for name, out in (("key", key), ("value", value)):
        x = cache[name][block, :, slot].float() * cache[name + "_scales"][block][..., None]
        out.copy_(x.view(out.shape))
    state["read_bounds"].copy_(bounds)


def _plain_cached(state):
    case, cache, bounds = state["case"], state["cache"], state["bounds"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    count, most = len(bounds) - 1, state["most"]
    table = cache["table"].clamp(min=0).long()
    tokens = table.shape[1] * BLOCK
    k, v = (
        (cache[n][table].float() * cache[n + "_scales"][table][..., None, None])  # [sequences, blocks, kv heads, 64, 128]
        .permute(0, 2, 1, 3, 4)
        .reshape(count, kv_heads, 1, tokens, DIM)
        for n in ("key", "value")
    )
    new = bounds.diff()
    sequence, place = _places(bounds, case["rows"])
    q = torch.zeros(count, most, heads, DIM, device=k.device)
    q[sequence, place.long()] = state["q"].view(-1, heads, DIM).float() / math.sqrt(DIM)
    q = q.view(count, most, kv_heads, heads // kv_heads, DIM).permute(0, 2, 3, 1, 4)
    index = torch.arange(tokens, device=k.device, dtype=torch.int32)
    position = torch.arange(most, device=k.device, dtype=torch.int32) + (cache["lengths"] - new)[:, None]
    visible = (index < cache["lengths"][:, None, None]).expand(count, most, tokens)
    if case["causal"]:
        free = state["prefix"] if state["prefix"] is not None else torch.zeros_like(new)
        visible = visible & ((index <= position[..., None]) | (index < free[:, None, None]))
    scores = (q @ k.transpose(-1, -2)).view(count, heads, most, tokens)
    p, total = _weights(scores, position[:, None], index, visible[:, None], case, state["slopes"])
    p = p.view(count, kv_heads, heads // kv_heads, most, tokens)
    out = (p @ v).view(count, heads, most, DIM) / total.masked_fill(total == 0, 1.0)
    state["out"].copy_(out.transpose(1, 2)[sequence, place.long()])


# ---------------------------------------------------------------------------------------------------- figures
def _pairs(case):
    """Visible (query, key) pairs of a head."""
    pairs = 0
    for n, m in zip(*_lengths(case)):
        free = min(case["prefix"], m)
        if not case["causal"]:
            pairs += n * m
        else:  # query i sees max(free, m - n + i + 1) keys
            late = min(n, max(0, n - (free - (m - n))))  # queries whose own position lies past the prefix
            pairs += (n - late) * free + late * m - late * (late - 1) // 2
    return pairs


def work(case):
    """Inputs read once, outputs written once, two operations per multiply-add of a visible pair."""
    new, seen = _lengths(case)
    kv_heads = case["kv_heads"]
    if case["kind"] == "append":
        rows, blocks = sum(new), sum(-(-n // BLOCK) - (n - a) // BLOCK for n, a in zip(seen, new) if a)
        # new rows in, their blocks out with what they held before read once; then every token's codes in and its bf16 out
        older = sum((n - a) % BLOCK for n, a in zip(seen, new) if a)
        once = rows * DIM * (2 + 1) + older * DIM + blocks * 8 + sum(seen) * DIM * (1 + 2)
        return {"bytes": 2 * kv_heads * once, "flops": 0}
    heads = case["heads"]
    queries = 2 * sum(new) * heads * DIM * 2
    keys = 2 * sum(seen) * kv_heads * DIM * (1 if case["kind"] == "cached" else 2)
    return {"bytes": queries + keys, "flops": 4 * heads * DIM * _pairs(case)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_document(q, k, v, case, free, slopes):
    """[n, heads, 128] from q [n, heads, 128] against k, v [m, kv heads, 128], all in 64 bits."""
    n, heads, _ = q.shape
    m, kv_heads, _ = k.shape
    out = torch.zeros(n, heads, DIM, dtype=torch.float64, device=q.device)
    if n == 0 or m == 0:
        return out
    keys = torch.arange(m, device=q.device)
    for h in range(heads):
        mine, kh, vh = q[:, h], k[:, h // (heads // kv_heads)], v[:, h // (heads // kv_heads)]
        for a in range(0, n, 8192):
            at = torch.arange(a, min(n, a + 8192), device=q.device)[:, None] + (m - n)
            s = mine[a : a + 8192] @ kh.T / math.sqrt(DIM)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if slopes is not None:
                s -= slopes[h].double() * (at - keys).abs()
            if case["causal"]:
                s[(keys > at) & (keys >= free)] = -math.inf
            lse = torch.logsumexp(s, 1, keepdim=True)
            weights = torch.exp(s - lse).nan_to_num(0.0)  # a row that sees nothing: zeros
            out[a : a + 8192, h] = weights @ vh
    return out


def _exact_blocks(cache, name, s, length):
    order = cache["table"][s, : -(-length // BLOCK)].long()
    x = cache[name][order].double() * cache[name + "_scales"][order].double()[..., None, None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], DIM)[:length]


def exact(case, seed):
    state = prepare(case, seed)
    new, seen = _lengths(case)
    ends, key_ends = _ends(new), _ends(seen)
    kv_heads = case["kv_heads"]
    if case["kind"] == "append":
        return _exact_append(state, new, seen, ends)
    heads, total = case["heads"], case.get("total_heads", case["heads"])
    out = torch.zeros(case["rows"], total, DIM, dtype=torch.float64, device="cuda")
    q = state["q"].double().view(-1, heads, DIM)
    for d, (n, m) in enumerate(zip(new, seen)):
        if case["kind"] == "cached":
            k, v = (_exact_blocks(state["cache"], name, d, m) for name in ("key", "value"))
        else:
            k, v = (state[name][key_ends[d] : key_ends[d + 1]].double().view(m, kv_heads, DIM) for name in "kv")
        rows = slice(ends[d], ends[d + 1])
        out[rows, total - heads :] = _exact_document(q[rows], k, v, case, min(case["prefix"], m), state["slopes"])
    return out


def _exact_append(state, new, seen, ends):
    cache, found = state["cache"], []
    scales = {}
    for name in ("key", "value"):
        scales[name] = cache[name + "_scales"].double()
        parts = []
        for s, (n, m) in enumerate(zip(new, seen)):
            x = state[name[0]][ends[s] : ends[s + 1]].double().view(n, -1, DIM)
            rows = _exact_blocks(cache, name, s, m)
            for b in range((m - n) // BLOCK, -(-m // BLOCK)) if n else ():
                low, high = max(0, b * BLOCK - (m - n)), min(n, (b + 1) * BLOCK - (m - n))
                fresh, place = x[low:high], int(cache["table"][s, b])
                kept = max(0, (m - n) - b * BLOCK)
                need = (fresh.abs().amax((0, 2)) / 127).clamp(min=1e-10)
                scale = torch.maximum(need, scales[name][place]) if kept else need
                older = rows[b * BLOCK : b * BLOCK + kept]
                rows[b * BLOCK : b * BLOCK + kept] = torch.round(older / scale[:, None]) * scale[:, None]
                codes = torch.round(fresh / scale[:, None]).clamp(-127, 127)
                rows[b * BLOCK + kept : b * BLOCK + kept + len(fresh)] = codes * scale[:, None]
                scales[name][place] = scale
            parts.append(rows)
        found.append(torch.cat(parts).view(sum(seen), -1))
    return [*found, None, scales["key"], scales["value"]]
