"""Cases of the 8-bit paged KV cache's operators: what they are timed on, and what they must compute.

Three operators (kvsnap_b200.cache8), all on one layer's or one model's paged cache held as
float8_e4m3fn codes ``[2, blocks, block_size, kv_heads, head_dim]`` (0: keys, 1: values) with one
float32 scale a block, side and head, ``[blocks, 2, kv_heads]``, always a power of two:

* append: new keys and values, rotated on the way, into the pages of their sequences. The scale of a
  page that already holds tokens only grows; its older codes are then rounded again to the new scale.
  What the touched pages then stand for is read back with expand, and counts.
* attend: softmax(q k^T) v of every new token over its sequence's pages, causal.
* convert: whole blocks between 16-bit caches and the 8-bit one (compress, expand), every layer at once.

``own`` false: the plain form, in elementary torch operations. ``own`` true: the framework's calls.
"""
import math
import types

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0
ROTARY_BASE = 1000000.0


def listed():
    eight = {"q_heads": 32, "kv_heads": 8, "head_dim": 128, "block_size": 16, "dtype": "bf16"}      # Qwen3-8B
    small = {"q_heads": 16, "kv_heads": 8, "head_dim": 128, "block_size": 16, "dtype": "bf16"}      # Qwen3-1.7B
    large = {"q_heads": 64, "kv_heads": 8, "head_dim": 128, "block_size": 16, "dtype": "bf16"}      # Qwen3-32B
    shard = {"q_heads": 8, "kv_heads": 1, "head_dim": 128, "block_size": 16, "dtype": "fp16"}       # its TP-8 shard
    seven = {"q_heads": 28, "kv_heads": 4, "head_dim": 64, "block_size": 32, "dtype": "fp16"}       # 7 heads a group
    return [
        # One chat's decode step behind an 8k context: pure latency.
        {"name": "append_step_1", "op": "append", "interleaved": False, "seqs": 1, "new": 1, "new_hi": 1,
         "context": 8191, "context_hi": 8191, **eight},
        # A decode step of many sessions of unlike lengths, as they rotate through a worker.
        {"name": "append_step_64", "op": "append", "interleaved": False, "seqs": 64, "new": 1, "new_hi": 1,
         "context": 511, "context_hi": 8191, **eight},
        # Next turns of a few chats: ragged chunks that start and end inside pages.
        {"name": "append_turns", "op": "append", "interleaved": True, "seqs": 5, "new": 17, "new_hi": 701,
         "context": 130, "context_hi": 4099, **seven},
        # A whole 8k prompt.
        {"name": "append_prompt", "op": "append", "interleaved": False, "seqs": 1, "new": 8192, "new_hi": 8192,
         "context": 0, "context_hi": 0, **eight},
        # Decode of one short chat: latency.
        {"name": "attend_step_short", "op": "attend", "seqs": 1, "new": 1, "new_hi": 1,
         "context": 128, "context_hi": 128, **small},
        # Decode of one restored 32k session: few rows, a long axis to split.
        {"name": "attend_step_32k", "op": "attend", "seqs": 1, "new": 1, "new_hi": 1,
         "context": 32767, "context_hi": 32767, **large},
        # Decode of 64 rotating sessions of 512 to 8192 tokens.
        {"name": "attend_step_64", "op": "attend", "seqs": 64, "new": 1, "new_hi": 1,
         "context": 511, "context_hi": 8191, **eight},
        # Decode on one tensor-parallel shard: one KV head, all query heads of its group.
        {"name": "attend_step_shard", "op": "attend", "seqs": 16, "new": 1, "new_hi": 1,
         "context": 4001, "context_hi": 32767, **shard},
        # The next turn of three restored chats: a chunk of new tokens over a long cached context.
        {"name": "attend_turns", "op": "attend", "seqs": 3, "new": 97, "new_hi": 385,
         "context": 5003, "context_hi": 8191, **eight},
        # A whole 8k prompt, attending to itself.
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "new": 8192, "new_hi": 8192,
         "context": 0, "context_hi": 0, **eight},
        # An 8k session restored from a 16-bit snapshot goes into the 8-bit cache, every layer.
        {"name": "compress_session", "op": "compress", "layers": 36, "tokens": 8192, "kv_heads": 8, "head_dim": 128,
         "block_size": 16, "dtype": "bf16"},
        # A short session goes back to a 16-bit cache; its last block is partly filled.
        {"name": "expand_session", "op": "expand", "layers": 28, "tokens": 597, "kv_heads": 8, "head_dim": 128,
         "block_size": 16, "dtype": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "compress", "expand"])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
    case = {"op": op, "kv_heads": kv_heads, "head_dim": rng.choice([64, 128]), "block_size": rng.choice([16, 32]),
            "dtype": rng.choice(["bf16", "fp16"])}
    if op in ("compress", "expand"):
        case.update(layers=rng.randint(1, 36), tokens=_log_uniform(rng, 5, 8192))
        return case
    case["q_heads"] = kv_heads * group
    step = rng.random() < 0.5
    if step:
        seqs = _log_uniform(rng, 1, 64)
        new = new_hi = 1
    else:
        seqs = _log_uniform(rng, 1, 6)
        new = _log_uniform(rng, 2, 300)
        new_hi = _log_uniform(rng, new, 700)
    context = 0 if rng.random() < 0.1 else _log_uniform(rng, 20, 8000)
    context_hi = context if context == 0 else _log_uniform(rng, context, 32000 if seqs <= 2 and step else 8191)
    case.update(seqs=seqs, new=new, new_hi=new_hi, context=context, context_hi=context_hi)
    if op == "append":
        case["interleaved"] = rng.random() < 0.3
    return case


def _spread(lo, hi, count, turn):
    """``count`` whole numbers from lo to hi, evenly over their logarithm, in an order that mixes long and short."""
    if count == 1 or lo == hi:
        return [hi] * count
    at = [((i + 1) * turn) % 1.0 for i in range(count)]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** u)) - 1 for u in at]


def _sizes(case):
    """(new tokens, cached tokens before them) of each sequence."""
    return (_spread(case["new"], case["new_hi"], case["seqs"], 0.7548776662466927),
            _spread(case["context"], case["context_hi"], case["seqs"], 0.6180339887498949))


def _pages(tokens, block_size):
    return -(-tokens // block_size)


def _needed_scale(amax):
    """The smallest power of two s with amax <= 448 s; 0 for an empty block."""
    mantissa, exponent = torch.frexp(amax)
    shift = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-126)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), shift), torch.zeros_like(amax))


def _codes(values, scale):
    """float8_e4m3fn codes of fp32 values at a (broadcast) scale."""
    ratio = torch.where(scale > 0, values / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(values))
    return ratio.clamp(-LARGEST, LARGEST).to(E4M3)


def _normal(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _rotary(positions, dim):
    """cos and sin, [positions, dim / 2, 2] in 32 bits from 64-bit angles."""
    rate = ROTARY_BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * rate
    return torch.stack((angle.cos(), angle.sin()), dim=-1).to(torch.float32)


def _compressed_pool(blocks, case, gen):
    """A layer's 8-bit cache of ``blocks`` pages as earlier appends leave it: heads of unlike size, wide channels."""
    shape = (blocks, case["block_size"], case["kv_heads"], case["head_dim"])
    heads = torch.exp2(torch.randint(-2, 3, (2, 1, 1, case["kv_heads"], 1), generator=gen, device="cuda").float())
    values = torch.stack((_normal(shape, gen), _normal(shape, gen))) * heads
    scales = _needed_scale(values.abs().amax(dim=(2, 4)))                     # [2, blocks, heads]
    codes = _codes(values, scales[:, :, None, :, None])
    return codes, scales.permute(1, 0, 2).contiguous()


def _paged(case, gen, spare=8):
    """Block table, query starts and lengths of the case's sequences over a shuffled pool."""
    new, context = _sizes(case)
    lengths = [n + c for n, c in zip(new, context)]
    counts = [_pages(n, case["block_size"]) for n in lengths]
    blocks = sum(counts) + spare
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    firsts = [sum(counts[:i]) for i in range(len(counts))]
    column = torch.arange(max(counts), device="cuda", dtype=torch.int64)[None]
    within = torch.tensor(counts, device="cuda")[:, None]
    at = (torch.tensor(firsts, device="cuda")[:, None] + torch.minimum(column, within - 1)).clamp(min=0)
    table = torch.where(column < within, order[at], torch.zeros_like(order[at])).contiguous()
    start = torch.tensor([0] + [sum(new[: i + 1]) for i in range(len(new))], dtype=torch.int32, device="cuda")
    return types.SimpleNamespace(blocks=blocks, table=table, start=start, total=sum(new), max_query=max(new),
                                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))


def _projections(case, total, gen):
    """Query, key and value as the views of one fused projection that a model has in hand."""
    qh, kh, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    fused = _normal((total, (qh + 2 * kh) * d), gen, DTYPES[case["dtype"]])
    q, k, v = fused.split((qh * d, kh * d, kh * d), dim=1)
    return q.unflatten(1, (qh, d)), k.unflatten(1, (kh, d)), v.unflatten(1, (kh, d))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = types.SimpleNamespace(case=case)
    n, h, d, op = case["block_size"], case["kv_heads"], case["head_dim"], case["op"]
    if op in ("append", "attend"):
        s.paged = _paged(case, gen)
        s.codes, s.scales = _compressed_pool(s.paged.blocks, case, gen)
        s.q, s.k, s.v = _projections(case, s.paged.total, gen)
    else:
        count = _pages(case["tokens"], n)
        s.blocks8 = torch.randperm(count + 5, generator=gen, device="cuda")[:count]
        s.blocks16 = torch.randperm(count + 9, generator=gen, device="cuda")[:count]
        names = ["layers.%d" % i for i in range(case["layers"])]
        s.caches = {name: _normal((2, count + 9, n, h, d), gen, DTYPES[case["dtype"]]) for name in names}
        if op == "compress":                     # where the compressed blocks are read back
            s.targets = {name: torch.zeros((2, count, n, h, d), dtype=DTYPES[case["dtype"]], device="cuda")
                         for name in names}
            s.target_blocks = torch.randperm(count, generator=gen, device="cuda")
        s.codes, s.scales = {}, {}
        for name in names:
            if op == "expand":
                s.codes[name], s.scales[name] = _compressed_pool(count + 5, case, gen)
            else:
                s.codes[name] = torch.zeros((2, count + 5, n, h, d), dtype=E4M3, device="cuda")
                s.scales[name] = torch.zeros((count + 5, 2, h), device="cuda")
    if op == "append":
        new, context = _sizes(case)
        s.rotary = _rotary(max(a + b for a, b in zip(new, context)), d)
        rows = [(i, p) for i, (a, b) in enumerate(zip(new, context)) for p in range(b // n, _pages(a + b, n))]
        at = torch.tensor(rows, device="cuda")
        s.touched = s.paged.table[at[:, 0], at[:, 1]].to(torch.int64)
        s.read = torch.zeros((2, len(rows), n, h, d), dtype=DTYPES[case["dtype"]], device="cuda")
        s.read_blocks = torch.arange(len(rows), device="cuda")
    if own:
        from kvsnap_b200 import cache8
        if op in ("append", "attend"):
            s.batch = cache8.PagedBatch(s.paged.table, s.paged.start, s.paged.lengths, max_query=s.paged.max_query)
            s.cache = cache8.PagedCache8({"layer": s.codes}, {"layer": s.scales})
            if op == "append":
                s.back = s.cache.converter({"layer": s.read})
        else:
            s.cache = cache8.PagedCache8(s.codes, s.scales)
            s.converter = s.cache.converter(s.caches)
            s.back = s.cache.converter(s.targets) if op == "compress" else None
    return s


def _token_rows(p):
    """Of each new token: its sequence, its position, its place among the sequence's new tokens."""
    token = torch.arange(p.total, device="cuda")
    seq = torch.searchsorted(p.start[1:].to(torch.int64), token, right=True)
    place = token - p.start[seq]
    return seq, p.lengths[seq] - (p.start[seq + 1] - p.start[seq]) + place, place


def _rotated(x, cos_sin, interleaved):
    x = x.to(torch.float32)
    cos, sin = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_append(s):
    case, p, n = s.case, s.paged, s.case["block_size"]
    seq, position, _ = _token_rows(p)
    page = p.table[seq, position // n].to(torch.int64)
    slot = position % n
    fresh = torch.stack((_rotated(s.k, s.rotary[position], case["interleaved"]), s.v.to(torch.float32)), dim=1)
    # The scale each touched page needs for its new tokens, [blocks, 2, heads].
    amax = torch.zeros_like(s.scales)
    amax.index_reduce_(0, page, fresh.abs().amax(dim=-1), "amax")
    first = torch.full((s.scales.shape[0],), n, device="cuda", dtype=torch.int64)
    first.index_reduce_(0, page, slot, "amin")
    held = torch.where((first[s.touched] > 0)[:, None, None], s.scales[s.touched], torch.zeros(1, device="cuda"))
    scale = torch.maximum(held, _needed_scale(amax[s.touched]))
    # Older tokens of a touched page, at its new scale.
    old = s.codes[:, s.touched]
    again = _codes(old.to(torch.float32) * held.permute(1, 0, 2)[:, :, None, :, None],
                   scale.permute(1, 0, 2)[:, :, None, :, None])
    older = torch.arange(n, device="cuda")[None, :] < first[s.touched][:, None]
    bits = torch.where(older[None, :, :, None, None], again.view(torch.uint8), old.view(torch.uint8))
    s.codes.view(torch.uint8)[:, s.touched] = bits
    s.scales[s.touched] = scale
    new = _codes(fresh, s.scales[page][..., None])
    s.codes.view(torch.uint8)[:, page, slot] = new.view(torch.uint8).transpose(0, 1)
    values = s.codes[:, s.touched].to(torch.float32) * s.scales[s.touched].permute(1, 0, 2)[:, :, None, :, None]
    query = _rotated(s.q, s.rotary[position], case["interleaved"]).to(s.q.dtype)
    return {"query": query, "blocks": values.to(s.q.dtype)}


def _plain_attend(s):
    case, p = s.case, s.paged
    n, h, d = case["block_size"], case["kv_heads"], case["head_dim"]
    group = case["q_heads"] // h
    seq, position, place = _token_rows(p)
    table = p.table.to(torch.int64)
    held = s.codes[:, table].to(torch.float32) * s.scales[table].permute(2, 0, 1, 3)[:, :, :, None, :, None]
    keys, values = held.flatten(2, 3).permute(0, 1, 3, 2, 4)                  # [seqs, heads, tokens, dim]
    query = torch.zeros((case["seqs"], p.max_query, h, group, d), device="cuda")
    query[seq, place] = s.q.to(torch.float32).unflatten(1, (h, group))
    query = query.permute(0, 2, 3, 1, 4).flatten(2, 3)                        # [seqs, heads, group * rows, dim]
    scores = torch.matmul(query, keys.transpose(2, 3)) / math.sqrt(d)
    last = (p.lengths - (p.start[1:] - p.start[:-1]))[:, None] + torch.arange(p.max_query, device="cuda")
    hidden = torch.arange(keys.shape[2], device="cuda") > last.repeat(1, group)[:, None, :, None]
    scores.masked_fill_(hidden, -math.inf)
    scores.sub_(scores.amax(dim=-1, keepdim=True)).exp_()
    out = torch.matmul(scores, values) / scores.sum(dim=-1, keepdim=True)
    out = out.unflatten(2, (group, p.max_query)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return out[seq, place].to(s.q.dtype)


def _plain_compress(s):
    case, n = s.case, s.case["block_size"]
    names = sorted(s.caches)
    values = torch.stack([s.caches[name][:, s.blocks16] for name in names]).to(torch.float32)
    count = values.shape[2]
    slot = torch.arange(count * n, device="cuda").view(count, n)
    values = torch.where((slot < case["tokens"])[None, None, :, :, None, None], values, torch.zeros(1, device="cuda"))
    scale = _needed_scale(values.abs().amax(dim=(3, 5)))                      # [layers, 2, blocks, heads]
    codes = _codes(values, scale[:, :, :, None, :, None])
    return (codes.to(torch.float32) * scale[:, :, :, None, :, None]).to(DTYPES[case["dtype"]])


def _plain_expand(s):
    names = sorted(s.caches)
    codes = torch.stack([s.codes[name][:, s.blocks8].view(torch.uint8) for name in names]).view(E4M3)
    scale = torch.stack([s.scales[name][s.blocks8] for name in names]).permute(0, 2, 1, 3)
    return (codes.to(torch.float32) * scale[:, :, :, None, :, None]).to(DTYPES[s.case["dtype"]])


def _own(s):
    op, case = s.case["op"], s.case
    if op == "append":
        query = s.cache.append("layer", s.k, s.v, s.batch, query=s.q, rotary=s.rotary,
                               interleaved=case["interleaved"])
        s.back.expand(s.touched, s.read_blocks)
        return {"query": query, "blocks": s.read}
    if op == "attend":
        return s.cache.attend("layer", s.q, s.batch)
    if op == "compress":
        s.converter.compress(s.blocks16, s.blocks8, case["tokens"])
        s.back.expand(s.blocks8, s.target_blocks)
        return s.targets
    s.converter.expand(s.blocks8, s.blocks16)
    return s.caches


def run(s):
    """One pass."""
    if own:
        return _own(s)
    if s.case["op"] == "append":
        return _plain_append(s)
    if s.case["op"] == "attend":
        return _plain_attend(s)
    if s.case["op"] == "compress":
        values, into, blocks = _plain_compress(s), s.targets, s.target_blocks
    else:
        values, into, blocks = _plain_expand(s), s.caches, s.blocks16
    return {name: into[name].index_copy_(1, blocks, v) for name, v in zip(sorted(into), values)}


def work(case):
    """Bytes and operations of a pass: every input read once, every output written once."""
    h, d, n = case["kv_heads"], case["head_dim"], case["block_size"]
    two = 2                                                                   # bytes of a 16-bit element
    if case["op"] in ("compress", "expand"):
        elements = 2 * case["layers"] * case["tokens"] * h * d
        scales = 8 * case["layers"] * _pages(case["tokens"], n) * h
        again = elements * (two + 1) + scales                                 # one direction
        return {"bytes": again * (2 if case["op"] == "compress" else 1), "flops": 2 * elements}
    new, context = _sizes(case)
    total, qh = sum(new), case["q_heads"]
    if case["op"] == "append":
        touched = sum(_pages(a + b, n) - b // n for a, b in zip(new, context))
        kv, q, page = 2 * total * h * d, total * qh * d, 2 * touched * n * h * d
        rotary = 4 * total * d
        # projections in, codes and rotated query out; then the touched pages read and expanded
        return {"bytes": kv * (two + 1) + 2 * q * two + rotary + page * (1 + two) + 32 * touched * h,
                "flops": 6 * (kv // 2 + q) + 3 * kv}
    cached = sum(a + b for a, b in zip(new, context))
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, context))
    return {"bytes": 2 * cached * h * d + 8 * h * sum(_pages(a + b, n) for a, b in zip(new, context))
            + 2 * total * qh * d * two, "flops": 4 * d * qh * pairs}


def _nearest_e4m3(x):
    """Nearest value of the format to each x (ties to even), in 64 bits: 3 fraction bits, exponents -6 to 8."""
    size = x.abs().clamp(max=LARGEST)
    _, exponent = torch.frexp(size)
    step = torch.exp2((exponent.double() - 1).clamp(min=-6) - 3)
    return torch.sign(x) * torch.minimum(torch.round(size / step) * step, torch.full_like(size, LARGEST))


def _power_for(amax):
    """2^ceil(log2(amax / 448)), found from below and above in 64 bits."""
    power = torch.exp2(torch.floor(torch.log2(amax.clamp(min=1e-60) / LARGEST)) - 1)
    for _ in range(3):
        power = torch.where(amax > LARGEST * power, 2 * power, power)
    return torch.where(amax > 0, power.clamp(min=2.0 ** -126), torch.zeros_like(power))


def _stored(values, power):
    """What values stand for once held at a scale (0: an empty block)."""
    safe = torch.where(power > 0, power, torch.ones_like(power))
    return torch.where(power > 0, _nearest_e4m3(values / safe) * safe, torch.zeros_like(values))


def _turned(x, positions, interleaved):
    """x [tokens, heads, dim] turned by its positions' angles, as complex numbers."""
    dim = x.shape[-1]
    rate = torch.exp(-math.log(ROTARY_BASE) * torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None, None] * rate)
    if interleaved:
        return torch.view_as_real(torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
    pairs = torch.complex(x[..., : dim // 2].double(), x[..., dim // 2:].double()) * turn
    return torch.cat((pairs.real, pairs.imag), dim=-1)


def _exact_append(s):
    case, p, n = s.case, s.paged, s.case["block_size"]
    query, blocks = [], []
    for i, (new, context) in enumerate(zip(*_sizes(case))):
        first = int(p.start[i])
        rows = slice(first, first + new)
        where = context + torch.arange(new, device="cuda")
        query.append(_turned(s.q[rows], where, case["interleaved"]))
        fresh = torch.stack((_turned(s.k[rows], where, case["interleaved"]), s.v[rows].double()))
        low, high = context // n, _pages(context + new, n)
        pages = p.table[i, low:high].long()
        held = s.scales[pages].double().permute(1, 0, 2)                      # [2, pages, heads]
        if context % n == 0:
            held[:, 0] = 0
        held[:, 1:] = 0
        codes = s.codes[:, pages].double()
        values = torch.zeros_like(codes)
        values[:, 0, : context % n] = codes[:, 0, : context % n] * held[:, 0, None, :, None]
        flat = values.flatten(1, 2)
        flat[:, context - low * n: context - low * n + new] = fresh
        arrived = flat.clone()
        arrived[:, : context - low * n] = 0
        power = torch.maximum(held, _power_for(arrived.unflatten(1, (-1, n)).abs().amax(dim=(2, 4))))
        stored = _stored(flat.unflatten(1, (-1, n)), power[:, :, None, :, None]).flatten(1, 2)
        behind = context - low * n + new                                      # slots behind keep their codes
        stored[:, behind:] = (codes * power[:, :, None, :, None]).flatten(1, 2)[:, behind:]
        blocks.append(stored.unflatten(1, (-1, n)))
    return {"query": torch.cat(query), "blocks": torch.cat(blocks, dim=1)}


def _exact_attend(s):
    case, p, h = s.case, s.paged, s.case["kv_heads"]
    group = case["q_heads"] // h
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for i, (new, context) in enumerate(zip(*_sizes(case))):
        length, first = new + context, int(p.start[i])
        pages = p.table[i, : _pages(length, case["block_size"])].long()
        kv = (s.codes[:, pages].double() * s.scales[pages].double().permute(1, 0, 2)[:, :, None, :, None]).flatten(1, 2)[:, :length]
        for head in range(h):
            for row in range(0, new, 1024):
                many = min(1024, new - row)
                q = s.q[first + row: first + row + many, head * group: (head + 1) * group].double()
                score = torch.einsum("rgd,td->grt", q, kv[0, :, head]) * case["head_dim"] ** -0.5
                seen = torch.arange(length, device="cuda") <= context + row + torch.arange(many, device="cuda")[:, None]
                weight = torch.softmax(torch.where(seen, score, torch.full_like(score, -math.inf)), dim=-1)
                out[first + row: first + row + many, head * group: (head + 1) * group] = torch.einsum("grt,td->rgd", weight, kv[1, :, head])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    got = {}
    for name in sorted(s.caches):
        if case["op"] == "compress":
            values = s.caches[name][:, s.blocks16].double().flatten(1, 2)
            values[:, case["tokens"]:] = 0
            values = values.unflatten(1, (-1, case["block_size"]))
            got[name] = s.targets[name].double()
            got[name][:, s.target_blocks] = _stored(values, _power_for(values.abs().amax(dim=(2, 4)))[:, :, None, :, None])
        else:
            got[name] = s.caches[name].double()
            held = s.scales[name][s.blocks8].double().permute(1, 0, 2)
            got[name][:, s.blocks16] = s.codes[name][:, s.blocks8].double() * held[:, :, None, :, None]
    return got
