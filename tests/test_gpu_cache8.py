"""The 8-bit paged cache on a B200 against its definition in 64 bits (tests/cache8_reference.py).

Append and conversion: codes equal the nearest ones exactly where nothing is rotated, and stand within half
a step of the exactly rotated value where it is; scales are the definition's. Attention: within the bound
that cache8_reference.attend derives.
"""
import math

import pytest
import torch

from cache8_reference import E4M3, HALF, attend, nearest_code, power_for, rotate, rows_of

pytestmark = pytest.mark.gpu

BASE = 10000.0


def make_codes(order, blocks, block_size, heads, dim):
    """A zeroed uint8 cache [2, blocks, block_size, heads, dim], in one of the storage orders an engine uses."""
    if order == "sides":                     # [2, B, N, H, D]
        return torch.zeros((2, blocks, block_size, heads, dim), dtype=torch.uint8, device="cuda")
    if order == "heads":                     # [2, B, H, N, D]
        return torch.zeros((2, blocks, heads, block_size, dim), dtype=torch.uint8, device="cuda").transpose(2, 3)
    wide = torch.zeros((blocks, block_size, heads, 2 * dim), dtype=torch.uint8, device="cuda")      # K and V side by side
    return wide.unflatten(3, (2, dim)).permute(3, 0, 1, 2, 4)


class Paged:
    """A batch of sequences (new rows, cached tokens) over a shuffled pool, its cache filled with random codes."""

    def __init__(self, sequences, *, dim=128, block_size=16, heads=2, order="sides", seed=0, pad_rows=0, spare=3,
                 max_query="bound", poison=False, lengths=None):
        from kvsnap_b200.cache8 import PagedBatch, PagedCache8
        gen = torch.Generator().manual_seed(seed)
        self.block_size, self.heads, self.dim = block_size, heads, dim
        self.start, self.lengths = [0], []
        for new, context in sequences:
            self.start.append(self.start[-1] + new)
            self.lengths.append(new + context)
        if lengths is not None:
            self.lengths = list(lengths)
        counts = [-(-n // block_size) for n in self.lengths]
        blocks = sum(counts) + spare
        order_ids = torch.randperm(blocks, generator=gen).tolist()
        width = max(counts + [1]) + 2
        # Entries behind a sequence's pages are never read: give them ids outside the cache.
        self.table = [[] for _ in counts]
        at = 0
        for s, count in enumerate(counts):
            self.table[s] = order_ids[at: at + count] + [-7 if s % 2 else 1 << 30] * (width - count)
            at += count
        self.unowned = order_ids[at:]
        self.rows = self.start[-1] + pad_rows
        values = torch.randn((2, blocks, block_size, heads, dim), generator=gen)
        codes = (values * 100).clamp(-448, 448).to(E4M3).view(torch.uint8)
        scales = torch.exp2(torch.randint(-8, -4, (blocks, 2, heads), generator=gen).float())
        if poison:                            # nothing of this may be read as a token
            nan = torch.tensor(0x7F, dtype=torch.uint8)
            codes[:, self.unowned] = nan
            scales[self.unowned] = math.nan
            for s, length in enumerate(self.lengths):
                if length % block_size:
                    codes[:, self.table[s][length // block_size], length % block_size:] = nan
        self.codes_gpu = make_codes(order, blocks, block_size, heads, dim)
        self.codes_gpu.copy_(codes)
        self.scales_gpu = scales.cuda()
        self.cache = PagedCache8({"l": self.codes_gpu.view(E4M3)}, {"l": self.scales_gpu})
        bound = max([n for n, _ in sequences] + [0]) if max_query == "bound" else max_query
        self.batch = PagedBatch(torch.tensor(self.table, dtype=torch.int32).reshape(len(counts), width).cuda(),
                                torch.tensor(self.start, dtype=torch.int32).cuda(),
                                torch.tensor(self.lengths, dtype=torch.int32).cuda(), max_query=bound)
        self.gen = gen

    def random(self, heads, dtype, seed=1, fused=True):
        gen = torch.Generator().manual_seed(seed)
        x = torch.randn((self.rows, heads, self.dim), generator=gen).to(dtype)
        if not fused:
            return x, x.cuda()
        held = torch.zeros((self.rows, heads * self.dim + 48), dtype=dtype, device="cuda")     # rows of a wider tensor
        view = held[:, 16: 16 + heads * self.dim].unflatten(1, (heads, self.dim))
        view.copy_(x)
        return x, view

    def codes(self):
        return self.codes_gpu.cpu().contiguous()

    def scales(self):
        return self.scales_gpu.cpu()


def check_attend(p, dtype, group, *, scale=None, out=None, seed=1):
    q, q_gpu = p.random(p.heads * group, dtype, seed)
    got = p.cache.attend("l", q_gpu, p.batch, scale=scale, out=out)
    p.cache.check()
    expected, bound = attend(q, p.codes(), p.scales(), p.table, p.start, p.lengths, p.block_size,
                             p.dim ** -0.5 if scale is None else scale)
    got = got.cpu().to(torch.float64)
    owned = [row for _, row, _ in rows_of(p.start, p.lengths)]
    assert torch.isfinite(got[owned]).all()
    over = ((got - expected).abs() - bound)[owned]
    assert (over <= 0).all(), f"worst {over.max().item():.3g} over its bound"
    return got


SHAPES = [
    # head_dim, block_size, kv_heads, group, type
    (128, 16, 8, 4, torch.bfloat16),
    (128, 16, 1, 8, torch.float16),
    (64, 32, 4, 7, torch.float16),
    (64, 16, 2, 1, torch.bfloat16),
    (128, 48, 3, 2, torch.bfloat16),
    (128, 16, 2, 16, torch.float16),
    (64, 16, 5, 3, torch.float16),
    (128, 128, 2, 5, torch.bfloat16),
]

STEPS = [
    [(1, 0)],
    [(1, 1)],
    [(1, 15), (1, 16), (1, 17)],
    [(1, 127), (1, 128), (1, 0), (1, 255), (1, 63)],
    [(1, 700), (1, 3), (1, 1500)],
]

CHUNKS = [
    [(2, 0)],
    [(3, 14), (1, 0), (0, 5), (20, 100)],
    [(33, 0), (1, 300)],
    [(129, 127)],
    [(70, 513), (64, 64), (5, 1)],
    [(300, 0)],
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", STEPS, ids=str)
def test_attend_step(shape, sequences):
    dim, block_size, heads, group, dtype = shape
    check_attend(Paged(sequences, dim=dim, block_size=block_size, heads=heads, poison=True), dtype, group)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", CHUNKS, ids=str)
def test_attend_chunk(shape, sequences):
    dim, block_size, heads, group, dtype = shape
    check_attend(Paged(sequences, dim=dim, block_size=block_size, heads=heads, poison=True), dtype, group)


@pytest.mark.parametrize("count,longest,heads,group", [
    (64, 300, 8, 4), (64, 900, 8, 2), (130, 250, 8, 1), (12, 2100, 8, 4), (3, 2600, 8, 2), (160, 100, 1, 8), (5, 1500, 3, 4)])
def test_attend_steps_cut_or_not(count, longest, heads, group):
    """Batches on both sides of the rule that cuts a step's work: many units of several chunks, uneven and even."""
    even, uneven = [(1, longest)] * count, [(1 + s % 2, s * 37 % longest) for s in range(count)]
    for sequences in (even, uneven):
        check_attend(Paged(sequences, dim=64, heads=heads, poison=True), torch.bfloat16, group)


@pytest.mark.parametrize("order", ["sides", "heads", "beside"])
@pytest.mark.parametrize("sequences", [[(1, 200), (1, 31)], [(40, 75), (2, 9)]], ids=str)
def test_attend_storage_orders(order, sequences):
    check_attend(Paged(sequences, heads=4, order=order, poison=True), torch.bfloat16, 4)


@pytest.mark.parametrize("max_query", [None, 1, 9])
def test_attend_without_a_bound_and_with_a_loose_one(max_query):
    check_attend(Paged([(1, 200), (1, 31), (1, 0)], max_query=max_query), torch.bfloat16, 4)


@pytest.mark.parametrize("sequences,lengths", [
    ([(1, 5), (1, 0), (1, 30)], [6, 0, 31]),              # a padded entry of a captured batch
    ([(4, 0), (3, 9)], [2, 12]),                          # rows before the sequence's first token
    ([(40, 0), (0, 0), (9, 0)], [17, 0, 0]),
])
def test_rows_that_see_nothing_are_zeros(sequences, lengths):
    p = Paged(sequences, lengths=lengths, poison=True)
    got = check_attend(p, torch.bfloat16, 2)
    for s, row, position in rows_of(p.start, p.lengths):
        if position < 0:
            assert (got[row] == 0).all()


@pytest.mark.parametrize("sequences", [[(1, 40), (1, 3)], [(19, 40), (2, 3)]], ids=str)
def test_rows_of_nobody_are_left(sequences):
    p = Paged(sequences, pad_rows=13)
    out = torch.full((p.rows, p.heads * 4, p.dim), 7.0, dtype=torch.float16, device="cuda")
    p.cache.attend("l", p.random(p.heads * 4, torch.float16)[1], p.batch, out=out)
    p.cache.check()
    assert (out[p.start[-1]:] == 7).all() and (out[: p.start[-1]] != 7).any()


@pytest.mark.parametrize("sequences", [[(1, 300)], [(30, 300)]], ids=str)
@pytest.mark.parametrize("scale", [0.0, 0.02, 1.7])
def test_attend_scale(sequences, scale):
    check_attend(Paged(sequences), torch.float16, 2, scale=scale)


@pytest.mark.parametrize("sequences", [[(1, 530)], [(45, 530)]], ids=str)
@pytest.mark.parametrize("side", [0, 1])
def test_attend_scales_far_apart_and_zero(sequences, side):
    """Blocks of values a thousand times smaller or larger than their neighbours, and empty blocks."""
    p = Paged(sequences, seed=3)
    powers = torch.tensor([2.0 ** -8, 2.0 ** -18, 0.0, 2.0 ** -9, 2.0 ** -13])
    turn = powers[torch.arange(p.scales_gpu.shape[0]) % 5]
    p.scales_gpu[:, side] = turn[:, None].cuda()
    check_attend(p, torch.bfloat16, 4)


@pytest.mark.parametrize("sequences", [[(1, 100)], [(20, 100)]], ids=str)
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -20, 2.0 ** 60])
def test_attend_query_sizes(sequences, size):
    """Queries far from 1 in size: bf16's exponents do not fit 16-bit products unscaled."""
    p = Paged(sequences)
    q, q_gpu = p.random(p.heads * 2, torch.bfloat16)
    q, q_gpu = q * size, q_gpu * size
    got = p.cache.attend("l", q_gpu, p.batch, scale=0.1 / size).cpu().double()
    expected, bound = attend(q, p.codes(), p.scales(), p.table, p.start, p.lengths, p.block_size, 0.1 / size)
    assert ((got - expected).abs() <= bound).all()


@pytest.mark.parametrize("sequences", [[(1, 90)], [(24, 90)]], ids=str)
def test_attend_nan_is_kept_to_the_rows_that_see_it(sequences):
    """A NaN among a sequence's own values reaches the rows that see it, not rows before it or other sequences."""
    p = Paged(sequences + [(2, 50)])
    last = p.lengths[0] - 1
    p.codes_gpu[1, p.table[0][last // 16], last % 16, 0, 5] = 0x7F
    q_gpu = p.random(p.heads * 2, torch.bfloat16)[1]
    got = p.cache.attend("l", q_gpu, p.batch).cpu()
    final = p.start[1] - 1
    assert got[final, :2, 5].isnan().all()
    got[final, :2, 5] = 0
    assert got.isfinite().all()


def test_attend_long_and_split():
    """One long sequence beside short ones: the long axis is split and joined."""
    check_attend(Paged([(1, 9000), (1, 5), (1, 700)], heads=1), torch.bfloat16, 2)
    check_attend(Paged([(9, 6000), (1, 5)], heads=1), torch.float16, 4)


def test_attend_many_sequences():
    p = Paged([(1, (37 * i) % 211) for i in range(300)], heads=1, dim=64)
    check_attend(p, torch.float16, 4)


def test_attend_offsets_beyond_32_bits():
    """Blocks that lie more than 4 GiB into a side, and a side more than 4 GiB from the other."""
    from kvsnap_b200.cache8 import PagedBatch, PagedCache8
    blocks, heads, dim = 290000, 8, 128
    codes = torch.zeros((2, blocks, 16, heads, dim), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((blocks, 2, heads), device="cuda")
    cache = PagedCache8({"l": codes.view(E4M3)}, {"l": scales})
    table = [[289999, 3, 289990, 289991, 270000]]
    gen = torch.Generator().manual_seed(5)
    key, value = (torch.randn((70, heads, dim), generator=gen).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((70, 16, dim), generator=gen).to(torch.bfloat16)
    batch = PagedBatch(torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor([0, 70], dtype=torch.int32).cuda(),
                       torch.tensor([70], dtype=torch.int32).cuda())
    cache.append("l", key.cuda(), value.cuda(), batch)
    got = cache.attend("l", q.cuda(), batch).cpu().double()
    cache.check()
    small = codes[:, table[0]].cpu()
    for i in range(5):
        rows = slice(16 * i, min(70, 16 * i + 16))
        for h in range(heads):
            power = power_for(value[rows, h].abs().max().item())
            assert scales[table[0][i], 1, h].item() == power
            assert torch.equal(small[1, i, : len(range(70)[rows]), h], nearest_code(value[rows, h].double(), power))
    expected, bound = attend(q, small, scales[table[0]].cpu(), [[0, 1, 2, 3, 4]], [0, 70], [70], 16, dim ** -0.5)
    assert ((got - expected).abs() <= bound).all()


# ---- append ------------------------------------------------------------------------------


def check_append(p, dtype, *, group=0, rotary_dim=0, interleaved=False, base=BASE, data=None):
    from kvsnap_b200.cache8 import rotary_table
    before_codes, before_scales = p.codes(), p.scales()
    (key, key_gpu), (value, value_gpu) = p.random(p.heads, dtype, 11), p.random(p.heads, dtype, 12)
    if data is not None:
        key_gpu.copy_(data[0]), value_gpu.copy_(data[1])
        key, value = data
    q = q_gpu = None
    if group:
        q, q_gpu = p.random(p.heads * group, dtype, 13)
    rotary = rotary_table(max(p.lengths + [1]), rotary_dim, base) if rotary_dim else None
    got_q = p.cache.append("l", key_gpu, value_gpu, p.batch, query=q_gpu, rotary=rotary, interleaved=interleaved)
    p.cache.check()
    codes, scales = p.codes(), p.scales()
    positions = {row: position for _, row, position in rows_of(p.start, p.lengths)}
    at = [max(positions.get(row, 0), 0) for row in range(p.rows)]
    exact_k = rotate(key.double(), at, rotary_dim, base, interleaved) if rotary_dim else key.double()
    # 32-bit rotation: two products and a sum of 2^-24 each, of sizes up to |a| + |b| (pairs lie in one row).
    slack = 3 * 2.0 ** -24 * 2 * key.double().abs().nan_to_num(0, 0, 0).amax(dim=2) if rotary_dim \
        else torch.zeros(key.shape[:2], dtype=torch.float64)
    expected_codes, expected_scales = before_codes.clone(), before_scales.clone()
    n = p.block_size
    for s, length in enumerate(p.lengths):
        new = p.start[s + 1] - p.start[s]
        held = max(length - new, 0)
        if new == 0 or length == 0:
            continue
        for page in range(held // n, -(-length // n)):
            block, first = p.table[s][page], max(held - page * n, 0)
            end = min(length - page * n, n)
            rows = [p.start[s + 1] - length + page * n + slot for slot in range(first, end)]
            for side, rows_in in ((0, exact_k), (1, value.double())):
                for h in range(p.heads):
                    x = rows_in[rows, h]
                    finite = x[x.isfinite()]
                    old = before_scales[block, side, h].item() if first else 0.0
                    power = max(old, power_for(finite.abs().max().item() if finite.numel() else 0.0))
                    if side == 0 and rotary_dim and scales[block, side, h].item() != power:
                        # a border of the scale within the rotation's rounding
                        power = scales[block, side, h].item()
                        near = finite.abs().max().item()
                        assert power_for(near - slack[rows, h].max().item()) <= power <= power_for(near + slack[rows, h].max().item())
                    expected_scales[block, side, h] = power
                    if first:
                        older = before_codes[side, block, :first, h].view(E4M3).double() * old
                        expected_codes[side, block, :first, h] = nearest_code(older, power) if power > old \
                            else before_codes[side, block, :first, h]
                    want = nearest_code(x, power)
                    got = codes[side, block, first:end, h]
                    if side == 0 and rotary_dim:
                        stands = got.view(E4M3).double() * power
                        allowed = torch.maximum(2.0 ** -4 * x.abs(), torch.full_like(x, 2.0 ** -10 * power)) \
                            + slack[rows, h][:, None] * (1 + 2.0 ** -4)
                        good = ((stands - x.clamp(-448 * power, 448 * power)).abs() <= allowed) | (x.isnan() & stands.isnan())
                        assert good.all()
                        want = got
                    expected_codes[side, block, first:end, h] = want
    assert torch.equal(scales, expected_scales)
    assert torch.equal(codes, expected_codes)
    if group:
        exact_q = rotate(q.double(), at, rotary_dim, base, interleaved)
        q_slack = 3 * 2.0 ** -24 * 2 * q.double().abs().amax(dim=2, keepdim=True)
        half = HALF[dtype]
        for row, position in positions.items():
            if position >= 0:
                off = (got_q[row].cpu().double() - exact_q[row]).abs()
                assert (off <= half * exact_q[row].abs() + q_slack[row] * (1 + half) + 2.0 ** -25).all()


APPENDS = [
    [(1, 0)],
    [(1, 15), (1, 16), (1, 33), (1, 0), (1, 47)],
    [(5, 3), (16, 16), (0, 9), (40, 31), (1, 0)],
    [(100, 0)],
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", APPENDS, ids=str)
def test_append_plain(shape, sequences):
    dim, block_size, heads, _, dtype = shape
    check_append(Paged(sequences, dim=dim, block_size=block_size, heads=heads), dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (64, 64), (128, 32), (64, 48)])
@pytest.mark.parametrize("sequences", APPENDS[1:3], ids=str)
def test_append_rotated(interleaved, dim, rotary_dim, sequences):
    check_append(Paged(sequences, dim=dim, pad_rows=3), torch.bfloat16, group=3, rotary_dim=rotary_dim,
                 interleaved=interleaved)
    check_append(Paged(sequences, dim=dim, order="beside"), torch.float16, group=1, rotary_dim=rotary_dim,
                 interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,block_size,rotary_dim", [(128, 48, 128), (64, 80, 64), (128, 32, 48)])
def test_append_rotated_to_pages_of_more_rows_than_a_warp_holds(interleaved, dim, block_size, rotary_dim):
    p = Paged([(100, 7), (3, 46), (50, 0), (1, 90)], dim=dim, block_size=block_size, heads=3)
    check_append(p, torch.float16, group=2, rotary_dim=rotary_dim, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_of_a_long_chunk_turns_its_queries_in_a_launch_of_their_own(interleaved):
    p = Paged([(1900, 5), (0, 40), (700, 33), (1, 0)], heads=8, pad_rows=5)
    check_append(p, torch.bfloat16, group=4, rotary_dim=128, interleaved=interleaved)
    check_append(Paged([(2500, 9)], dim=64, heads=4), torch.float16, group=9, rotary_dim=32, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_rotated_values_not_finite(interleaved):
    p = Paged([(6, 20), (1, 3), (2, 1)], heads=2, dim=64)
    values = torch.randn(p.rows, 2, 64, generator=torch.Generator().manual_seed(3))
    values[1, 0, 5], values[2, 1, 40], values[3, 0, 0], values[6, 1, 63] = math.inf, -math.inf, math.nan, math.inf
    values = values.to(torch.bfloat16)
    check_append(p, torch.bfloat16, data=(values, values), rotary_dim=64, interleaved=interleaved)


def test_append_far_positions():
    """Angles of far positions come from 64 bits."""
    p = Paged([(1, 131071), (3, 99990)], heads=1, dim=64)
    check_append(p, torch.bfloat16, group=1, rotary_dim=64)


@pytest.mark.parametrize("sequences", [[(1, 20), (1, 7)], [(9, 20), (30, 7)]], ids=str)
def test_append_grows_a_scale_and_keeps_a_large_one(sequences):
    """New tokens a thousand times larger re-round a page's older codes; much smaller ones leave its scale."""
    for size in (1000.0, 0.001):
        p = Paged(sequences, heads=2)
        data = [(torch.randn(p.rows, 2, 128, generator=torch.Generator().manual_seed(i)) * size).to(torch.bfloat16)
                for i in (4, 5)]
        check_append(p, torch.bfloat16, data=data)


def test_append_values_at_borders_and_not_finite():
    """448 times a power of two is its scale's largest value; infinities saturate; NaN stays; zeros have scale 0."""
    p = Paged([(6, 0), (2, 18), (1, 3)], heads=2, dim=64)
    values = torch.zeros(p.rows, 2, 64)
    values[0, 0, :4] = torch.tensor([448.0, -3.0, 2.0 ** -10, 1.5])
    values[1, 1, :3] = torch.tensor([450.0, math.inf, -math.inf])
    values[2, 1, 0] = math.nan
    values[6, 0, :2] = torch.tensor([2.0 ** -130, -(2.0 ** -133)])
    values[8, 1, 0] = math.inf
    check_append(p, torch.bfloat16, data=(values.to(torch.bfloat16), values.flip(2).to(torch.bfloat16)))


def test_append_to_a_reused_page_starts_anew():
    """A page that an earlier sequence left, codes and a large scale, is new once its first slot is written."""
    p = Paged([(2, 16), (1, 0)], heads=1)
    p.scales_gpu.fill_(2.0 ** 40)
    check_append(p, torch.bfloat16)


@pytest.mark.parametrize("lengths", [[0, 5], [2, 0]])
def test_append_padded_entries_write_nothing(lengths):
    check_append(Paged([(1, 0), (1, 0)], lengths=[lengths[0] and 1, lengths[1] and 1], pad_rows=2), torch.bfloat16)
    check_append(Paged([(4, 0), (4, 1)], lengths=lengths, pad_rows=2), torch.bfloat16)


# ---- conversion -----------------------------------------------------------------------------


@pytest.mark.parametrize("dim,block_size,heads,dtype", [(128, 16, 8, torch.bfloat16), (64, 32, 3, torch.float16),
                                                       (128, 48, 1, torch.bfloat16), (64, 16, 2, torch.bfloat16),
                                                       (128, 64, 2, torch.float16)])
@pytest.mark.parametrize("tokens", [None, 0, 1, 45, 64])
def test_convert(dim, block_size, heads, dtype, tokens):
    from kvsnap_b200.cache8 import PagedCache8
    gen = torch.Generator().manual_seed(9)
    names, blocks8, blocks16 = ["b", "a", "c"], 9, 7
    cache = PagedCache8.allocate(names, blocks8, block_size, heads, dim)
    for name in names:
        cache.codes[name].view(torch.uint8).fill_(0x21)
        cache.scales[name].fill_(3.0)
    wide = {}
    for i, name in enumerate(names):
        x = torch.randn((2, blocks16, block_size, heads, dim), generator=gen) * 4.0 ** (i - 1)
        x[:, 2, : block_size // 2] *= 100
        x[0, 4] = 0
        wide[name] = x.to(dtype)
    wide["a"][1, 2, 0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan]).to(dtype)
    gpu = {name: x.cuda() for name, x in wide.items()}
    source, target = [2, 4, 6, 0], [8, 1, 5, 2]
    converter = cache.converter(gpu)
    converter.compress(source, torch.tensor(target).cuda(), tokens)
    cache.check()
    for name in names:
        codes, scales = cache.codes[name].view(torch.uint8).cpu(), cache.scales[name].cpu()
        left = [b for b in range(blocks8) if b not in target]
        assert (codes[:, left] == 0x21).all() and (scales[left] == 3.0).all()
        for i, (a, b) in enumerate(zip(source, target)):
            valid = block_size if tokens is None else min(max(tokens - i * block_size, 0), block_size)
            for side in range(2):
                for h in range(heads):
                    x = wide[name][side, a, :, h].double().clone()
                    x[valid:] = 0
                    finite = x[x.isfinite()]
                    power = power_for(finite.abs().max().item())
                    assert scales[b, side, h].item() == power
                    assert torch.equal(codes[side, b, :, h], nearest_code(x, power))
    back = {name: torch.full_like(x, 5) for name, x in gpu.items()}
    cache.converter(back).expand(target, source)
    cache.check()
    for name in names:
        codes, scales = cache.codes[name].cpu().double(), cache.scales[name].cpu().double()
        values = (codes[:, target] * scales[target].permute(1, 0, 2)[:, :, None, :, None]).to(dtype)
        assert torch.equal(back[name][:, source].cpu().nan_to_num(99), values.nan_to_num(99))
        assert (back[name][:, [b for b in range(blocks16) if b not in source]] == 5).all()


def test_convert_nothing_and_one_layer_of_many():
    from kvsnap_b200.cache8 import PagedCache8
    cache = PagedCache8.allocate(["a", "b"], 2, 16, 1, 64)
    wide = torch.randn((2, 3, 16, 1, 64), device="cuda").to(torch.bfloat16)
    converter = cache.converter({"b": wide})
    converter.compress([], [])
    assert not cache.codes["b"].view(torch.uint8).any()
    converter.compress([2], [1])
    cache.check()
    assert cache.codes["b"].view(torch.uint8)[:, 1].any() and not cache.codes["a"].view(torch.uint8).any()


# ---- streams, graphs, status ------------------------------------------------------------------


def step(p, dtype=torch.bfloat16, group=2):
    from kvsnap_b200.cache8 import rotary_table
    rotary = rotary_table(max(p.lengths) + 1, p.dim)
    k, v, q = (p.random(h, dtype, s)[1] for h, s in ((p.heads, 21), (p.heads, 22), (p.heads * group, 23)))

    def run():
        return p.cache.attend("l", p.cache.append("l", k, v, p.batch, query=q, rotary=rotary), p.batch)
    return run


@pytest.mark.parametrize("sequences", [[(1, 700), (1, 20)], [(50, 700), (3, 20)], [(4800, 40), (20, 5)]], ids=str)
def test_a_captured_step_replays_on_new_contents(sequences):
    p = Paged(sequences)
    run = step(p)
    before = (p.codes_gpu.clone(), p.scales_gpu.clone())
    expected = run().clone()
    again = run()
    assert torch.equal(again, expected)                     # the same bits every time
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        p.codes_gpu.copy_(before[0]), p.scales_gpu.copy_(before[1])
        out.fill_(9)
        graph.replay()
        assert torch.equal(out, expected)
    # Shorter sequences under the same graph: lengths are read on the GPU.
    shorter = [max(n - 17, 0) for n in p.lengths]
    p.batch.lengths.copy_(torch.tensor(shorter, dtype=torch.int32))
    p.codes_gpu.copy_(before[0]), p.scales_gpu.copy_(before[1])
    graph.replay()
    replayed = out.clone()
    p.codes_gpu.copy_(before[0]), p.scales_gpu.copy_(before[1])
    assert torch.equal(run(), replayed)
    p.cache.check()


def test_two_graphs_and_two_streams_do_not_share_workspaces():
    """Two captured attentions, replayed at once on two streams many times, keep their results."""
    runs, graphs, outs, expected = [], [], [], []
    for seed in (1, 2):
        p = Paged([(1, 5000), (1, 900 * seed), (20, 2000)], seed=seed, heads=2)
        q = p.random(8, torch.bfloat16, 30 + seed)[1]
        expected.append(p.cache.attend("l", q, p.batch).clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(p.cache.attend("l", q, p.batch))
        graphs.append(graph)
        runs.append((p, q))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        for (p, q), stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                p.cache.attend("l", q, p.batch)
    torch.cuda.synchronize()
    for out, want in zip(outs, expected):
        assert torch.equal(out, want)


def test_calls_run_on_the_current_stream():
    """Inputs made on a side stream behind a long queue of work, used there without a wait: order is the stream's."""
    p = Paged([(1, 300), (20, 77)])
    before = (p.codes_gpu.clone(), p.scales_gpu.clone())
    run = step(p)
    expected = run().clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    p.codes_gpu.zero_(), p.scales_gpu.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn((4096, 4096), device="cuda")
        for _ in range(20):
            x = x @ x * 1e-3
        p.codes_gpu.copy_(before[0]), p.scales_gpu.copy_(before[1])
        got = run()
    side.synchronize()
    assert torch.equal(got, expected)
    p.cache.check()


def test_check_waits_for_calls_on_other_streams():
    p = Paged([(1, 40), (1, 70)], heads=2)
    p.batch.table[1, 2] = -1
    q = p.random(4, torch.bfloat16)[1]
    x = torch.randn((8192, 8192), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):                                 # tens of milliseconds ahead of the call
            x @ x
        p.cache.attend("l", q, p.batch)
    with pytest.raises(ValueError, match="block id"):
        p.cache.check()


def test_the_first_call_of_a_process_may_be_captured():
    """No kernel of the cache has run in the process: a capture of the first step replays right."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
import test_gpu_cache8 as t
p = t.Paged([(1, 700), (40, 50)], heads=2)
before = (p.codes_gpu.clone(), p.scales_gpu.clone())
run = t.step(p)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
first = out.clone()
p.codes_gpu.copy_(before[0]), p.scales_gpu.copy_(before[1])
assert torch.equal(run(), first) and first.isfinite().all() and first.any()
p.cache.check()
print("captured first")
"""
    here = Path(__file__).resolve().parent
    got = subprocess.run([sys.executable, "-c", code], cwd=here, env={**__import__("os").environ, "PYTHONPATH": f"{here}:{here.parent}"},
                         capture_output=True, text=True, timeout=300)
    assert "captured first" in got.stdout, got.stderr[-2000:]


def test_a_bad_block_is_skipped_and_reported():
    """A block id outside the cache: recorded, its tokens left out, everything else as without it."""
    p = Paged([(1, 40), (1, 70), (3, 33)], heads=2)
    p.batch.table[1, 2] = p.scales_gpu.shape[0]
    q = p.random(4, torch.bfloat16)[1]
    got = p.cache.attend("l", q, p.batch)
    with pytest.raises(ValueError, match="block id"):
        p.cache.check()
    p.cache.check()                                         # reported once
    expected, bound = attend(q.cpu(), p.codes(), p.scales(), p.table, p.start, p.lengths, 16, p.dim ** -0.5)
    for row in (0, 2, 3, 4):
        assert ((got[row].cpu().double() - expected[row]).abs() <= bound[row]).all()
    assert got.isfinite().all()
    before = p.codes()
    p.batch.table[1, 4] = -1                                # position 70 lies in page 4
    k = p.random(2, torch.bfloat16, 3)[1]
    p.cache.append("l", k, k, p.batch)
    with pytest.raises(ValueError, match="block id"):
        p.cache.check()
    changed = {b for b in range(before.shape[1]) if not torch.equal(before[:, b], p.codes()[:, b])}
    assert changed <= {p.table[0][2], p.table[2][2]}


@pytest.mark.parametrize("what", ["length", "rows", "bound"])
def test_a_batch_that_does_not_fit_is_skipped_and_reported(what):
    p = Paged([(1, 40), (1, 70)], heads=2)
    if what == "length":
        p.batch.lengths[1] = 16 * p.batch.table.shape[1] + 1
    elif what == "rows":
        p.batch.start[2] = 9
    else:
        p = Paged([(1, 40), (2, 70)], heads=2, max_query=1)
    before = p.codes()
    q, k = p.random(4, torch.bfloat16)[1], p.random(2, torch.bfloat16, 3)[1]
    p.cache.attend("l", q, p.batch)
    with pytest.raises(ValueError, match="length"):
        p.cache.check()
    p.cache.append("l", k, k, p.batch)
    with pytest.raises(ValueError, match="length"):
        p.cache.check()
    after = p.codes()
    assert all(torch.equal(before[:, b], after[:, b]) for b in p.table[1][:5])


def test_a_position_behind_the_rotary_table_is_reported():
    from kvsnap_b200.cache8 import rotary_table
    p = Paged([(3, 40)], heads=1)
    k = p.random(1, torch.bfloat16, 3)[1]
    p.cache.append("l", k, k, p.batch, rotary=rotary_table(42, 128))
    with pytest.raises(ValueError, match="rotary"):
        p.cache.check()


def test_no_rows_and_no_sequences():
    from kvsnap_b200.cache8 import PagedBatch, PagedCache8
    cache = PagedCache8.allocate(["l"], 4, 16, 2, 64)
    none = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    batch = PagedBatch(none, torch.zeros(1, dtype=torch.int32, device="cuda"),
                       torch.zeros(0, dtype=torch.int32, device="cuda"))
    for rows in (0, 3):
        q = torch.zeros((rows, 4, 64), dtype=torch.bfloat16, device="cuda")
        k = torch.zeros((rows, 2, 64), dtype=torch.bfloat16, device="cuda")
        assert cache.attend("l", q, batch).shape == q.shape
        cache.append("l", k, k, batch)
    cache.check()


# ---- a session's way: filled, saved, restored elsewhere, read on -----------------------------------


@pytest.mark.parametrize("heads,staging", [(8, 512 << 20), (1, 512 << 20), (2, 1 << 20)])
def test_a_session_is_saved_and_restored_in_8_bits(heads, staging):
    """Prompt, save to pinned memory (codes, scales, checksums), restore into other blocks, next turn, step.

    The packed blocks are the cache's own bytes with the last block's free slots zeroed; what is attended to
    after the restore is bit for bit what it was before.
    """
    import hashlib

    from kvsnap_b200.cache8 import PagedBatch, PagedCache8, rotary_table
    from kvsnap_b200.dataplane import TorchBlockDataPlane
    from oracle import oracle
    names, dim, group, length = [f"layers.{i}" for i in range(3)], 128, 4, 403
    count = -(-length // 16)
    cache = PagedCache8.allocate(names, 120, 16, heads, dim)
    for name in names:                                       # what earlier sessions left
        cache.codes[name].view(torch.uint8).random_(0, 0x7E)
        cache.scales[name].fill_(2.0 ** -3)
    gen = torch.Generator().manual_seed(heads)
    order = torch.randperm(120, generator=gen).tolist()
    saved, restored, more = order[:count], order[count:2 * count], order[2 * count:2 * count + 3]
    rotary = rotary_table(1024, dim, 1e6)

    def batch(blocks, new, total):
        return PagedBatch(torch.tensor([blocks], dtype=torch.int32).cuda(), torch.tensor([0, new], dtype=torch.int32).cuda(),
                          torch.tensor([total], dtype=torch.int32).cuda(), max_query=new)

    def turn(blocks, new, total, seed):
        g = torch.Generator().manual_seed(seed)
        outs = []
        for name in names:
            q, k, v = (torch.randn((new, h, dim), generator=g).to(torch.bfloat16).cuda() for h in (heads * group, heads, heads))
            b = batch(blocks, new, total)
            outs.append(cache.attend(name, cache.append(name, k, v, b, query=q, rotary=rotary), b))
        return outs

    turn(saved, length, length, 1)
    cache.check()
    before = {name: (cache.codes[name].view(torch.uint8).cpu(), cache.scales[name].cpu()) for name in names}
    plane = TorchBlockDataPlane(cache.codes, 16, 64 << 20, scales=cache.scales, staging_bytes=staging)
    try:
        plane.warm_up()
        size = plane.block_bytes
        assert size == 3 * (2 * 16 * heads * dim + 8 * heads)
        pinned = plane.pool.reserve(size * count)
        targets = [(pinned, i * size) for i in range(count)]
        digests = []
        plane.save_gather(saved, targets, length, digests=digests)
        packed = [pinned.read_range(i * size, size) for i in range(count)]
        for i, block in enumerate(saved):
            expected = b""
            for name in names:
                codes, scales = before[name]
                sides = codes[:, block].clone()
                if i == count - 1:
                    sides[:, length % 16:] = 0
                expected += sides[0].numpy().tobytes() + scales[block].numpy().tobytes() + sides[1].numpy().tobytes()
            assert packed[i] == expected
            assert digests[i] == (hashlib.sha256(expected).hexdigest(), oracle.crc32c(expected))
        expected = turn(saved + more[:1], 9, length + 9, 2) + turn(saved + more[:1], 1, length + 10, 3)
        plane.load_scatter(restored, targets, expected_crc32c=[c for _, c in digests])
        again = turn(restored + more[1:2], 9, length + 9, 2) + turn(restored + more[1:2], 1, length + 10, 3)
        for a, b in zip(again, expected):
            assert torch.equal(a, b)
        cache.check()
        pinned.close()
    finally:
        plane.close()


def test_a_16_bit_session_goes_on_in_8_bits():
    """Blocks of a 16-bit cache compressed, attended to and expanded: what is read is what the codes stand for."""
    from kvsnap_b200.cache8 import PagedBatch, PagedCache8
    names, heads, dim, length = ["a", "b"], 2, 64, 70
    wide = {name: torch.randn((2, 9, 16, heads, dim), device="cuda").to(torch.float16) for name in names}
    cache = PagedCache8.allocate(names, 9, 16, heads, dim)
    converter = cache.converter(wide)
    source, blocks = [8, 0, 3, 5, 1], [2, 7, 4, 0, 6]
    converter.compress(source, blocks, length)
    batch = PagedBatch(torch.tensor([blocks], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(),
                       torch.tensor([length], dtype=torch.int32).cuda(), max_query=1)
    q = torch.randn((1, 4, dim), device="cuda").to(torch.float16)
    for name in names:
        got = cache.attend(name, q, batch).cpu().double()
        expected, bound = attend(q.cpu(), cache.codes[name].view(torch.uint8).cpu(), cache.scales[name].cpu(), [blocks],
                                 [0, 1], [length], 16, dim ** -0.5)
        assert ((got - expected).abs() <= bound).all()
    back = {name: torch.zeros_like(t) for name, t in wide.items()}
    cache.converter(back).expand(blocks, source)
    cache.check()
    for name in names:
        values = wide[name][:, source].cpu().double().flatten(1, 2)[:, :length]
        off = (back[name][:, source].cpu().double().flatten(1, 2)[:, :length] - values).abs()
        # half a step of the format, or of its smallest numbers at the block's scale (amax < 8: 2^-5)
        assert (off <= torch.maximum(2.0 ** -4 * values.abs(), torch.full_like(values, 2.0 ** -15))).all()
        assert (back[name][:, source].cpu().flatten(1, 2)[:, length:] == 0).all()
