"""Calls of the 8-bit cache at the edges of what it takes, on a B200: bounds of no rows, launches that cannot be,
batches and positions that do not fit, and the sizes at which its kernels change their way.
"""
import pytest
import torch

from cache8_reference import attend
from test_gpu_cache8 import Paged, check_append, check_attend

pytestmark = pytest.mark.gpu


def expand_one(cache):
    """A conversion of one block: any later call of the thread."""
    codes = cache.codes["l"]
    wide = torch.zeros((2, 1, *codes.shape[2:]), dtype=torch.bfloat16, device="cuda")
    cache.converter({"l": wide}).expand([0], [0])
    torch.cuda.synchronize()


def wide_table(p, width):
    """The batch of `p` over a table of `width` pages a sequence."""
    from kvsnap_b200.cache8 import PagedBatch
    held = p.batch.table
    table = torch.zeros((held.shape[0], width), dtype=torch.int32, device="cuda")
    table[:, : held.shape[1]] = held
    return PagedBatch(table, p.batch.start, p.batch.lengths, max_query=p.batch.max_query)


@pytest.mark.parametrize("group", [1, 4, 24])
@pytest.mark.parametrize("width", [5, 96, 4000])
@pytest.mark.parametrize("seqs", [1, 7])
def test_a_bound_of_no_rows(seqs, width, group):
    """A padded step in which no sequence has rows, on both sides of the rule that cuts a step: nothing is written."""
    p = Paged([(0, 37)] * seqs, heads=8, dim=64, pad_rows=5, max_query=0)
    p.batch = wide_table(p, width)
    before = p.codes(), p.scales()
    out = torch.full((5, 8 * group, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q, k = p.random(8 * group, torch.bfloat16)[1], p.random(8, torch.bfloat16)[1]
    p.cache.append("l", k, k, p.batch)
    p.cache.attend("l", q, p.batch, out=out)
    expand_one(p.cache)
    p.cache.check()
    assert (out == 7).all() and torch.equal(p.codes(), before[0]) and torch.equal(p.scales(), before[1])


def test_a_launch_that_cannot_be_leaves_later_calls_alone():
    """More query heads than a grid holds: the call fails, and the calls after it do not."""
    from kvsnap_b200.cache8 import rotary_table
    p = Paged([(1, 3)], heads=2, dim=64)
    k = p.random(2, torch.bfloat16)[1]
    q = torch.zeros((1, 8 * 65536, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        p.cache.append("l", k, k, p.batch, query=q, rotary=rotary_table(8, 64))
    expand_one(p.cache)
    p.cache.check()


@pytest.mark.parametrize("group", [1, 24])
def test_rows_beyond_a_bound_of_none_are_reported(group):
    p = Paged([(0, 37), (2, 20)], heads=2, dim=64, max_query=0)
    out = torch.full((2, 2 * group, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    p.cache.attend("l", p.random(2 * group, torch.bfloat16)[1], p.batch, out=out)
    with pytest.raises(ValueError, match="length"):
        p.cache.check()
    assert (out == 7).all()


@pytest.mark.parametrize("sequences,bound", [([(5, 20), (9, 3), (1, 16)], 8), ([(1, 20), (0, 3)], 0), ([(2, 4)], 1)], ids=str)
def test_an_append_keeps_to_its_bound(sequences, bound):
    """A sequence of more rows than max_query is left out and reported; the others are appended."""
    p = Paged(sequences, heads=2, dim=64, max_query=bound)
    held, k = p.codes(), p.random(2, torch.bfloat16, 3)[1]
    p.cache.append("l", k, k, p.batch)
    with pytest.raises(ValueError, match="length"):
        p.cache.check()
    now = p.codes()
    for (new, _), row, length in zip(sequences, p.table, p.lengths):
        pages = row[: -(-length // p.block_size)]
        same = all(torch.equal(held[:, b], now[:, b]) for b in pages)
        assert same == (new > bound or new == 0)


@pytest.mark.parametrize("sequences,positions", [
    ([(3, 40)], 42), ([(3, 40)], 40), ([(3, 40)], 17), ([(40, 5), (1, 16), (9, 0)], 21), ([(1, 20), (1, 9), (1, 16)], 16),
    ([(20, 0), (2, 3)], 1)], ids=str)
def test_positions_behind_the_rotary_table_are_left_out(sequences, positions):
    """Their tokens are not written and set no scale; all others are as if the call ended before them."""
    from kvsnap_b200.cache8 import PagedBatch, rotary_table
    p, same = Paged(sequences, heads=2, dim=64, seed=4), Paged(sequences, heads=2, dim=64, seed=4)
    k, v = p.random(2, torch.bfloat16, 3)[1].clone(), p.random(2, torch.bfloat16, 5)[1].clone()
    q = p.random(4, torch.bfloat16, 6)[1]
    for s, length in enumerate(p.lengths):                 # what is left out is the largest
        behind = min(max(length - positions, 0), p.start[s + 1] - p.start[s])
        k[p.start[s + 1] - behind: p.start[s + 1]] *= 100
        v[p.start[s + 1] - behind: p.start[s + 1]] *= 100
    table = rotary_table(64, 64)
    got_q = p.cache.append("l", k, v, p.batch, query=q, rotary=table[:positions].contiguous())
    with pytest.raises(ValueError, match="rotary"):
        p.cache.check()
    # The same rows, sequence by sequence, up to the table's end.
    for s, length in enumerate(p.lengths):
        new = p.start[s + 1] - p.start[s]
        held = length - new
        kept = min(max(positions - held, 0), new)
        if not kept:
            continue
        rows = slice(p.start[s], p.start[s] + kept)
        one = PagedBatch(p.batch.table[s: s + 1], torch.tensor([0, kept], dtype=torch.int32).cuda(),
                         torch.tensor([held + kept], dtype=torch.int32).cuda())
        want_q = same.cache.append("l", k[rows], v[rows], one, query=q[rows], rotary=table)
        assert torch.equal(got_q[rows], want_q)
    same.cache.check()
    assert torch.equal(p.codes(), same.codes()) and torch.equal(p.scales(), same.scales())


# ---- sizes at which the kernels change their way --------------------------------------------------


def test_more_sequences_than_a_step_finds_in_one_pass():
    """More than 512 sequences whose work is cut: a CTA's share is sought a part of them at a time."""
    sequences = [(1, 250 + s * 37 % 350) for s in range(600)]
    check_attend(Paged(sequences, dim=64, heads=8, poison=True), torch.bfloat16, 2)


def test_more_sequences_than_a_chunk_call_scans_at_once():
    """More than 256 sequences of 1 or 20 new tokens: both kernels, and the second scan of the chunks' one."""
    sequences = [(20 if s % 3 == 0 else 1, s * 29 % 150) for s in range(300)]
    check_attend(Paged(sequences, dim=64, heads=2, poison=True), torch.float16, 2)


@pytest.mark.parametrize("heads,group", [(3, 2), (5, 1), (6, 2), (7, 2), (16, 2), (10, 1), (14, 1), (24, 1)])
def test_heads_that_do_not_fill_a_cta(heads, group):
    """Numbers of KV heads that share a CTA's 16 warps with some to spare, and several groups of heads."""
    sequences = [(1, s * 41 % 230) for s in range(60)]
    check_attend(Paged(sequences, dim=64, heads=heads, poison=True), torch.bfloat16, group)
    check_attend(Paged([(1 + s % 2, s * 41 % 1900) for s in range(30)], dim=64, heads=heads), torch.float16, group)


@pytest.mark.parametrize("group,rows", [(16, 1), (12, 1), (5, 3), (3, 5), (8, 2), (9, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_steps_of_9_to_16_rows_a_head(dim, group, rows):
    sequences = [(rows, 300 + s * 53 % 700) for s in range(9)]
    check_attend(Paged(sequences, dim=dim, heads=2, poison=True), torch.bfloat16, group)


@pytest.mark.parametrize("group", [17, 24, 40])
def test_groups_of_more_than_16_heads(group):
    check_attend(Paged([(1, 300), (2, 40), (0, 9), (1, 0)], dim=64, heads=2, poison=True), torch.bfloat16, group)


@pytest.mark.parametrize("sequences,width", [([(1, 128)], 2560), ([(1, 200 + s) for s in range(64)], 2560),
                                             ([(1, 300 + s % 400) for s in range(128)], 300)], ids=["one", "64", "128"])
def test_a_table_wider_than_its_sequences(sequences, width):
    """An engine's table is as wide as its longest sequence may be: the same results as over a trimmed one."""
    p = Paged(sequences, dim=64, heads=4)
    q, q_gpu = p.random(8, torch.bfloat16)
    got = p.cache.attend("l", q_gpu, wide_table(p, width)).cpu().double()
    p.cache.check()
    expected, bound = attend(q, p.codes(), p.scales(), p.table, p.start, p.lengths, p.block_size, p.dim ** -0.5)
    assert ((got - expected).abs() <= bound).all()


def test_an_append_over_many_sequences():
    check_append(Paged([(1 + s % 3, s * 31 % 90) for s in range(300)], dim=64, heads=2), torch.bfloat16, group=1, rotary_dim=64)


@pytest.mark.parametrize("sequences", [[(1, 90), (1, 33)], [(24, 90), (20, 7)]], ids=str)
def test_nan_queries_and_keys_reach_who_they_concern(sequences):
    """A NaN in a row's query is that row's and head's; one in a key is the rows' that see it, of its head."""
    p = Paged(sequences, heads=2, dim=64)
    q, q_gpu = p.random(8, torch.bfloat16)
    q[0, 5, 7] = float("nan")                              # KV head 1
    last = p.lengths[1] - 1                                # the last token of sequence 1
    p.codes_gpu[0, p.table[1][last // 16], last % 16, 0, 9] = 0x7F
    q_gpu.copy_(q)
    got = p.cache.attend("l", q_gpu, p.batch).cpu().double()
    p.cache.check()
    final = p.start[2] - 1
    assert got[0, 5].isnan().all() and got[final, :4].isnan().all()
    got[0, 5] = 0
    got[final, :4] = 0
    q[0, 5, 7] = 0
    expected, bound = attend(q, p.codes(), p.scales(), p.table, p.start, p.lengths, p.block_size, p.dim ** -0.5)
    expected[0, 5] = 0
    expected[final, :4] = 0
    bound = bound.nan_to_num(1.0)
    assert ((got - expected).abs() <= bound).all()


@pytest.mark.parametrize("sequences", [[(1, 700), (1, 20)], [(1, 40)] * 70, [(300, 200), (2, 90), (40, 0)]], ids=["cut", "whole", "chunks"])
def test_the_output_may_be_the_query(sequences):
    p = Paged(sequences, heads=2, dim=64)
    q = p.random(8, torch.bfloat16)[1].contiguous()
    expected = p.cache.attend("l", q, p.batch)
    assert p.cache.attend("l", q, p.batch, out=q) is q
    p.cache.check()
    assert torch.equal(q, expected)
