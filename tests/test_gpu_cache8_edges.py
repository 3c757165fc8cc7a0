"""Calls of the 8-bit cache at the edges of what it takes, on a B200: bounds of no rows, launches that cannot be,
batches and positions that do not fit, and the sizes at which its kernels change their way.
"""
import pytest
import torch

from test_gpu_cache8 import Paged

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
