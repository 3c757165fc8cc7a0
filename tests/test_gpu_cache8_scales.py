"""The 8-bit cache's attention over pages whose scales lie far apart, on a B200 against 64 bits.

A page of values far larger than its neighbours, which carries little or no weight, must leave the rest as it
is; and rows must not depend on the scales of tokens behind them.
"""
import pytest
import torch

from cache8_reference import E4M3, HALF, rows_of
from test_gpu_cache8 import Paged

pytestmark = pytest.mark.gpu


def attend_by_pages(q, p, scale):
    """(out, bound) float64 [rows, q_heads, dim], as cache8_reference.attend, with a bound that counts pages' scales.

    A token's weight in the values' sum is its softmax weight times its page's scale, w_j s_j. It reaches 16 bits
    once: half a step of fp16, 2^-11, and where it is below fp16's normal numbers 2^-25 of a unit that is at
    most twice the largest w_j s_j of the row's tokens (the unit is a power of two, rounded up). Chunks
    hold codes of 64 tokens relative to their largest page, up to 2^6 above a token's own, so 2^6 times that.
    """
    q_heads, dim = q.shape[1:]
    group = q_heads // p.heads
    codes, scales = p.codes().view(E4M3).double(), p.scales().double()
    out = torch.zeros(p.rows, q_heads, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for s, row, position in rows_of(p.start, p.lengths):
        if position < 0:
            continue
        pages = torch.tensor(p.table[s][: -(-p.lengths[s] // p.block_size)])
        held = codes[:, pages].flatten(1, 2)[:, : position + 1].repeat_interleave(group, dim=2)      # [2, tokens, q_heads, dim]
        by = scales[pages].permute(1, 0, 2).repeat_interleave(p.block_size, dim=1)[:, : position + 1]
        by = by.repeat_interleave(group, dim=2)                                                       # [2, tokens, q_heads]
        key, value = held * by[..., None]
        score = torch.einsum("hd,thd->ht", q[row].double(), key) * scale
        size = torch.einsum("hd,thd->ht", q[row].double().abs(), key.abs()).amax(dim=1) * scale
        weight = torch.softmax(score, dim=-1)
        out[row] = torch.einsum("ht,thd->hd", weight, value)
        spread = torch.einsum("ht,thd->hd", weight, value.abs())
        relative = 2.0 ** -11 + 2 * (dim + 4) * 2.0 ** -24 * size + (position + 65) * 2.0 ** -24 + 2.0 ** -20
        reach = 2.0 ** 6 if (p.start[s + 1] - p.start[s]) * group > 16 else 1.0
        unit = 2 * (weight * by[1].T).amax(dim=1)
        bound[row] = relative[:, None] * spread + (2.0 ** -25 * reach * unit)[:, None] * held[1].abs().sum(dim=0)
    half = HALF[q.dtype]
    return out, bound * (1 + half) + half * out.abs()


def check(p, q, q_gpu, scale):
    got = p.cache.attend("l", q_gpu, p.batch, scale=scale).cpu().double()
    p.cache.check()
    expected, bound = attend_by_pages(q, p, scale)
    owned = [row for _, row, _ in rows_of(p.start, p.lengths)]
    assert torch.isfinite(got[owned]).all()
    over = ((got - expected).abs() / bound)[owned]
    assert (over <= 1).all(), f"worst {over.max().item():.3g} of its bound"


SHAPES = [(128, 16, 2, 4), (64, 32, 3, 2)]            # head_dim, block_size, kv_heads, group


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", [[(1, 530)], [(1, 900), (1, 85), (2, 300)], [(45, 530)], [(150, 20), (30, 700)]],
                         ids=str)
@pytest.mark.parametrize("place", ["first", "some"])
@pytest.mark.parametrize("above,below", [(16, 87), (30, 87), (30, 30), (100, 110), (7, 9), (64, 1), (100, 9)])
def test_a_large_page_of_little_weight(shape, sequences, place, above, below):
    """Pages 2^above larger than the others whose tokens weigh about 2^-below of them.

    Where they make up the result, the others still count in the softmax.
    """
    dim, block_size, heads, group = shape
    p = Paged(sequences, dim=dim, block_size=block_size, heads=heads, seed=7)
    codes, scales = p.codes(), torch.full_like(p.scales(), 2.0 ** (-60 if above > 60 else -9))
    scales[:, 0] = 2.0 ** -6
    large = [b for row, length in zip(p.table, p.lengths) for i, b in enumerate(row[: -(-length // block_size)])
             if (i == 0 if place == "first" else i % 5 == 2)]
    scales[large, 1] *= 2.0 ** above
    # Dimension 0 alone tells large pages from others: q_0 k_0 scale = -below ln 2 there, and 0 elsewhere.
    codes[0, ..., 0] = 0
    codes[0][large, ..., 0] = torch.tensor([-448.0]).to(E4M3).view(torch.uint8)
    p.codes_gpu.copy_(codes), p.scales_gpu.copy_(scales)
    scale = 0.05
    q, q_gpu = p.random(heads * group, torch.bfloat16, 3)
    q[..., 0] = below * 0.6931 / (7 * scale)
    q_gpu.copy_(q)
    check(p, q, q_gpu, scale)


@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("above", [8, 16, 30, 70])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", [[(5, 3), (6, 40)], [(45, 530), (20, 50)], [(400, 0)]], ids=str)
def test_rows_do_not_depend_on_the_scales_of_later_tokens(side, above, shape, sequences):
    """The last page of a sequence, 2^above larger in keys or values: rows before it keep their bits' worth."""
    dim, block_size, heads, group = shape
    p = Paged(sequences, dim=dim, block_size=block_size, heads=heads, seed=8)
    scales = torch.full_like(p.scales(), 2.0 ** -8)
    for s, length in enumerate(p.lengths):
        scales[p.table[s][(length - 1) // block_size], side] *= 2.0 ** above
    p.scales_gpu.copy_(scales)
    q, q_gpu = p.random(heads * group, torch.bfloat16, 4)
    check(p, q, q_gpu, dim ** -0.5)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", [[(1, 530)], [(45, 530)], [(130, 0), (3, 64)]], ids=str)
def test_pages_of_zeros_among_small_and_large_ones(shape, sequences):
    """Values of zero count in the softmax and in nothing else, whatever the pages around them hold."""
    dim, block_size, heads, group = shape
    p = Paged(sequences, dim=dim, block_size=block_size, heads=heads, seed=9)
    powers = torch.tensor([2.0 ** -100, 0.0, 0.0, 0.0, 0.0, 0.0, 2.0 ** -97, 2.0 ** -60, 0.0])
    scales = p.scales()
    for row, length in zip(p.table, p.lengths):
        for i, b in enumerate(row[: -(-length // block_size)]):
            scales[b, 1] = powers[i % 9]
    p.scales_gpu.copy_(scales)
    q, q_gpu = p.random(heads * group, torch.bfloat16, 5)
    check(p, q, q_gpu, dim ** -0.5)


@pytest.mark.parametrize("sequences", [[(1, 530)], [(45, 530)]], ids=str)
def test_values_all_zero(sequences):
    p = Paged(sequences, seed=10)
    p.scales_gpu[:, 1] = 0
    got = p.cache.attend("l", p.random(8, torch.float16)[1], p.batch)
    p.cache.check()
    assert (got[: p.start[-1]] == 0).all()


@pytest.mark.parametrize("sequences", [[(1, 530), (1, 40)], [(45, 530), (17, 9)]], ids=str)
def test_scales_that_are_no_powers_of_two(sequences):
    """A cache that others filled: any positive scale counts as it is (chunks hold its fraction in 16 bits)."""
    p = Paged(sequences, seed=11)
    gen = torch.Generator().manual_seed(1)
    p.scales_gpu.copy_(torch.rand(p.scales_gpu.shape, generator=gen) * 0.01 + 0.001)
    q, q_gpu = p.random(8, torch.bfloat16, 6)
    got = p.cache.attend("l", q_gpu, p.batch).cpu().double()
    p.cache.check()
    expected, bound = attend_by_pages(q, p, p.dim ** -0.5)
    # chunks: code * fraction rounds to fp16, 2^-11 more of values, and of keys in the products' sums
    for s, row, position in rows_of(p.start, p.lengths):
        more = torch.zeros(())
        if (p.start[s + 1] - p.start[s]) * 4 > 16:
            pages = torch.tensor(p.table[s][: -(-p.lengths[s] // 16)])
            by = p.scales()[pages].double().permute(1, 0, 2).repeat_interleave(16, dim=1)[:, : position + 1]
            held = (p.codes().view(E4M3)[:, pages].double().flatten(1, 2)[:, : position + 1] * by[..., None]).repeat_interleave(4, dim=2)
            size = torch.einsum("hd,thd->ht", q[row].double().abs(), held[0].abs()) * p.dim ** -0.5
            score = torch.einsum("hd,thd->ht", q[row].double(), held[0]) * p.dim ** -0.5
            weight = torch.softmax(score, dim=-1)
            spread = torch.einsum("ht,thd->hd", weight, held[1].abs())
            # a key's rounding moves each score by at most 2^-11 of its products' size, numerator and sum alike
            more = (2.0 ** -11 + 2 * (torch.expm1(2.0 ** -11 * size.amax(dim=1)))[:, None]) * spread
        assert ((got[row] - expected[row]).abs() <= bound[row] + more).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("sequences", [[(1, 530)], [(3, 200), (1, 40)], [(45, 530)], [(300, 0), (70, 90)]], ids=str)
@pytest.mark.parametrize("size", [2.0 ** 24, 2.0 ** 27, 2.0 ** 40, 2.0 ** 90])
def test_scores_so_large_that_one_token_takes_all(shape, sequences, size):
    """Scores of `size` and its quarters: a row is the value of the one largest that it sees, exactly.

    Scores beyond 2^24 lie further apart than weights reach; what bounds them is 32 bits.
    """
    dim, block_size, heads, group = shape
    p = Paged(sequences, dim=dim, block_size=block_size, heads=heads, seed=12)
    codes, scales = p.codes(), p.scales()
    scales[:, 0] = 1.0
    first = torch.zeros(codes.shape[1], block_size, heads)
    late = 20                                              # the largest from here on; token 0 before it
    for row, length in zip(p.table, p.lengths):
        for i, b in enumerate(row[: -(-length // block_size)]):
            first[b] = -448.0
        first[row[0], 0] = 112.0
        if length > late:
            first[row[late // block_size], late % block_size] = 448.0
    codes[0] = 0
    codes[0][..., 0] = first.to(E4M3).view(torch.uint8)
    p.codes_gpu.copy_(codes), p.scales_gpu.copy_(scales)
    q, q_gpu = p.random(heads * group, torch.bfloat16, 7)
    q[..., 0] = 1.5
    q_gpu.copy_(q)
    got = p.cache.attend("l", q_gpu, p.batch, scale=size / 672).cpu()
    p.cache.check()
    for s, row, position in rows_of(p.start, p.lengths):
        at = late if position >= late else 0
        block = p.table[s][at // block_size]
        value = codes[1, block, at % block_size].view(E4M3).float() * scales[block, 1][:, None]
        assert torch.equal(got[row].float(), value.repeat_interleave(group, dim=0))
