"""Attention over the paged cache where the precision of its parts shows: the
weights' own bits, values far smaller than their neighbours, values as large as
bf16 holds, and rows that a query does not see.  All kernels alike, whatever else
is in the batch."""
import pytest
import torch

import bmx
from _paged_check import D, U8, attention_reference, normal
from test_gpu_paged import case, check

pytestmark = pytest.mark.gpu

# A kernel each: single tokens, up to 32 and up to 64 query rows per kv head,
# tiles of 128 and of 256 rows; a chunk beside single tokens; shared rows before
# single tokens, before drafts and before prompts
BATCHES = [
    ((8, 2), [1, 1, 1, 1], [0, 3, 11, 40], 0), ((8, 2), [6, 1, 3], [0, 5, 9], 0), ((8, 2), [14, 1, 9], [0, 5, 9], 0),
    ((8, 2), [48, 20], [0, 3], 0), ((64, 1), [200], [0], 0), ((8, 2), [40, 1, 1, 1], [0, 2, 5, 12], 0),
    ((8, 2), [1] * 8, [0, 1, 2, 3, 5, 7, 9, 20], 16), ((8, 2), [6, 1], [0, 4], 16), ((8, 2), [14, 1], [0, 4], 16),
    ((8, 2), [40, 1], [0, 4], 16),
]


@pytest.mark.parametrize("heads,new,past,shared", BATCHES)
@pytest.mark.parametrize("scale", [0.25, -0.6, 1.0])
def test_weights_have_16_bits(gpu, heads, new, past, shared, scale):
    """Scores of one dimension are exact before the scale; values are positive, so
    that nothing cancels.  A weight is then off by the two roundings of its score
    in base 2 (below 2^5: 2^-18 together), the exponential's (2^-22) and its two bf16
    pieces (U8 each: 2^-16); the fp32 sums of L terms and the parts' joining by at
    most 2^-23 a term and as much for 32 more steps; scores and sums together below
    (L + 64) 2^-23.  An output is that, then rounded to bf16 by at most half a
    step of its binade.  With weights of 11 bits a few outputs in a hundred lie
    outside."""
    q, cache, batch, lens, lists = case(21, heads, 16, new, [p + shared for p in past], common=shared // 16)
    q[..., 1:] = 0
    q[..., 0] = q[..., 0].clamp(-4, 4)
    cache.k[..., 1:] = 0
    cache.k[..., 0] = cache.k[..., 0].clamp(-4, 4)
    cache.v.copy_(0.5 + cache.v.float().abs().clamp(max=1.5))
    got = bmx.attention_paged(q, cache, batch, scale=scale, shared=shared).double().view(sum(new), heads[0], D)
    want, _ = attention_reference(q, cache.k, cache.v, new, lens, lists, scale, shared, half=False)
    rel = U8 * U8 + (max(lens) + 64) * 2.0 ** -23
    step = torch.exp2(torch.floor(torch.log2(want * (1 + rel))) - 7)
    off = (got - want).abs() - step / 2 - rel * want
    assert not (off > 0).any(), f"{int((off > 0).sum())} of {off.numel()} off, worst by {float((off / want).max()):.3g}"


@pytest.mark.parametrize("heads,new,past,shared", BATCHES)
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -28, 2.0 ** -34, 2.0 ** -100])
def test_small_values_beside_others(gpu, heads, new, past, shared, size):
    """A dimension far smaller than those around it, one that holds a single value,
    and single small values: as precise as any other."""
    q, cache, batch, lens, lists = case(22, heads, 16, new, [p + shared for p in past], common=shared // 16)
    cache.v[..., 9] *= size
    cache.v[..., 26] = 1.9921875 * size
    cache.v[:, :, 3::4, 41] *= size
    got = check(q, cache, batch, new, lens, lists, shared=shared, half=False).view(-1, D)
    # the mean of equal values: their one rounding, and that of the weights' sum (2^-16)
    assert ((got[:, 26].double() / (1.9921875 * size) - 1).abs() <= U8 + 2.0 ** -15).all()


LARGE = [  # (heads, new tokens, their sequences' other rows, shared rows)
    ((8, 2), [1, 1, 1], [300, 9000, 70000], 0), ((8, 2), [6, 1], [9000, 3], 0), ((8, 2), [14, 1], [9000, 3], 0),
    ((8, 2), [40, 1], [9000, 3], 0), ((64, 1), [200], [3000], 0), ((8, 2), [1] * 3, [30, 4000, 0], 8000), ((8, 2), [40, 1], [4, 4000], 8000),
]


@pytest.mark.parametrize("heads,new,past,shared", LARGE)
def test_values_of_2_to_the_120_over_many_rows(gpu, heads, new, past, shared):
    """A mean of large values is no larger than they are: their weighted sum must
    not leave fp32 before it is divided."""
    q, cache, batch, lens, lists = case(24, heads, 16, new, [p + shared for p in past], common=shared // 16, std=0.0)
    cache.v.copy_((1 + 0.9 * normal(25, *cache.v.shape).abs().clamp(max=1)) * 2.0 ** 120)
    check(q, cache, batch, new, lens, lists, shared=shared, half=False)  # every key alike
    q.copy_(normal(26, *q.shape).to(torch.bfloat16))
    check(q, cache, batch, new, lens, lists, shared=shared, half=False)


@pytest.mark.parametrize("heads,new,past,shared", BATCHES)
def test_values_next_to_the_largest(gpu, heads, new, past, shared):
    q, cache, batch, lens, lists = case(26, heads, 16, new, [p + shared for p in past], common=shared // 16)
    cache.v.copy_((1 + 0.9 * normal(27, *cache.v.shape).abs().clamp(max=1)) * 2.0 ** 126 * normal(28, *cache.v.shape).sign())
    check(q, cache, batch, new, lens, lists, shared=shared, half=False)
    # keys whose scores rise slowly, so that the maximum lags behind them
    q[..., 1:] = 0
    q[..., 0] = 1
    cache.k[..., 1:] = 0
    for pages in lists:
        for j, pg in enumerate(pages):
            cache.k[pg, :, :, 0] = (16 * j + torch.arange(16, device="cuda", dtype=torch.float32)) / 8
    cache.v.abs_()
    check(q, cache, batch, new, lens, lists, shared=shared, scale=1.0, half=False)


@pytest.mark.parametrize("heads,new", [((8, 2), [4, 2]), ((16, 2), [4, 2]), ((32, 2), [4, 2]), ((8, 2), [100, 40]), ((6, 2), [257, 33]),
                                       ((64, 1), [200, 190])])
@pytest.mark.parametrize("value", [2.0 ** 20, -2.0 ** 127, 2.0 ** -40])
def test_hidden_values_change_no_bit(gpu, heads, new, value):
    """A finite value of a later token's row, of whatever size, leaves the tokens
    before it as they were, bit by bit."""
    hkv = heads[1]
    q, cache, batch, lens, lists = case(23, heads, 16, new, [30, 61])
    want = check(q, cache, batch, new, lens, lists, half=False)
    at = lens[0] - new[0] // 2
    pg, r = lists[0][at // 16], at % 16
    cache.v[pg, 0, r] = value
    got = check(q, cache, batch, new, lens, lists, half=False)
    first = new[0] - new[0] // 2
    g, w = (x.view(sum(new), hkv, -1) for x in (got, want))
    assert torch.equal(g[:first], w[:first]) and torch.equal(g[new[0]:], w[new[0]:]) and torch.equal(g[:, 1:], w[:, 1:])


@pytest.mark.parametrize("heads,new", [((8, 2), [4, 2]), ((16, 2), [4, 2]), ((32, 2), [4, 2]), ((8, 2), [100, 40]), ((6, 2), [257, 33]),
                                       ((64, 1), [200, 190])])
@pytest.mark.parametrize("size", [3.0, 50.0])
def test_hidden_keys_change_no_bit(gpu, heads, new, size):
    """So does a key of a later token's row that scores far above all others: the
    rows of a wave keep their maxima by themselves."""
    hkv = heads[1]
    q, cache, batch, lens, lists = case(29, heads, 16, new, [30, 61])
    want = check(q, cache, batch, new, lens, lists, half=False)
    first = new[0] - new[0] // 2
    at = lens[0] - new[0] // 2  # a row that the later half of the first sequence's tokens see
    pg, r = lists[0][at // 16], at % 16
    cache.k[pg, 0, r] = (size * q[0, first].float()).to(torch.bfloat16)  # (as one of these asks)
    got = check(q, cache, batch, new, lens, lists, half=False)
    g, w = (x.view(sum(new), hkv, -1) for x in (got, want))
    assert torch.equal(g[:first], w[:first]) and torch.equal(g[new[0]:], w[new[0]:]) and torch.equal(g[:, 1:], w[:, 1:])


@pytest.mark.parametrize("heads,new,past,shared", BATCHES)
def test_other_queries_change_no_bit(gpu, heads, new, past, shared):
    """Nor does a query that scores far higher than the others."""
    q, cache, batch, lens, lists = case(30, heads, 16, new, [p + shared for p in past], common=shared // 16)
    want = check(q, cache, batch, new, lens, lists, shared=shared, half=False).view(sum(new), heads[0], D)
    q[0, 0] = cache.k[lists[0][0], 0, 0] * 4
    got = check(q, cache, batch, new, lens, lists, shared=shared, half=False).view(sum(new), heads[0], D)
    assert torch.equal(got[1:], want[1:]) and torch.equal(got[0, 1:], want[0, 1:])
