"""Attention over the paged cache of batches with many packed rows: few of them
in use, and enough for tiles of 256 query rows."""
import math

import pytest
import torch

import bmx
from _paged_check import D, attention_reference, hold, layout, normal, rotated
from test_gpu_paged import cache_of

pytestmark = pytest.mark.gpu

PAGE = 16


def dirty(n_heads, n_kv_heads, batch, shared):
    """A workspace with its counters zero and the rest NaN."""
    ws = bmx.attention_paged_workspace(n_heads, n_kv_heads, batch, shared=shared)
    ws[bmx.PAGED_COUNTER_BYTES:].fill_(255)
    return ws


@pytest.mark.parametrize("n", [1, 6, 14])
@pytest.mark.parametrize("tokens,first", [(6144, 6100), (6144, 3071), (6144, 0), (6200, 5), (20000, 19900)])
def test_few_rows_of_many_behind_shared_ones(gpu, n, tokens, first):
    """Two sequences of n tokens somewhere among many packed rows."""
    hq, hkv, shared, new = 8, 2, 32, [n, n]
    lens = [shared + n + 9, shared + n + 40]
    lists, n_pages = layout(1, new, lens, PAGE, common=shared // PAGE)
    cache = cache_of(2, n_pages, hkv, PAGE)
    q = normal(3, hq, tokens, D).to(torch.bfloat16)
    one = bmx.PagedBatch.of(new, lens, lists)
    batch = bmx.PagedBatch(one.starts + first, one.lens, one.pages, tokens, max_new=n)
    out = torch.full((tokens, hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    bmx.attention_paged(q, cache, batch, shared=shared, workspace=dirty(hq, hkv, batch, shared), out=out)
    want, bound = attention_reference(q[:, first:first + 2 * n].contiguous(), cache.k, cache.v, new, lens, lists,
                                      1 / math.sqrt(D), shared, half=False)
    hold(out[first:first + 2 * n], want, bound)
    assert (out[:first] == 7).all() and (out[first + 2 * n:] == 7).all()


def test_a_long_sequence_before_a_short_one_behind_shared_rows(gpu):
    """Of a sequence with more than max_new new tokens the first max_new are
    answered, and those of the sequences behind it."""
    hq, hkv, shared, new = 8, 2, 32, [6100, 2]
    lens = [shared + 6100, shared + 30]
    lists, n_pages = layout(4, new, lens, PAGE, common=shared // PAGE)
    cache = cache_of(5, n_pages, hkv, PAGE)
    q = normal(6, hq, 6144, D).to(torch.bfloat16)
    one = bmx.PagedBatch.of(new, lens, lists)
    batch = bmx.PagedBatch(one.starts, one.lens, one.pages, 6144, max_new=2)
    out = torch.full((6144, hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    bmx.attention_paged(q, cache, batch, shared=shared, workspace=dirty(hq, hkv, batch, shared), out=out)
    rows = [0, 1, 6100, 6101]
    want, bound = attention_reference(q[:, rows].contiguous(), cache.k, cache.v, [2, 2], [shared + 2, lens[1]], lists,
                                      1 / math.sqrt(D), shared, half=False)
    hold(out[rows], want, bound)
    assert (out[2:6100] == 7).all() and (out[6102:] == 7).all()


def test_append_of_more_tokens_than_a_grid_row(gpu):
    """2^24 tokens and some, of which the first and the last few belong to sequences."""
    T, new = (1 << 24) + 5, [3, 4]
    lens = [3, 20]
    lists, n_pages = layout(7, new, lens, PAGE)
    cache = cache_of(8, n_pages, 1, PAGE)
    x = [torch.zeros(T, D, dtype=torch.bfloat16, device="cuda") for _ in "qkv"]
    rows = [0, 1, 2, T - 4, T - 3, T - 2, T - 1]
    for i, t in enumerate(x):
        t[rows] = normal(9 + i, 7, D).to(torch.bfloat16)
    w = [(1 + 0.3 * normal(12 + i, D)).to(torch.bfloat16) for i in range(2)]
    one = bmx.PagedBatch.of(new, lens, lists)
    starts = torch.tensor([0, 3, T - 4, T], dtype=torch.int32, device="cuda")
    # (the sequence between them has no pages, so its tokens no rows)
    three = bmx.PagedBatch(starts, torch.tensor([3, 0, 20], dtype=torch.int32, device="cuda"),
                           torch.stack([one.pages[0], torch.full_like(one.pages[0], -1), one.pages[1]]), T)
    got = bmx.qk_norm_rope_paged(*x, *w, cache, three)
    pos = torch.tensor([0, 1, 2, 16, 17, 18, 19], device="cuda")
    for y, w1, g in ((x[0], w[0], got[0, rows]), (x[1], w[1], torch.cat([cache.k[lists[0][0], 0, :3], cache.k[lists[1][1], 0, :4]]))):
        want, bound = rotated(y[rows].view(7, 1, D), w1, pos, 1e-6, 1e6)
        assert ((g.double() - want[:, 0]).abs() <= bound[:, 0]).all()
    assert torch.equal(torch.cat([cache.v[lists[0][0], 0, :3], cache.v[lists[1][1], 0, :4]]), x[2][rows])


# ---------------------------------------------------------------------------
# tiles of 256 query rows: 12288 a sequence
# ---------------------------------------------------------------------------
WIDE = [  # heads, new tokens, cached rows before them (own ones), shared rows
    ((64, 1), [200], [0], 0), ((64, 1), [193], [7], 0),     # one tile after another, the last ragged
    ((64, 1), [200], [5000], 0), ((64, 8), [1600], [3000], 0),  # cut along the keys, and joined
    ((40, 1), [620, 1], [33, 900], 0),                      # 40 rows to a token: tiles that end inside one
    ((64, 1), [390, 3], [0, 100], 48), ((64, 1), [200, 190], [3000, 0], 1008), ((48, 1), [500, 1, 300], [5, 700, 40], 16),
]


def wide(seed, heads, new, past, shared):
    lens = [n + p + shared for n, p in zip(new, past)]
    assert sum(new) * heads[0] // heads[1] >= 12288 * len(new)
    lists, n_pages = layout(seed, new, lens, PAGE, common=shared // PAGE)
    cache = cache_of(seed, n_pages, heads[1], PAGE)
    q = (1.5 * normal(seed + 9, heads[0], sum(new), D)).to(torch.bfloat16)
    return q, cache, lens, lists


def attend(q, cache, new, lens, lists, shared):
    batch = bmx.PagedBatch.of(new, lens, lists)
    got = bmx.attention_paged(q, cache, batch, shared=shared, workspace=dirty(q.shape[0], cache.n_kv_heads, batch, shared))
    want, bound = attention_reference(q, cache.k, cache.v, new, lens, lists, 1 / math.sqrt(D), shared, half=False)
    hold(got, want, bound)
    return got


@pytest.mark.parametrize("heads,new,past,shared", WIDE)
def test_wide_tiles(gpu, heads, new, past, shared):
    q, cache, lens, lists = wide(20, heads, new, past, shared)
    want = attend(q, cache, new, lens, lists, shared)
    # rows of nobody
    used = torch.zeros(cache.n_pages, PAGE, dtype=torch.bool, device="cuda")
    for pages, n in zip(lists, lens):
        for j in range(n):
            used[pages[j // PAGE], j % PAGE] = True
    for x in (cache.k, cache.v):
        x[(~used)[:, None, :, None].expand_as(x)] = math.nan
    assert torch.equal(attend(q, cache, new, lens, lists, shared), want)
    # pages that do not exist, among the first sequence's own
    lists[0][shared // PAGE + 1], lists[0][-1] = -3, cache.n_pages
    attend(q, cache, new, lens, lists, shared)


@pytest.mark.parametrize("heads,new,past,shared", WIDE)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_wide_tiles_values_not_finite(gpu, heads, new, past, shared, bad):
    """One that the later half of the first sequence's tokens see, and one that all see."""
    q, cache, lens, lists = wide(21, heads, new, past, shared)
    hkv, rep = heads[1], heads[0] // heads[1]
    want = attend(q, cache, new, lens, lists, shared)
    first = new[0] // 2
    at = lens[0] - new[0] + first
    cache.v[lists[0][at // PAGE], 0, at % PAGE, 77] = bad
    got = attend(q, cache, new, lens, lists, shared)
    g, w = (x.view(sum(new), hkv, rep, D) for x in (got, want))
    assert torch.equal(g[:first], w[:first]) and torch.equal(g[new[0]:], w[new[0]:])
    assert not torch.isfinite(g[first:new[0], 0, :, 77]).any()
    cache.v[lists[0][0], 0, 0, 5] = bad
    g = attend(q, cache, new, lens, lists, shared).view(sum(new), hkv, rep, D)
    assert not torch.isfinite(g[:sum(new) if shared else new[0], 0, :, 5]).any()


@pytest.mark.parametrize("heads,new,past,shared", WIDE)
def test_wide_tiles_of_large_and_small_values(gpu, heads, new, past, shared):
    q, cache, lens, lists = wide(22, heads, new, past, shared)
    cache.v[..., 3::5] *= 2.0 ** -40
    cache.v[:, :, 2::7] *= 2.0 ** 100
    attend(q, cache, new, lens, lists, shared)
