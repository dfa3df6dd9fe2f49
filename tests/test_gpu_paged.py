"""The paged KV cache of a batch on the GPU: rows normed, rotated and appended,
and attention of packed sequences over their pages, against the definitions in
float64."""
import math

import pytest
import torch

import bmx
from _paged_check import D, U24, attention_reference, hold, layout, normal, rotated, rows_of

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1e6


def cache_of(seed, n_pages, hkv, page):
    """Every row of every page holds something."""
    k = normal(seed, n_pages, hkv, page, D) * (0.5 + normal(seed + 1, 1, hkv, 1, D).abs()) + 0.7 * normal(seed + 2, 1, hkv, 1, D)
    return bmx.PagedKvCache(k.to(torch.bfloat16), normal(seed + 3, n_pages, hkv, page, D).to(torch.bfloat16))


def case(seed, heads, page, new, past, common=0, std=1.5):
    hq, hkv = heads
    lens = [n + p for n, p in zip(new, past)]
    lists, n_pages = layout(seed, new, lens, page, common=common)
    cache = cache_of(seed, n_pages, hkv, page)
    q = (std * normal(seed + 9, hq, sum(new), D)).to(torch.bfloat16)
    return q, cache, bmx.PagedBatch.of(new, lens, lists), lens, lists


def check(q, cache, batch, new, lens, lists, shared=0, scale=None, what="", half=None, **kw):
    got = bmx.attention_paged(q, cache, batch, scale=scale, shared=shared, **kw)
    if half is None:  # more query rows per kv head than 64, or shared ones: weights in fp16
        half = shared > 0 or batch.max_new * (q.shape[0] // cache.n_kv_heads) > 64
    out, bound = attention_reference(q, cache.k, cache.v, new, lens, lists, 1 / math.sqrt(D) if scale is None else scale,
                                     shared, half=half)
    T = sum(new)
    hold(got[:T], out[:T], bound[:T], what)
    return got


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
APPENDS = [
    ((32, 8), 64, [1], [4095]), ((32, 8), 16, [1] * 65, [(37 * i) % 200 for i in range(65)]),
    ((16, 8), 32, [5, 0, 1, 40, 33], [0, 7, 31, 30, 0]), ((6, 2), 128, [129, 1], [0, 127]), ((10, 2), 256, [3, 2], [255, 300]),
    ((64, 8), 16, [17], [15]), ((8, 8), 4096, [2, 3], [4095, 5]), ((1, 1), 16, [1], [0]),
    ((4, 2), 16, [0] * 70 + [2] + [0] * 200 + [1] * 30, [i % 19 for i in range(301)]),
]


def projections(seed, heads, T):
    hq, hkv = heads
    x = [(normal(seed + i, T, h * D) * (0.2 + normal(seed + 5, T, 1).abs())).to(torch.bfloat16) for i, h in enumerate((hq, hkv, hkv))]
    w = [(1 + 0.3 * normal(seed + 7 + i, D)).to(torch.bfloat16) for i in range(2)]
    return (*x, *w)


def positions(new, lens):
    return torch.cat([torch.arange(n - m, n) for m, n in zip(new, lens)]).cuda()


def check_append(heads, cache, batch, new, lens, lists, q, k, v, qn, kn, eps=EPS, theta=THETA, **kw):
    hq, hkv = heads
    T = sum(new)
    before = cache.k.clone(), cache.v.clone()
    got = bmx.qk_norm_rope_paged(q, k, v, qn, kn, cache, batch, eps=eps, theta=theta, **kw)
    pos = positions(new, lens)
    want, bound = rotated(q[:T].view(T, hq, D), qn, pos, eps, theta)
    assert ((got[:, :T].transpose(0, 1).double() - want).abs() <= bound).all()
    want_k, bound_k = rotated(k[:T].view(T, hkv, D), kn, pos, eps, theta)
    page, t = cache.page_size, 0
    touched = torch.zeros(cache.n_pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(new):
        for i in range(n):
            p = lens[b] - n + i
            pg, r = lists[b][p // page], p % page
            touched[pg, r] = True
            assert ((cache.k[pg, :, r].double() - want_k[t]).abs() <= bound_k[t]).all(), (b, i)
            assert torch.equal(cache.v[pg, :, r], v[t].view(hkv, D)), (b, i)
            t += 1
    for now, was in zip((cache.k, cache.v), before):
        assert ((now == was) | touched[:, None, :, None]).all()
    return got


@pytest.mark.parametrize("heads,page,new,past", APPENDS)
def test_append(gpu, heads, page, new, past):
    lens = [n + p for n, p in zip(new, past)]
    lists, n_pages = layout(3, new, lens, page)
    check_append(heads, cache_of(1, n_pages, heads[1], page), bmx.PagedBatch.of(new, lens, lists), new, lens, lists,
                 *projections(11, heads, sum(new)))


def test_append_leaves_other_rows(gpu):
    """Rows behind the last sequence, and before the first, stay as they were."""
    heads, new, lens = (4, 2), [2, 3], [20, 3]
    lists, n_pages = layout(4, new, lens, 16)
    cache = cache_of(5, n_pages, 2, 16)
    x = projections(6, heads, 9)
    starts = torch.tensor([1, 3, 6], dtype=torch.int32, device="cuda")
    one = bmx.PagedBatch.of(new, lens, lists)
    batch = bmx.PagedBatch(starts, one.lens, one.pages, 9)
    out = torch.full((4, 9, D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = bmx.qk_norm_rope_paged(*x, cache, batch, out=out)
    assert (got[:, :1] == 7).all() and (got[:, 6:] == 7).all()
    want, bound = rotated(x[0][1:6].view(5, 4, D), x[3], positions(new, lens), EPS, THETA)
    assert ((got[:, 1:6].transpose(0, 1).double() - want).abs() <= bound).all()


@pytest.mark.parametrize("theta", [1e4, 1e6])
def test_append_far_positions(gpu, theta):
    """Positions up to 2^24 - 1, where an angle in fp32 would be off by half a radian."""
    new, lens = [4, 3], [1 << 24, 1000003]
    lists = [[-1] * 4095 + [1], [-1] * (1000003 // 4096) + [0] + [-1] * (4095 - 1000003 // 4096)]
    cache = cache_of(8, 2, 2, 4096)
    check_append((4, 2), cache, bmx.PagedBatch.of(new, lens, lists), new, lens, lists, *projections(9, (4, 2), 7), theta=theta)


@pytest.mark.parametrize("len0", [(1 << 24) + 2, (1 << 24) + 300, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [[5, 1], [60, 1], [300, 1]])
def test_lengths_past_the_largest_table(gpu, len0, new):
    """Of a table of 2^24 rows: what lies past it is not written, and sees all that is there."""
    heads, lens = (4, 2), [len0, 40]
    lists = [[-1] * 4095 + [1], [0] + [-1] * 4095]
    cache = cache_of(33, 2, 2, 4096)
    x = projections(34, heads, sum(new))
    batch = bmx.PagedBatch.of(new, lens, lists)
    before = cache.k.clone(), cache.v.clone()
    q = bmx.qk_norm_rope_paged(*x, cache, batch)
    inside = max(0, (1 << 24) - (len0 - new[0]))  # tokens with a row
    assert torch.equal(cache.v[1, :, 4096 - inside:], x[2][:inside].view(inside, 2, D).transpose(0, 1))
    cache.k[1, :, 4096 - inside:], cache.v[1, :, 4096 - inside:] = (y[1, :, 4096 - inside:] for y in before)
    assert torch.equal(cache.k[1], before[0][1]) and torch.equal(cache.v[1], before[1][1])
    got = bmx.attention_paged(q, cache, batch)
    # the same rows as a short sequence's
    cut = [4096 + max(0, len0 - (1 << 24)), 40]
    short = [[1], [0]]
    want, bound = attention_reference(q, cache.k, cache.v, new, cut, short, 1 / math.sqrt(D), cap=4096)
    hold(got, want, bound)


def test_append_without_a_page(gpu):
    """Page numbers that do not exist, positions outside the table: no cache row, the queries all the same."""
    heads, new = (4, 2), [3, 2, 2, 1]
    lens = [18, 5, 1, 33]      # the third begins at position -1, the fourth lies past the table
    lists = [[0, 99], [-5, 2], [1, 2], [0, 2]]
    cache = cache_of(2, 3, 2, 16)
    x = projections(3, heads, 8)
    k0, v0 = cache.k.clone(), cache.v.clone()
    got = bmx.qk_norm_rope_paged(*x, cache, bmx.PagedBatch.of(new, lens, lists))
    pos = positions(new, lens)
    want, bound = rotated(x[0].view(8, 4, D), x[3], pos, EPS, THETA)
    assert ((got.transpose(0, 1).double() - want).abs() <= bound).all()
    written = [(0, 15, 0), (1, 0, 6)]  # page, row, token: the first sequence's first, the third's second
    for pg, r, t in written:
        assert torch.equal(cache.v[pg, :, r], x[2][t].view(2, D)) and not torch.equal(cache.k[pg, :, r], k0[pg, :, r])
        cache.k[pg, :, r], cache.v[pg, :, r] = k0[pg, :, r], v0[pg, :, r]
    assert torch.equal(cache.k, k0) and torch.equal(cache.v, v0)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
EDGES = [0, 1, 14, 15, 16, 17, 30, 31, 32, 62, 63, 64, 95, 126, 127, 128, 129, 255, 256, 1000]


@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (6, 2), (10, 2), (16, 1), (40, 1), (64, 1), (21, 7)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode(gpu, heads, page):
    new = [1] * len(EDGES)
    check(*(c := case(1, heads, page, new, EDGES))[:3], new, *c[3:])


@pytest.mark.parametrize("past", [0, 4096, 131071])
@pytest.mark.parametrize("heads", [(32, 8), (1, 1)])
def test_decode_one(gpu, heads, past):
    check(*(c := case(2, heads, 64, [1], [past]))[:3], [1], *c[3:])


@pytest.mark.parametrize("heads,most", [((32, 8), 4), ((32, 8), 8), ((64, 8), 8), ((16, 8), 30), ((6, 2), 21), ((10, 2), 3)])
def test_verify(gpu, heads, most):
    """Several tokens each, the empty sequence among them: up to 64 rows per kv head."""
    new = [most, 0, 1, 2, most, most - 1, 1, most]
    past = [0, 40, 0, 15, 127, 1000, 2049, 31]
    check(*(c := case(3, heads, 32, new, past))[:3], new, *c[3:])


PROMPTS = [
    ((32, 8), 64, [4096], [0]), ((32, 8), 16, [1, 17, 333, 0, 1000, 2], [0] * 6), ((32, 8), 128, [2048], [2048]),
    ((64, 8), 32, [9, 100, 31], [3, 1000, 64]), ((16, 8), 256, [513, 1], [255, 3000]), ((6, 2), 16, [127, 128, 129, 43], [5, 0, 64, 63]),
    ((10, 2), 64, [300], [77]), ((8, 8), 64, [65, 64, 63, 200], [0, 1, 63, 500]), ((1, 1), 16, [70], [16]),
    ((5, 1), 32, [1000], [9000]), ((32, 8), 32, [509] + [1] * 31, [1503] + [97 * i for i in range(31)]),
    ((128, 1), 16, [1, 2], [33, 5]), ((32, 8), 64, [64], [30000]),
]


@pytest.mark.parametrize("heads,page,new,past", PROMPTS)
def test_prompts(gpu, heads, page, new, past):
    check(*(c := case(4, heads, page, new, past))[:3], new, *c[3:])


def test_prompts_of_many_lengths(gpu):
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 90, (60,), generator=g).tolist()
    past = torch.randint(0, 300, (60,), generator=g).tolist()
    check(*(c := case(5, (4, 2), 16, new, past))[:3], new, *c[3:])


@pytest.mark.parametrize("heads,page,shared,new,past", [
    ((32, 8), 64, 4096, [1] * 64, [11 * i for i in range(64)]), ((8, 8), 16, 16, [1, 1, 1], [0, 1, 200]),
    ((6, 2), 32, 96, [1, 0, 2, 3], [0, 5, 31, 32]), ((32, 8), 256, 512, [40, 1, 0, 200], [0, 3, 9, 100]),
    ((64, 8), 16, 80, [5] * 9, [0] * 9), ((5, 1), 16, 1008, [70, 1], [0, 0]), ((32, 8), 128, 16384, [1, 1], [100, 1]),
    ((4, 4), 64, 64, [1], [0])])
def test_shared_rows(gpu, heads, page, shared, new, past):
    common = shared // page
    q, cache, batch, lens, lists = case(6, heads, page, new, [p + shared for p in past], common=common)
    got = check(q, cache, batch, new, lens, lists, shared=shared)
    # sequence 0's table names the pages: the others' entries for them are not read
    for b in range(1, len(new)):
        batch.pages[b, :common] = -1
    assert torch.equal(bmx.attention_paged(q, cache, batch, shared=shared), got)


@pytest.mark.parametrize("new,past", [([1, 1, 1], [50, 3, 200]), ([3, 1, 4], [50, 3, 200]), ([90, 1, 40], [50, 3, 70])])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.5])
def test_scales(gpu, new, past, scale):
    check(*(c := case(7, (8, 2), 16, new, past))[:3], new, *c[3:], scale=scale)


@pytest.mark.parametrize("new,past", [([1, 1, 1], [50, 3, 2000]), ([3, 1, 4], [50, 3, 200]), ([90, 1, 400], [50, 3, 70])])
@pytest.mark.parametrize("shared", [0, 160])
@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** 20, 2.0 ** 100, 2.0 ** -100])
def test_values_of_any_size(gpu, new, past, shared, size):
    """All values small or large; then one row, or 8 values of one, among others of size 1."""
    past = [p + shared for p in past]
    q, cache, batch, lens, lists = case(7, (8, 2), 16, new, past, common=shared // 16)
    plain = cache.v.clone()
    cache.v.mul_(size)
    check(q, cache, batch, new, lens, lists, shared=shared, half=False)
    for b, at in ((0, 5), (2, 60), (2, 100 + shared)):  # (in the shared rows, or not)
        cache.v.copy_(plain)
        pg, r = lists[b][at // 16], at % 16
        cache.v[pg, 0, r] *= size
        cache.v[pg, 1, r, 40:48] *= size
        check(q, cache, batch, new, lens, lists, shared=shared, half=size < 1 or None)
        cache.v[pg, :, r] = 0
        check(q, cache, batch, new, lens, lists, shared=shared)


@pytest.mark.parametrize("new,past", [([3, 1, 4], [500, 3, 200]), ([10, 1, 9], [500, 3, 200]), ([90, 1, 400], [50, 3, 70])])
@pytest.mark.parametrize("shared", [0, 160])
@pytest.mark.parametrize("size", [2.0 ** -10, 2.0 ** -17, 2.0 ** -24])
def test_small_dimensions(gpu, new, past, shared, size):
    """Dimensions whose values are far smaller than their neighbours' keep their precision."""
    q, cache, batch, lens, lists = case(8, (8, 2), 16, new, [p + shared for p in past], common=shared // 16)
    cache.v[..., 3::5].mul_(size)
    check(q, cache, batch, new, lens, lists, shared=shared)


@pytest.mark.parametrize("new,past", [([1, 1, 1, 1], [50, 3, 200, 0]), ([3, 1, 4, 2], [50, 3, 200, 0]), ([90, 1, 40, 70], [50, 3, 70, 0])])
@pytest.mark.parametrize("shared", [0, 32])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_nobody_sees(gpu, new, past, shared, bad):
    """NaN and infinities past the sequences' ends and on pages of nobody change no bit."""
    past = [p + shared for p in past]
    q, cache, batch, lens, lists = case(8, (8, 2), 16, new, past, common=shared // 16)
    want = check(q, cache, batch, new, lens, lists, shared=shared)
    used = torch.zeros(cache.n_pages, 16, dtype=torch.bool, device="cuda")
    for pages, n in zip(lists, lens):
        for j in range(n):
            used[pages[j // 16], j % 16] = True
    hide = (~used)[:, None, :, None].expand_as(cache.k)
    cache.k[hide] = bad
    cache.v[hide] = bad
    assert torch.equal(bmx.attention_paged(q, cache, batch, shared=shared), want)


@pytest.mark.parametrize("heads,new", [((8, 2), [4, 2]), ((16, 2), [4, 2]), ((32, 2), [4, 2]), ((8, 2), [100, 40]), ((6, 2), [257, 33])])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_that_some_see(gpu, heads, new, bad):
    """A new token's value that is not finite: the earlier tokens' outputs keep
    their bits, the later ones' are not finite in that dimension alone (and
    right in the others: `check`)."""
    past = [30, 61]
    q, cache, batch, lens, lists = case(10, heads, 16, new, past)
    want = check(q, cache, batch, new, lens, lists)
    at = lens[0] - new[0] // 2  # a row half of the first sequence's tokens see
    pg, r = lists[0][at // 16], at % 16
    cache.v[pg, 0, r, 5] = bad
    cache.v[pg, 1, r, 77] = bad
    got = check(q, cache, batch, new, lens, lists)
    rep, first = heads[0] // 2, new[0] - new[0] // 2  # tokens of the first sequence before `at`
    g, w = (x.view(sum(new), 2, rep, D).clone() for x in (got, want))
    assert torch.equal(g[:first], w[:first])
    assert torch.equal(g[new[0]:], w[new[0]:])
    for h, d in ((0, 5), (1, 77)):
        bits = g[first:new[0], h, :, d]
        assert (torch.isnan(bits) | (bits == bad)).all()
    # a key: those that see it are lost, the others stay
    cache.v[pg, 0, r, 5] = cache.v[pg, 1, r, 77] = 1.0
    want = check(q, cache, batch, new, lens, lists).view(sum(new), 2, rep, D)
    cache.k[pg, 0, r, 3] = math.nan
    got = bmx.attention_paged(q, cache, batch).view(sum(new), 2, rep, D)
    assert torch.isnan(got[first:new[0], 0]).all()
    assert torch.equal(got[:first], want[:first]) and torch.equal(got[new[0]:], want[new[0]:])
    assert torch.equal(got[:, 1], want[:, 1])


@pytest.mark.parametrize("new,past", [([1, 1, 1], [50, 100, 200]), ([3, 1, 4], [50, 100, 200]), ([90, 1, 40], [50, 100, 70])])
def test_pages_that_do_not_exist(gpu, new, past):
    q, cache, batch, lens, lists = case(12, (8, 2), 16, new, past)
    lists[0][1], lists[1][0], lists[2][-1] = -7, cache.n_pages, 1 << 30
    lists[2][2] = -1
    batch = bmx.PagedBatch.of(new, lens, lists)
    check(q, cache, batch, new, lens, lists)
    # a sequence of which nothing exists
    lists[0] = [-1] * len(lists[0])
    got = check(q, cache, bmx.PagedBatch.of(new, lens, lists), new, lens, lists)
    assert (got[:new[0]] == 0).all()


@pytest.mark.parametrize("new,lens", [([2, 3, 1], [1, 0, 20]), ([3, 1, 2], [-5, 1, -1]), ([70, 40, 1], [3, 0, 20])])
def test_tokens_that_see_nothing(gpu, new, lens):
    """More new tokens than cached rows: those at negative positions get zeros."""
    lists, n_pages = layout(13, new, lens, 16)
    lists = [x + [0] * (3 - len(x)) for x in lists]
    cache = cache_of(14, n_pages, 2, 16)
    q = normal(15, 8, sum(new), D).to(torch.bfloat16)
    got = check(q, cache, bmx.PagedBatch.of(new, lens, lists), new, lens, lists)
    row = 0
    for n, L in zip(new, lens):
        assert (got[row:row + max(0, n - max(L, 0))] == 0).all()
        row += n


@pytest.mark.parametrize("new", [[2, 3], [80, 31]])
def test_rows_of_no_sequence_stay(gpu, new):
    q, cache, one, lens, lists = case(16, (8, 2), 16, new, [20, 3])
    T = sum(new)
    q = torch.cat([torch.full((8, 2, D), math.nan, dtype=torch.bfloat16, device="cuda"), q,
                   torch.full((8, 5, D), math.nan, dtype=torch.bfloat16, device="cuda")], 1).contiguous()
    batch = bmx.PagedBatch(one.starts + 2, one.lens, one.pages, T + 7, max_new=max(new))
    for shared in (0, 16):
        for b in range(1, 2):
            batch.pages[b, 0] = batch.pages[0, 0]
        lists[1][0] = lists[0][0]
        use, past = (new, [20, 3])
        if shared:  # every sequence has the shared rows
            batch.lens.copy_(torch.tensor([n + 20 for n in new], dtype=torch.int32))
            lens = [n + 20 for n in new]
            wide, n_pages = layout(17, new, lens, 16, common=1)
            cache = cache_of(18, n_pages, 2, 16)
            lists = wide
            batch = bmx.PagedBatch(one.starts + 2, batch.lens, bmx.PagedBatch.of(new, lens, wide).pages, T + 7, max_new=max(new))
        out = torch.full((T + 7, 8 * D), 7.0, dtype=torch.bfloat16, device="cuda")
        got = bmx.attention_paged(q, cache, batch, out=out, shared=shared)
        assert (got[:2] == 7).all() and (got[2 + T:] == 7).all()
        want, bound = attention_reference(q[:, 2:2 + T].contiguous(), cache.k, cache.v, new, lens, lists, 1 / math.sqrt(D), shared)
        hold(got[2:2 + T], want, bound)


@pytest.mark.parametrize("hkv,seqs", [(4, 2048), (4, 2049), (2, 4096), (3, 4096)])
@pytest.mark.parametrize("n", [1, 5])
def test_many_sequences(gpu, hkv, seqs, n):
    """As many pairs of sequences and kv heads as there are counters, and more; some
    sequences empty, some long."""
    new = [n if b % 7 else 0 for b in range(seqs)]
    past = [(37 * b) % 50 + (3000 if b % 500 == 1 else 0) for b in range(seqs)]
    q, cache, batch, lens, lists = case(21, (4 * hkv, hkv), 64, new, past)
    got = bmx.attention_paged(q, cache, batch)
    for b in (1, 2, 3, 499, 501, 1001, 1501, seqs - 2):
        if new[b]:
            at = sum(new[:b])
            want, bound = attention_reference(q[:, at:at + n].contiguous(), cache.k, cache.v, [n], [lens[b]], [lists[b]],
                                              1 / math.sqrt(D), half=False)
            hold(got[at:at + n], want, bound, f"sequence {b}")


@pytest.mark.parametrize("new,max_new", [([6, 2, 9], 4), ([60, 2, 90], 50)])
def test_tokens_past_max_new_stay(gpu, new, max_new):
    q, cache, one, lens, lists = case(19, (8, 2), 16, new, [20, 3, 40])
    batch = bmx.PagedBatch(one.starts, one.lens, one.pages, sum(new), max_new=max_new)
    out = torch.full((sum(new), 8 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = bmx.attention_paged(q, cache, batch, out=out)
    want, bound = attention_reference(q, cache.k, cache.v, new, lens, lists, 1 / math.sqrt(D))
    row = 0
    for n in new:
        m = min(n, max_new)
        hold(got[row:row + m], want[row:row + m], bound[row:row + m])
        assert (got[row + m:row + n] == 7).all()
        row += n


def test_pages_past_4_gib(gpu):
    """Pages whose offsets need more than 32 bits, in bytes and in values."""
    n_pages = (5 << 30) // (8 * 256 * D)
    k = torch.zeros(n_pages, 8, 256, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    cache = bmx.PagedKvCache(k, v)
    far = [n_pages - 1, 0, n_pages - 2, n_pages // 2 + 1, 3]
    for i, p in enumerate(far):
        k[p], v[p] = (normal(20 + 2 * i + j, 8, 256, D).to(torch.bfloat16) for j in range(2))
    for new in ([1, 1], [3, 2], [200, 1]):
        lens = [700, 600]
        lists = [[far[0], far[1], far[2]], [far[3], far[4], far[0]]]
        q = normal(31, 32, sum(new), D).to(torch.bfloat16)
        check(q, cache, bmx.PagedBatch.of(new, lens, lists), new, lens, lists)
    x = projections(32, (32, 8), 2)
    check_append((32, 8), cache, bmx.PagedBatch.of([1, 1], [701, 601], lists), [1, 1], [701, 601], lists, *x)


@pytest.mark.parametrize("new,past,shared", [([1, 1, 1, 1], [500, 3, 2000, 0], 0), ([3, 1, 4, 2], [50, 3, 200, 0], 32),
                                             ([90, 1, 400, 70], [50, 3, 70, 0], 0), ([90, 1, 40, 70], [50, 3, 70, 0], 32)])
def test_equal_calls_give_equal_bits(gpu, new, past, shared):
    past = [p + shared for p in past]
    q, cache, batch, lens, lists = case(33, (8, 2), 16, new, past, common=shared // 16)
    ws = bmx.attention_paged_workspace(8, 2, batch, shared=shared)
    first = check(q, cache, batch, new, lens, lists, shared=shared, workspace=ws)
    for fill in (0, 255, 127):
        ws[bmx.PAGED_COUNTER_BYTES:].fill_(fill)  # any contents
        assert torch.equal(bmx.attention_paged(q, cache, batch, shared=shared, workspace=ws), first)
        assert not ws[:bmx.PAGED_COUNTER_BYTES].any()


@pytest.mark.parametrize("new,shared", [([1, 1, 1, 0], 0), ([1, 1, 1, 0], 32), ([3, 2, 0, 60], 0), ([3, 2, 0, 60], 32)])
def test_graph_replays_with_other_batches(gpu, new, shared):
    """A captured append and attention, replayed with other lengths, starts and
    pages between eager calls; two graphs with a workspace each."""
    heads, page, T = (8, 2), 16, sum(new) + 3
    lens = [n + p + shared for n, p in zip(new, [100, 31, 0, 7])]
    lists, n_pages = layout(40, new, [n + 40 for n in lens], page, common=shared // page)
    batch = bmx.PagedBatch.of(new, lens, lists)
    batch = bmx.PagedBatch(batch.starts, batch.lens, batch.pages, T, max_new=max(new))
    cache = cache_of(41, n_pages, 2, page)
    x = projections(42, heads, T)
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        ws = bmx.attention_paged_workspace(8, 2, batch, shared=shared)
        qo = torch.zeros(8, T, D, dtype=torch.bfloat16, device="cuda")
        out = torch.zeros(T, 8 * D, dtype=torch.bfloat16, device="cuda")

        def step():
            bmx.qk_norm_rope_paged(*x, cache, batch, out=qo)
            bmx.attention_paged(qo, cache, batch, shared=shared, workspace=ws, out=out)

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append((g, qo, out, ws))
    for turn in range(4):
        cur = new if turn % 2 == 0 else new[::-1]
        now = [(7 * turn) % 30 + n + shared + (11 if turn else 0) for n in cur]
        other = bmx.PagedBatch.of(cur, now, lists)
        batch.starts.copy_(other.starts)
        batch.lens.copy_(other.lens)
        for xi in x[:3]:
            xi.copy_(normal(50 + turn, *xi.shape).to(torch.bfloat16))
        for g, qo, out, _ in graphs:
            g.replay()
        want_q = torch.zeros_like(graphs[0][1])
        bmx.qk_norm_rope_paged(*x, cache, other if other.tokens == T else batch, out=want_q)
        n = sum(cur)
        want = check(want_q[:, :n].contiguous(), cache, other, cur, now, lists, shared=shared)
        torch.cuda.synchronize()
        for g, qo, out, _ in graphs:
            assert torch.equal(qo[:, :n], want_q[:, :n])
            ref, bound = attention_reference(want_q[:, :n].contiguous(), cache.k, cache.v, cur, now, lists, 1 / math.sqrt(D), shared)
            hold(out[:n], ref, bound)
        assert torch.equal(graphs[0][2], graphs[1][2])


def test_two_streams_at_once(gpu):
    cases = [case(60 + i, (32, 8), 64, new, past) for i, (new, past) in enumerate([([1] * 9, [400 * j for j in range(9)]), ([300, 7, 1], [5, 900, 2000])])]
    news = [[1] * 9, [300, 7, 1]]
    want = [check(*c[:3], n, *c[3:]) for c, n in zip(cases, news)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            got[i].append(bmx.attention_paged(*c[:3], stream=s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_batch_grows_like_its_sequences(gpu):
    """Three steps of a batch -- packed prompts, a chunk beside decode steps, a
    plain decode step -- appended and attended, against each sequence alone in a
    contiguous cache through the same projections."""
    hq, hkv, page = 8, 2, 16
    n_seqs, room = 4, 200
    lists, n_pages = layout(70, [], [room] * n_seqs, page)
    cache = bmx.PagedKvCache.empty(n_pages, hkv, page)
    alone = [(torch.zeros(hkv, room, D, dtype=torch.bfloat16, device="cuda"),) * 1 + (torch.zeros(hkv, room, D, dtype=torch.bfloat16, device="cuda"),) for _ in range(n_seqs)]
    lens = [0] * n_seqs
    for step, new in enumerate(([50, 1, 17, 0], [1, 30, 1, 64], [1, 1, 1, 1], [2, 1, 3, 1])):
        T = sum(new)
        lens = [a + b for a, b in zip(lens, new)]
        batch = bmx.PagedBatch.of(new, lens, lists)
        q, k, v, qn, kn = projections(80 + step, (hq, hkv), T)
        qo = bmx.qk_norm_rope_paged(q, k, v, qn, kn, cache, batch)
        out = bmx.attention_paged(qo, cache, batch)
        row = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            s = slice(row, row + n)
            kc, vc = alone[b]
            q1 = bmx.qk_norm_rope_kv(q[s].contiguous(), k[s].contiguous(), v[s].contiguous(), qn, kn, kc, vc, lens[b] - n)
            o1 = bmx.attention(q1, kc, vc, lens[b] - n)
            # the norm rounds to bf16 twice more there: three roundings against one,
            # each up to 2^-8 of a value of the pair
            got_k = rows_of(cache.k, lists[b], lens[b])[0].double()
            assert ((got_k - kc[:, :lens[b]].double()).abs().amax() / got_k.abs().amax()) < 4 * 2.0 ** -8 * math.sqrt(2)
            assert torch.equal(rows_of(cache.v, lists[b], lens[b])[0], vc[:, :lens[b]])
            assert float((out[s].double() - o1.double()).norm() / o1.double().norm()) < 4 * 2.0 ** -8
            row += n
        ref, bound = attention_reference(qo, cache.k, cache.v, new, lens, lists, 1 / math.sqrt(D))
        hold(out, ref, bound, f"step {step}")


def test_empty_calls(gpu):
    cache = cache_of(90, 2, 2, 16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    none = bmx.PagedBatch(i32(3), i32(2), i32(2, 1), 0)
    assert bmx.attention_paged(bf(4, 0, D), cache, none).shape == (0, 4 * D)
    assert bmx.qk_norm_rope_paged(bf(0, 4 * D), bf(0, 2 * D), bf(0, 2 * D), bf(D), bf(D), cache, none).shape == (4, 0, D)
    nobody = bmx.PagedBatch(i32(1), i32(0), i32(0, 1), 3)
    out = bf(3, 4 * D) + 7
    assert (bmx.attention_paged(bf(4, 3, D), cache, nobody, out=out) == 7).all()
    idle = bmx.PagedBatch(i32(3), i32(2) + 5, i32(2, 1), 3)  # two sequences without a new token
    for max_new in (1, 3):
        idle = bmx.PagedBatch(i32(3), i32(2) + 5, i32(2, 1), 3, max_new=max_new)
        assert (bmx.attention_paged(bf(64, 3, D), cache, idle, out=bf(3, 64 * D) + 7) == 7).all()
    torch.cuda.synchronize()


@pytest.mark.parametrize("new", [[1, 1, 1], [9, 2, 1], [120, 1, 33]])
@pytest.mark.parametrize("page,past", [(4096, [4090, 9000, 100]), (2048, [4090, 3, 2047])])
def test_large_pages(gpu, new, page, past):
    q, cache, batch, lens, lists = case(100, (8, 2), page, new, past)
    check(q, cache, batch, new, lens, lists)


@pytest.mark.parametrize("new", [[1, 1, 1], [6, 2, 1], [9, 1, 12], [90, 1, 40]])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_not_finite_in_shared_rows(gpu, new, bad):
    """Every query sees them: that dimension is lost, the others stay right."""
    q, cache, batch, lens, lists = case(101, (8, 2), 16, new, [300, 260, 500], common=10)
    want = check(q, cache, batch, new, lens, lists, shared=160)
    pg = lists[0][4]
    cache.v[pg, 1, 7, 9] = bad
    got = check(q, cache, batch, new, lens, lists, shared=160).view(-1, 2, 4, D)
    assert (torch.isnan(got[:, 1, :, 9]) | (got[:, 1, :, 9] == bad)).all()
    assert torch.equal(got[:, 0], want.view(-1, 2, 4, D)[:, 0])


@pytest.mark.parametrize("new,past", [([1, 1, 1], [50, 100, 2000]), ([3, 1, 4], [50, 100, 2000]), ([11, 1, 9], [50, 100, 2000]),
                                      ([90, 1, 400], [50, 100, 70])])
@pytest.mark.parametrize("shared", [0, 32])
def test_scores_of_minus_infinity(gpu, new, past, shared):
    """Keys whose product with a query is -inf have no weight; all of them: zeros."""
    q, cache, batch, lens, lists = case(102, (8, 2), 16, new, past, common=shared // 16)
    q[..., 0] = 1.0
    seen = cache.k.clone()
    cache.k[..., 0, 0] = -math.inf   # the first row of every page
    got = bmx.attention_paged(q, cache, batch, shared=shared)
    row = 0
    for b, n in enumerate(new):
        for i in {0, n - 1}:
            L = lens[b] - n + i + 1
            pages = lists[0][:shared // 16] + lists[b][shared // 16:]
            k, v = (rows_of(x, pages, L)[0].double() for x in (seen, cache.v))
            s = (q[:, row + i].double().view(2, 4, D) @ k.transpose(1, 2).contiguous()) / math.sqrt(D)
            s[..., ::16] = -math.inf
            want = s.softmax(-1) @ v
            # (an output's rounding and 2^-11 of a weight's, with the values' largest)
            assert (got[row + i].view(2, 4, D).double() - want).abs().max() <= 2.0 ** -8 * float(want.abs().max()) + 2.0 ** -11 * 6
        row += n
    cache.k[..., 0] = -math.inf
    assert (bmx.attention_paged(q, cache, batch, shared=shared) == 0).all()


def test_python_refusals(gpu):
    q, cache, batch, lens, lists = case(103, (8, 2), 16, [2, 3], [20, 30])
    x = projections(104, (8, 2), 5)

    def refused(code, f, *a, **k):
        with pytest.raises(bmx.BmxError) as e:
            f(*a, **k)
        assert e.value.code == code, e.value

    att, app = bmx.attention_paged, bmx.qk_norm_rope_paged
    for bad in (q.float(), q.cpu(), q.transpose(0, 1)):
        refused(bmx.BMX_E_ARG, att, bad, cache, batch)
    for bad in (q[:, :4].contiguous(), q[:5].contiguous(), q[..., :64].contiguous(), q.view(-1)):
        refused(bmx.BMX_E_SHAPE, att, bad, cache, batch)
    refused(bmx.BMX_E_ARG, att, q, cache, batch, shared=8)
    refused(bmx.BMX_E_ARG, att, q, cache, batch, shared=-16)
    refused(bmx.BMX_E_ARG, att, q, cache, batch, shared=1 << 20)
    refused(bmx.BMX_E_ARG, att, q, cache, batch, out=q)
    refused(bmx.BMX_E_ARG, att, q, cache, batch, out=q.float())
    refused(bmx.BMX_E_SHAPE, att, q, cache, batch, out=q.new_empty(5, 7 * D))
    ws = bmx.attention_paged_workspace(8, 2, batch)
    refused(bmx.BMX_E_ARG, att, q, cache, batch, workspace=ws[:-1])
    refused(bmx.BMX_E_ARG, att, q, cache, batch, workspace=ws.cpu())
    refused(bmx.BMX_E_ARG, att, q, cache, batch, workspace=ws[::2])
    for i in range(5):
        for bad, code in ((x[i].float(), bmx.BMX_E_ARG), (x[i].cpu(), bmx.BMX_E_ARG),
                          (x[i][..., :-1].contiguous(), bmx.BMX_E_SHAPE), (x[i][:4].contiguous(), bmx.BMX_E_SHAPE)):
            refused(code, app, *x[:i], bad, *x[i + 1:], cache, batch)
    refused(bmx.BMX_E_SHAPE, app, *x, cache, batch, out=q[:4].contiguous())
    refused(bmx.BMX_E_ARG, app, *x, cache, batch, out=x[0].view(8, 5, D))
    k = cache.k
    for bad, code in (((k, k[:-1]), bmx.BMX_E_SHAPE), ((k, k.float()), bmx.BMX_E_ARG), ((k[0], k[0]), bmx.BMX_E_SHAPE),
                      ((k.transpose(0, 1), k), bmx.BMX_E_ARG)):
        refused(code, bmx.PagedKvCache, *bad)
    for bad, code in (((batch.starts, batch.starts, batch.pages, 5), bmx.BMX_E_SHAPE), ((batch.starts.long(), batch.lens, batch.pages, 5), bmx.BMX_E_ARG),
                      ((batch.starts, batch.lens, batch.pages, -1), bmx.BMX_E_SHAPE), ((batch.starts, batch.lens, batch.pages, 5, 6), bmx.BMX_E_SHAPE),
                      ((batch.starts, batch.lens, batch.pages, 5, 0), bmx.BMX_E_SHAPE), ((batch.starts, batch.lens, batch.lens, 5), bmx.BMX_E_SHAPE)):
        refused(code, bmx.PagedBatch, *bad)
    with pytest.raises(bmx.BmxError):
        batch.lens = batch.lens.clone()
    refused(bmx.BMX_E_SHAPE, bmx.attention_paged_workspace, 7, 2, batch)
    refused(bmx.BMX_E_SHAPE, bmx.attention_paged_workspace, 8, 2, (5, 2, 6))
    check(q, cache, batch, [2, 3], lens, lists, workspace=ws)
