"""Attention over the 4-bit KV cache at the ends of its values' range: infinite
scales and biases, magnitudes up to 2^120, contexts whose values span the
exponent's range, groups far apart.  Through every kernel."""
import math

import pytest
import torch

import bmx
from _kv4_check import D, check
from test_gpu_kv4 import queries, random_cache

pytestmark = pytest.mark.gpu

# a call for each kernel: one token, few rows, more, tiles of 64, of 256, tiles over split keys
KERNELS = [(8, 2, 1, 700), (16, 2, 1, 700), (8, 2, 40, 70), (64, 8, 130, 70), (32, 8, 1024, 0), (64, 8, 40, 20000)]


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS)
@pytest.mark.parametrize("name", ["k_scales", "k_biases"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_key_is_not_dropped(gpu, Hq, Hkv, M, past, name, bad, sign):
    """An infinite scale or bias of a key, against queries of either sign: all
    outputs of the queries that see it and all weights of its kv head are not
    finite, whichever infinity the products give; the others keep their bits."""
    q = sign * queries(M, Hq, M).abs()
    out, w = [], []
    at = past + M // 2
    for spoil in (False, True):
        cache = random_cache(4, Hkv, past + M, past + M)
        cache.k[0, at, 8:] = 0x77777777  # (a nibble of 0 would make NaN of an infinite scale)
        if spoil:
            getattr(cache, name)[0, at, 1] = bad
        w.append(torch.zeros(Hkv, past + M, device="cuda"))
        out.append(bmx.attention_kv4(q, cache, past, weights=w[-1]).view(M, Hkv, Hq // Hkv, D))
    sees = M // 2
    assert not torch.isfinite(out[1][sees:, 0]).any() and not torch.isfinite(w[1][0]).any()
    assert torch.equal(out[1][:sees], out[0][:sees])
    assert torch.equal(out[1][:, 1:], out[0][:, 1:]) and torch.equal(w[1][1:], w[0][1:])


# calls whose waves take many rows each: one token, few rows, more, tiles of 64, of 256
LONG = [(8, 2, 1, 9000), (16, 2, 1, 9000), (4, 1, 1, 131071), (8, 2, 40, 9000), (64, 8, 130, 4500), (32, 8, 1024, 1000)]


@pytest.mark.parametrize("Hq,Hkv,M,past", LONG)
@pytest.mark.parametrize("kind", ["flat", "rising"])
def test_largest_values_over_many_rows(gpu, Hq, Hkv, M, past, kind):
    """Values of one sign up to 2^120, all rows weighing alike, or the weights
    rising by 2^60 along the context: the sums stay in range."""
    cache = random_cache(2, Hkv, past + M, past + M)
    g = torch.Generator().manual_seed(past)
    cache.v_scales.copy_(2.0 ** 115 * (1 + torch.rand(Hkv, past + M, 2, generator=g)))
    cache.v_biases.fill_(2.0 ** 119)
    if kind == "flat":
        check(bmx.attention_kv4, queries(M, Hq, M), cache, past, scale=0.0)
        return
    cache.k_scales.zero_()
    cache.k_biases.copy_((60 * math.log(2) * torch.arange(past + M) / (past + M))[:, None].expand(Hkv, -1, 2))
    q = torch.full((Hq, M, D), 1 / D, dtype=torch.bfloat16, device="cuda")  # scores: the keys' biases
    check(bmx.attention_kv4, q, cache, past, scale=1.0)


def scaled_cache(Hkv, rows, f):
    """Random rows whose values are multiplied by f, [rows, 2] per group."""
    cache = random_cache(2, Hkv, rows, rows)
    cache.v_scales.mul_(f.cuda())
    cache.v_biases.mul_(f.cuda())
    return cache


# ... and keys split over the grid next to few rows, short contexts
SPANS = KERNELS + [(32, 8, 512, 2000), (16, 1, 64, 20001), (64, 64, 200, 0), (32, 8, 70, 0)]


@pytest.mark.parametrize("Hq,Hkv,M,past", SPANS)
@pytest.mark.parametrize("kind", ["ends", "zeros", "late", "early", "steps", "once", "edge"])
def test_values_of_one_context_far_apart(gpu, Hq, Hkv, M, past, kind):
    """Rows of 2^-60 next to rows of 2^100, zero rows next to 2^71, one after
    the other, and at the end of what the tile kernel does in one pass: what a
    row weighs does not depend on its values."""
    n = past + M
    g = torch.Generator().manual_seed(M)
    half = torch.rand(n, 1, generator=g) < 0.5
    at = torch.arange(n)[:, None]
    f = {"ends": torch.where(half, 2.0 ** -60, 2.0 ** 100), "zeros": torch.where(half, 0.0, 2.0 ** 71),
         "late": torch.where(at < n // 2, 2.0 ** -60, 2.0 ** 100), "early": torch.where(at < n // 2, 2.0 ** 100, 2.0 ** -60),
         "steps": 2.0 ** (-60 + 160 * at / n).floor(), "once": torch.where(at == n - M // 2 - 1, 2.0 ** 100, 1.0),
         "edge": torch.where(half, 0.0, 2.0 ** (30 + 2 * torch.rand(n, 1, generator=g)).round())}[kind]
    check(bmx.attention_kv4, queries(M, Hq, M), scaled_cache(Hkv, n, f.expand(n, 2)), past)


@pytest.mark.parametrize("Hq,Hkv,M,past", [k for k in SPANS if k[2] > 30])
def test_rows_before_a_large_value_keep_their_bits(gpu, Hq, Hkv, M, past):
    """One row of 2^100 in the middle of the new tokens: the queries before it
    are computed as without it, the others to their bounds."""
    n, at = past + M, past + M // 2
    f = torch.ones(n, 2)
    q = queries(M, Hq, M)
    clean = bmx.attention_kv4(q, scaled_cache(Hkv, n, f), past)
    f[at] = 2.0 ** 100
    got = check(bmx.attention_kv4, q, scaled_cache(Hkv, n, f), past)
    assert torch.equal(got[:M // 2], clean[:M // 2])


@pytest.mark.parametrize("Hq,Hkv,M,past", SPANS)
@pytest.mark.parametrize("kind", ["2^-7", "2^-28", "2^-40", "2^60", "zero", "swapped", "outliers", "both"])
def test_groups_far_apart(gpu, Hq, Hkv, M, past, kind):
    """A group much smaller than the other of its row, everywhere, from row to
    row in turns, or next to a few rows whose other group is large: each
    group counts by itself, and keeps its precision."""
    n = past + M
    g = torch.Generator().manual_seed(M + 1)
    some = torch.rand(n, 1, generator=g)
    pair = lambda a, b: torch.tensor([[a, b]])
    f = {"2^-7": pair(2.0 ** -7, 1.0), "2^-28": pair(2.0 ** -28, 1.0), "2^-40": pair(1.0, 2.0 ** -40),
         "2^60": pair(1.0, 2.0 ** 60), "zero": pair(0.0, 1.0),
         "swapped": torch.where(some < 0.5, pair(2.0 ** -30, 1.0), pair(1.0, 2.0 ** -30)),
         "outliers": torch.where(some < 0.05, pair(2.0 ** 35, 1.0), pair(1.0, 1.0)),
         "both": torch.where(some < 0.5, pair(2.0 ** 100, 2.0 ** 20), pair(2.0 ** -20, 2.0 ** 60))}[kind]
    check(bmx.attention_kv4, queries(M, Hq, M), scaled_cache(Hkv, n, f.expand(n, 2)), past)


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("name", ["v_scales", "v_biases"])
def test_a_row_of_bad_values_leaves_the_weights_alone(gpu, Hq, Hkv, M, past, name, bad):
    """Both groups of a row's values not finite: the outputs of the queries that
    see it are not, the weights do not change, nor do the other queries' bits."""
    at, q = past + M // 2, queries(M, Hq, M)
    out, w = [], []
    for spoil in (False, True):
        cache = random_cache(4, Hkv, past + M, past + M)
        cache.v[0, at] = 0x77777777
        if spoil:
            getattr(cache, name)[0, at] = bad
        w.append(torch.zeros(Hkv, past + M, device="cuda"))
        out.append(bmx.attention_kv4(q, cache, past, weights=w[-1]).view(M, Hkv, Hq // Hkv, D))
    assert not torch.isfinite(out[1][M // 2:, 0]).any()
    assert torch.equal(out[1][:M // 2], out[0][:M // 2]) and torch.equal(out[1][:, 1:], out[0][:, 1:])
    # (the weights' sum is added up with another exponent for that row: a few roundings)
    assert ((w[1] - w[0]).abs() <= 16 * 2.0 ** -24 * w[0]).all()
