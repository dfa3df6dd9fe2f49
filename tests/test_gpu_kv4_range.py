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
