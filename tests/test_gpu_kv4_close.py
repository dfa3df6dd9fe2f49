"""Attention over the 4-bit KV cache and its weights, held to bounds that one
wrong row, group or key breaks (test_kv4_check.py plants such mistakes)."""
import pytest
import torch

import bmx
from _kv4_check import D, check
from test_gpu_kv4 import HEADS, queries, random_cache
from test_gpu_kv4_wide import WIDE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv", HEADS)
@pytest.mark.parametrize("past", [0, 1, 15, 31, 32, 63, 64, 127, 255, 256, 300, 1027])
def test_one_token(gpu, Hq, Hkv, past):
    check(bmx.attention_kv4, queries(past + 1, Hq, 1), random_cache(past, Hkv, past + 40, past + 1), past)


@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (64, 8), (6, 2), (4, 4), (24, 1), (5, 5)])
@pytest.mark.parametrize("M,past", [(2, 0), (2, 31), (5, 1336), (8, 511), (9, 30), (16, 0), (17, 100), (31, 0), (33, 70),
                                    (65, 0), (130, 201)])
def test_many_tokens(gpu, Hq, Hkv, M, past):
    check(bmx.attention_kv4, queries(M, Hq, M), random_cache(M, Hkv, past + M + 5, past + M), past)


@pytest.mark.parametrize("Hq,Hkv,M,past", WIDE + [(32, 8, 1, 4095), (4, 1, 1, 20001), (8, 2, 3, 9999), (4, 1, 40, 5000)])
def test_long_and_wide(gpu, Hq, Hkv, M, past):
    check(bmx.attention_kv4, queries(M, Hq, M), random_cache(M + past, Hkv, past + M + 3, past + M), past)


@pytest.mark.parametrize("Hq,Hkv,M,past", [(8, 2, 1, 599), (8, 2, 3, 500), (8, 2, 40, 500), (32, 8, 300, 500)])
@pytest.mark.parametrize("std", [15.0, 60.0])
def test_concentrated(gpu, Hq, Hkv, M, past, std):
    """Scores of tens and hundreds: a few keys take everything, the rest underflow."""
    check(bmx.attention_kv4, queries(1, Hq, M, std=std), random_cache(8, Hkv, past + M, past + M), past)


@pytest.mark.parametrize("Hq,Hkv,M,past", [(32, 8, 1, 5000), (32, 8, 9, 2000), (32, 8, 300, 700)])
def test_written_rows(gpu, Hq, Hkv, M, past):
    """Rows as kv4_write leaves them, of keys with large channels."""
    g = torch.Generator().manual_seed(past)
    n = past + M
    k = torch.randn(Hkv, n, D, generator=g) * (0.5 + torch.rand(Hkv, 1, D, generator=g)) + 0.7 * torch.randn(Hkv, 1, D, generator=g)
    v = torch.randn(Hkv, n, D, generator=g)
    cache = bmx.Kv4Cache.empty(Hkv, n)
    bmx.kv4_write(k.to(torch.bfloat16).cuda(), v.to(torch.bfloat16).cuda(), cache, 0)
    check(bmx.attention_kv4, queries(M, Hq, M), cache, past)
