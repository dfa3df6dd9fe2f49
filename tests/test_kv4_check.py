"""The checks of attention over the 4-bit KV cache reject what is wrong: plain
attention on the CPU passes them, and fails with each of these mistakes
planted in it."""
import math
from types import SimpleNamespace

import pytest
import torch

from _kv4_check import D, check, values, visible


def cache_of(seed, Hkv, rows):
    g = torch.Generator().manual_seed(seed)
    c = SimpleNamespace(n_kv_heads=Hkv, capacity=rows)
    for name, mid in (("k", 0.5), ("v", 0.0)):
        s = (0.05 + 0.4 * torch.rand(Hkv, rows, 2, generator=g)).to(torch.bfloat16)
        setattr(c, name, torch.randint(-2 ** 31, 2 ** 31, (Hkv, rows, 16), generator=g, dtype=torch.int64).to(torch.int32))
        setattr(c, name + "_scales", s)
        setattr(c, name + "_biases", (mid - 7.5 * s.float() + 0.3 * torch.randn(Hkv, rows, 2, generator=g)).to(torch.bfloat16))
    return c


def plain(mistake=None):
    """attention_kv4 in float32, P and V rounded to bf16 as the coarsest kernel does, with a mistake."""
    def call(q, cache, past, scale, weights):
        Hq, M, _ = q.shape
        rep, L = Hq // cache.n_kv_heads, past + M
        heads = []
        for h in range(cache.n_kv_heads):
            k = values(cache.k[h, :L], cache.k_scales[h, :L], cache.k_biases[h, :L]).float()
            v = values(cache.v[h, :L], cache.v_scales[h, :L], cache.v_biases[h, :L]).to(torch.bfloat16).float()
            see = visible(rep, M, past, q.device)
            if mistake == "mask":
                see[torch.arange(rep * M), past + torch.arange(rep * M) % M] = False  # a query misses its own row
            s = torch.mm(q[h * rep:(h + 1) * rep].float().reshape(rep * M, D), k.t()) * scale
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            if mistake == "key":
                p[:, L // 2] = 0
            out = torch.mm(p.to(torch.bfloat16).float(), v)
            if mistake == "row":
                out[(h + 1) * rep * M // (cache.n_kv_heads + 1)] = 0
            if mistake == "element":
                out[-1, out[-1].abs().argmax()] *= 1.05
            if mistake == "group":
                out[0, 64:] *= 1.04
            if weights is not None:
                weights[h, :L] += p.sum(0)
                if mistake == "weight":
                    weights[h, L // 3] -= p[-1, L // 3]
            heads.append(out.reshape(rep, M, D))
        return torch.cat(heads).transpose(0, 1).reshape(M, Hq * D).to(torch.bfloat16)

    return call


SHAPES = [(4, 2, 1, 200), (8, 2, 17, 50), (4, 1, 40, 300)]


def inputs(Hq, Hkv, M, past):
    g = torch.Generator().manual_seed(M)
    return (1.5 * torch.randn(Hq, M, D, generator=g)).to(torch.bfloat16), cache_of(past, Hkv, past + M)


@pytest.mark.parametrize("Hq,Hkv,M,past", SHAPES)
def test_plain_attention_passes(Hq, Hkv, M, past):
    check(plain(), *inputs(Hq, Hkv, M, past), past)


@pytest.mark.parametrize("Hq,Hkv,M,past", SHAPES)
@pytest.mark.parametrize("mistake", ["mask", "key", "row", "element", "group", "weight"])
def test_a_mistake_fails(Hq, Hkv, M, past, mistake):
    with pytest.raises(AssertionError):
        check(plain(mistake), *inputs(Hq, Hkv, M, past), past)
