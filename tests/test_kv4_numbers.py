"""Row numbers of the 4-bit KV cache's Python calls that do not fit a C int:
refused before the library is called, never cut to their low 32 bits.  No GPU:
the tensors live on the CPU, and any call into the library fails the test."""
from types import SimpleNamespace

import pytest
import torch

import bmx

BIG = [2 ** 32, 2 ** 32 + 7, 2 ** 33 + 3, -2 ** 32 + 7, 2 ** 31, 2 ** 64 + 7]


@pytest.fixture
def cache(monkeypatch):
    """A cache of 2 kv heads and 50 rows, on the CPU."""
    def reached(name, *args):
        raise AssertionError(f"{name} was called")

    bmx._torch()
    monkeypatch.setattr(bmx, "call", reached)
    monkeypatch.setattr(bmx, "_elsewhere", lambda device: False)
    monkeypatch.setattr(bmx, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(bmx, "_stream", lambda stream=None: 0)
    return SimpleNamespace(device=torch.device("cpu"), n_kv_heads=2, capacity=50,
                           k=torch.zeros(2, 50, 16, dtype=torch.int32), k_scales=torch.zeros(2, 50, 2, dtype=torch.bfloat16),
                           _ref=0)


def code(f, *a, **kw):
    with pytest.raises(bmx.BmxError) as e:
        f(*a, **kw)
    return e.value.code


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("n", BIG)
def test_rows(cache, n):
    unit = bf16(128)
    for M in (0, 1, 3):
        assert code(bmx.kv4_write, bf16(2, M, 128), bf16(2, M, 128), cache, n) == bmx.BMX_E_KV_CAPACITY
        assert code(bmx.qk_norm_rope_kv4, bf16(M, 512), bf16(M, 256), bf16(M, 256), unit, unit, cache,
                    n) == bmx.BMX_E_KV_CAPACITY
    assert code(bmx.kv4_read, cache, n, n + 1) == bmx.BMX_E_KV_CAPACITY
    for M in (0, 1):
        assert code(bmx.attention_kv4, bf16(4, M, 128), cache, n) == bmx.BMX_E_KV_CAPACITY


@pytest.mark.parametrize("n", BIG)
def test_evict(cache, n):
    w = torch.zeros(2, 50)
    assert code(bmx.kv4_evict, cache, w, n, 20) in (bmx.BMX_E_KV_CAPACITY, bmx.BMX_E_SHAPE)
    assert code(bmx.kv4_evict, cache, w, 40, n) in (bmx.BMX_E_KV_CAPACITY, bmx.BMX_E_SHAPE)
    assert code(bmx.kv4_evict, cache, w, 40, 20, sink=n) == bmx.BMX_E_SHAPE
    assert code(bmx.kv4_evict, cache, w, 40, 20, recent=n) == bmx.BMX_E_SHAPE


@pytest.mark.parametrize("n", BIG)
def test_position_and_workspace(cache, n):
    unit = bf16(128)
    if n < 0 or n >= 2 ** 63:  # (the library takes 64 bits)
        assert code(bmx.qk_norm_rope_kv4, bf16(1, 512), bf16(1, 256), bf16(1, 256), unit, unit, cache, 0,
                    position=n) == bmx.BMX_E_ARG
    for a in ((n, 2, 1, 10), (4, n, 1, 10), (4, 2, n, 10), (4, 2, 1, n)):
        assert code(bmx.attention_kv4_workspace, *a, device="cpu") == bmx.BMX_E_SHAPE
