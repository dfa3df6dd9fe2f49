"""Refusals of the paged KV cache's entry points: every bad argument returns its
code from the host checks (no GPU work is issued by any call here)."""
import ctypes

import pytest

import bmx

P = 0x10000000  # a plausible device address; never dereferenced


def kv(**kw):
    a = dict(k=P, v=2 * P, n_pages=10, n_kv_heads=2, page_size=16)
    a.update(kw)
    return bmx._PagedKvStruct(*[a[n] for n, _ in bmx._PagedKvStruct._fields_])


def batch(**kw):
    a = dict(starts=3 * P, lens=4 * P, pages=5 * P, n_seqs=3, max_pages=4, tokens=6, max_new=3)
    a.update(kw)
    return bmx._BatchStruct(*[a[n] for n, _ in bmx._BatchStruct._fields_])


def append(c, b, **k):
    return bmx.load().bmx_qk_norm_rope_paged(*[k.get(n, d) for n, d in (
        ("q", 6 * P), ("kp", 7 * P), ("vp", 8 * P), ("qn", 9 * P), ("kn", 10 * P), ("out", 11 * P))],
        c and ctypes.byref(c), b and ctypes.byref(b), k.get("Hq", 4), k.get("D", 128), 1e-6, 1e6, None)


def attend(c, b, **k):
    return bmx.load().bmx_attention_paged(k.get("q", 6 * P), c and ctypes.byref(c), b and ctypes.byref(b),
                                          k.get("out", 11 * P), k.get("Hq", 4), k.get("D", 128), k.get("shared", 0), 0.1,
                                          k.get("ws", 12 * P), k.get("wsb", 1 << 40), None)


@pytest.mark.parametrize("f", [append, attend])
def test_struct_refusals(f):
    assert f(None, batch()) == bmx.BMX_E_ARG and f(kv(), None) == bmx.BMX_E_ARG
    for n in ("k", "v"):
        assert f(kv(**{n: None}), batch()) == bmx.BMX_E_ARG
        assert f(kv(**{n: P + 8}), batch()) == bmx.BMX_E_ALIGN
    for n in ("starts", "lens", "pages"):
        assert f(kv(), batch(**{n: None})) == bmx.BMX_E_ARG
        assert f(kv(), batch(**{n: P + 2})) == bmx.BMX_E_ALIGN
    for size in (0, -16, 8, 24, 100, 8192, -2 ** 31):
        assert f(kv(page_size=size), batch()) == bmx.BMX_E_UNSUPPORTED and "page_size" in bmx.last_error()
    assert f(kv(), batch(), D=64) == bmx.BMX_E_UNSUPPORTED
    for n in ("n_pages", "n_kv_heads"):
        for v in (0, -1):
            assert f(kv(**{n: v}), batch()) == bmx.BMX_E_SHAPE
    assert f(kv(n_kv_heads=1025), batch(), Hq=1025) == bmx.BMX_E_SHAPE
    for heads in (0, -2, 5, 65536):
        assert f(kv(), batch(), Hq=heads) == bmx.BMX_E_SHAPE
    assert f(kv(), batch(n_seqs=-1)) == bmx.BMX_E_SHAPE and f(kv(), batch(n_seqs=4097)) == bmx.BMX_E_SHAPE
    assert f(kv(), batch(max_pages=0)) == bmx.BMX_E_SHAPE
    assert f(kv(), batch(max_pages=(1 << 20) + 1)) == bmx.BMX_E_SHAPE  # 2^24 rows
    assert f(kv(page_size=4096), batch(max_pages=4097)) == bmx.BMX_E_SHAPE
    assert f(kv(), batch(tokens=-1)) == bmx.BMX_E_SHAPE
    assert f(kv(), batch(max_new=0)) == bmx.BMX_E_SHAPE and f(kv(), batch(max_new=7)) == bmx.BMX_E_SHAPE
    assert f(kv(), batch(tokens=1 << 30, max_new=1)) == bmx.BMX_E_SHAPE
    # nothing to do
    assert f(kv(), batch(tokens=0, max_new=0)) == 0 and f(kv(), batch(n_seqs=0)) == 0


def test_append_refusals():
    for n in ("q", "kp", "vp", "qn", "kn", "out"):
        assert append(kv(), batch(), **{n: None}) == bmx.BMX_E_ARG
        assert append(kv(), batch(), **{n: P + 8}) == bmx.BMX_E_ALIGN
    for n, rows in (("q", 4), ("kp", 2), ("vp", 2)):  # q_out over an input, or over its end
        at = {"q": 6, "kp": 7, "vp": 8}[n] * P
        for out in (at, at + 6 * rows * 256 - 16, at - 6 * 4 * 256 + 16):
            assert append(kv(), batch(), out=out) == bmx.BMX_E_ARG and "overlaps" in bmx.last_error()


def test_attention_refusals():
    for n in ("q", "out", "ws"):
        assert attend(kv(), batch(), **{n: None}) == bmx.BMX_E_ARG
        assert attend(kv(), batch(), **{n: P + 8}) == bmx.BMX_E_ALIGN
    for out in (6 * P, 6 * P + 6 * 4 * 256 - 16):
        assert attend(kv(), batch(), out=out) == bmx.BMX_E_ARG and "overlaps" in bmx.last_error()
    for shared in (-16, 8, 17, 80):
        assert attend(kv(), batch(), shared=shared) == bmx.BMX_E_ARG and "shared" in bmx.last_error()
    for shared in (0, 32):
        for max_new in (3, 6):
            for heads in (4, 64):
                need = bmx.load().bmx_attention_paged_workspace_bytes(heads, 2, 6, 3, max_new, shared)
                assert need > 0
                rc = attend(kv(), batch(max_new=max_new), Hq=heads, shared=shared, wsb=need - 1, q=20 * P, out=21 * P)
                assert rc == bmx.BMX_E_ARG and "workspace" in bmx.last_error()
    # more blocks of keys than an int counts
    assert attend(kv(n_kv_heads=1024), batch(n_seqs=4096, max_pages=1 << 20, tokens=4096, max_new=1), Hq=1024,
                  q=20 * P, out=40 * P) == bmx.BMX_E_SHAPE
    # ... and of prompts, by all their tiles: 2^20 of 256 rows, 2^18 blocks each
    assert attend(kv(n_kv_heads=1), batch(n_seqs=1, max_pages=1 << 20, tokens=1 << 23, max_new=1 << 23), Hq=32, q=1 << 40,
                  out=1 << 42, wsb=1 << 45) == bmx.BMX_E_SHAPE and "too many" in bmx.last_error()


def test_workspace_query_refuses_what_the_call_refuses():
    q = bmx.load().bmx_attention_paged_workspace_bytes
    assert q(4, 2, 6, 3, 3, 0) > 0
    for bad in ((5, 2, 6, 3, 3), (0, 2, 6, 3, 3), (4, 0, 6, 3, 3), (4, 2, 0, 3, 3), (4, 2, 6, 0, 3), (4, 2, 6, 4097, 3),
                (4, 2, 6, 3, 0), (4, 2, 6, 3, 7), (4, 2, 1 << 30, 3, 1), (1025, 1025, 6, 3, 3)):
        assert q(*bad, 0) == 0 and q(*bad, 1) == 0


def test_workspace_grows_with_the_batch():
    """One sized for the largest step serves every smaller one of the same heads."""
    q = bmx.load().bmx_attention_paged_workspace_bytes
    for hq, hkv in ((32, 8), (6, 2), (64, 8), (40, 1)):
        for shared in (0, 1):
            for big in ((4096, 64, 4096), (64, 64, 1), (300, 17, 20)):
                most = q(hq, hkv, *big, shared)
                for tokens in (1, 2, 31, 64, 300, 1000, 4096):
                    for seqs in (1, 3, 17, 64):
                        for new in (1, 2, 5, 16, 17, 64, 300, 4096):
                            if tokens <= big[0] and seqs <= big[1] and new <= min(tokens, big[2]):
                                assert q(hq, hkv, tokens, seqs, new, shared) <= most, (hq, hkv, shared, big, tokens, seqs, new)
                                assert q(hq, hkv, tokens, seqs, new, 0) <= most


def test_workspace_never_shrinks():
    """More tokens, sequences or new tokens of one, and shared rows, need no less."""
    q = bmx.load().bmx_attention_paged_workspace_bytes
    sizes = [1, 2, 7, 60, 96, 97, 191, 192, 193, 384, 385, 1000, 1536, 2900, 6143, 6144, 6145, 12287, 12289]
    for hq, hkv in ((32, 8), (8, 8), (64, 1)):
        for shared in (0, 1):
            for tokens in sizes:
                for seqs in (1, 2, 3, 4, 7, 8, 9, 60, 400):
                    for new in sizes:
                        if new > tokens:
                            continue
                        n = q(hq, hkv, tokens, seqs, new, shared)
                        at = (hq, hkv, tokens, seqs, new, shared)
                        assert q(hq, hkv, tokens + 1, seqs, new, shared) >= n, at
                        assert q(hq, hkv, tokens, seqs + 1, new, shared) >= n, at
                        assert new == tokens or q(hq, hkv, tokens, seqs, new + 1, shared) >= n, at
                        assert q(hq, hkv, tokens, seqs, new, 1) >= n, at


def test_python_refusals_need_no_gpu():
    import torch

    x = torch.zeros(3, 2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(bmx.BmxError) as e:
        bmx.PagedKvCache(x, x)
    assert e.value.code == bmx.BMX_E_ARG and "GPU" in str(e.value)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(bmx.BmxError) as e:
        bmx.PagedBatch(i, i[:2], i[:2].reshape(2, 1), 5)
    assert e.value.code == bmx.BMX_E_ARG and "GPU" in str(e.value)
    with pytest.raises(bmx.BmxError) as e:
        bmx.PagedBatch.of([1], [1, 2], [[0]])
    assert e.value.code == bmx.BMX_E_SHAPE
    for sizes in ((0, 1, 1), (4, 5000, 1), (4, 1, 5), (1 << 40, 1, 1)):
        with pytest.raises(bmx.BmxError) as e:
            bmx.attention_paged_workspace(4, 2, sizes)
        assert e.value.code == bmx.BMX_E_SHAPE
