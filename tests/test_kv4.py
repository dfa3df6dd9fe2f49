"""Refusals of the 4-bit KV cache's entry points: every bad argument returns
its code from the host checks (no GPU work is issued by any call here)."""
import ctypes

import pytest

import bmx

P = 0x10000  # a plausible device address; never dereferenced


class Kv4(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "k_scales", "k_biases", "v", "v_scales", "v_biases")] + [
        (n, ctypes.c_int) for n in ("n_kv_heads", "capacity", "group_size", "bits")]


def kv4(**kw):
    a = dict(k=P, k_scales=2 * P, k_biases=3 * P, v=4 * P, v_scales=5 * P, v_biases=6 * P, n_kv_heads=2, capacity=100,
             group_size=64, bits=4)
    a.update(kw)
    return Kv4(*[a[n] for n, _ in Kv4._fields_])


def entry_points(c):
    """One valid-looking call of each entry point on cache struct c (None: a null pointer)."""
    lib, r = bmx.load(), None if c is None else ctypes.pointer(c)  # (the calls below keep c alive)
    big = 1 << 40
    return {
        "write": lambda **k: lib.bmx_kv4_write(*[k.get(n, d) for n, d in (
            ("kp", P), ("khs", 128), ("krs", 256), ("vp", P), ("vhs", 128), ("vrs", 256))], r, k.get("M", 4),
            k.get("D", 128), k.get("offset", 0), None),
        "read": lambda **k: lib.bmx_kv4_read(r, k.get("kp", P), k.get("vp", P), k.get("M", 4), k.get("D", 128),
                                             k.get("offset", 0), None),
        "rope": lambda **k: lib.bmx_qk_norm_rope_kv4(k.get("q", P), k.get("kp", P), k.get("vp", P), P, P,
                                                     k.get("out", P), r, k.get("M", 4), k.get("Hq", 4),
                                                     k.get("D", 128), k.get("offset", 0), k.get("position", 0), 1e-6,
                                                     1e6, None),
        "attention": lambda **k: lib.bmx_attention_gqa_kv4(k.get("q", P), r, k.get("out", P), k.get("weights", None),
                                                           k.get("Hq", 4), k.get("M", 4), k.get("D", 128),
                                                           k.get("offset", 0), 0.1, k.get("ws", P),
                                                           k.get("wsb", big), None),
        "evict": lambda **k: lib.bmx_kv4_evict(r, k.get("w", 7 * P), r if "into" not in k else k["into"],
                                               k.get("w_into", 7 * P), k.get("kept", 9 * P), k.get("length", 50),
                                               k.get("budget", 20), k.get("sink", 4), k.get("recent", 8),
                                               k.get("D", 128), k.get("ws"), k.get("wsb", 0), None),
    }


ALL = ("write", "read", "rope", "attention", "evict")


@pytest.mark.parametrize("op", ALL)
def test_cache_struct_refusals(op):
    assert entry_points(None)[op]() == bmx.BMX_E_ARG
    for name in ("k", "k_scales", "k_biases", "v", "v_scales", "v_biases"):
        assert entry_points(kv4(**{name: None}))[op]() == bmx.BMX_E_ARG
        assert entry_points(kv4(**{name: P + 8}))[op]() == bmx.BMX_E_ALIGN
    assert entry_points(kv4(bits=8))[op]() == bmx.BMX_E_UNSUPPORTED
    assert entry_points(kv4(group_size=32))[op]() == bmx.BMX_E_UNSUPPORTED
    assert entry_points(kv4())[op](D=64) == bmx.BMX_E_UNSUPPORTED
    assert entry_points(kv4(n_kv_heads=0))[op]() == bmx.BMX_E_SHAPE
    assert entry_points(kv4(capacity=0))[op]() == bmx.BMX_E_SHAPE
    assert entry_points(kv4(capacity=16776961))[op]() == bmx.BMX_E_SHAPE


@pytest.mark.parametrize("op", ("write", "read", "rope", "attention"))
def test_row_range_refusals(op):
    f = entry_points(kv4())[op]
    assert f(offset=97) == bmx.BMX_E_KV_CAPACITY
    assert f(offset=-1) == bmx.BMX_E_KV_CAPACITY
    assert f(offset=2 ** 31 - 1) == bmx.BMX_E_KV_CAPACITY
    assert f(M=101) == bmx.BMX_E_KV_CAPACITY
    assert f(M=-1) == bmx.BMX_E_SHAPE
    assert f(M=0) == 0  # nothing to do
    assert f(M=0, offset=100) == 0


def test_write_refusals():
    f = entry_points(kv4())["write"]
    assert f(kp=None) == bmx.BMX_E_ARG and f(vp=None) == bmx.BMX_E_ARG
    assert f(kp=P + 2) == bmx.BMX_E_ALIGN and f(vp=P + 8) == bmx.BMX_E_ALIGN
    for s in ("khs", "krs", "vhs", "vrs"):
        assert f(**{s: 4}) == bmx.BMX_E_ALIGN
        assert f(**{s: -128}) == bmx.BMX_E_SHAPE


def test_read_refusals():
    f = entry_points(kv4())["read"]
    assert f(kp=None) == bmx.BMX_E_ARG and f(vp=None) == bmx.BMX_E_ARG
    assert f(kp=P + 2) == bmx.BMX_E_ALIGN and f(vp=P + 8) == bmx.BMX_E_ALIGN


def test_rope_refusals():
    f = entry_points(kv4())["rope"]
    for n in ("q", "kp", "vp", "out"):
        assert f(**{n: None}) == bmx.BMX_E_ARG
    assert f(position=-1) == bmx.BMX_E_ARG
    assert f(Hq=0) == bmx.BMX_E_SHAPE


def test_attention_refusals():
    lib, f = bmx.load(), entry_points(kv4())["attention"]
    for n in ("q", "out", "ws"):
        assert f(**{n: None}) == bmx.BMX_E_ARG
        assert f(**{n: P + 8}) == bmx.BMX_E_ALIGN
    assert f(weights=P + 4) == bmx.BMX_E_ALIGN
    assert f(Hq=5) == bmx.BMX_E_SHAPE and f(Hq=0) == bmx.BMX_E_SHAPE
    need = lib.bmx_attention_kv4_workspace_bytes(4, 2, 4, 4, 0)
    assert need >= bmx.KV4_COUNTER_BYTES
    assert f(wsb=need - 1) == bmx.BMX_E_ARG and "workspace" in bmx.last_error()
    weigh = lib.bmx_attention_kv4_workspace_bytes(4, 2, 4, 4, 1)
    assert weigh >= need + 4 * 4 * 4  # the logarithms of the softmax sums
    assert f(wsb=weigh - 1, weights=P) == bmx.BMX_E_ARG


def test_attention_workspace_query_refuses_what_the_call_refuses():
    q = bmx.load().bmx_attention_kv4_workspace_bytes
    assert q(4, 3, 1, 10, 0) == 0 and q(0, 1, 1, 10, 0) == 0 and q(4, 0, 1, 10, 0) == 0
    assert q(4, 2, 0, 10, 0) == 0 and q(4, 2, 11, 10, 0) == 0 and q(4, 2, 1, 16776961, 0) == 0
    assert q(4, 2, -5, 10, 0) == 0 and q(4, 2, 1, -1, 0) == 0
    assert q(4, 2, 1, 16776960, 1) > 0
    assert q(65535, 1, 1 << 20, 16776960, 0) == 0  # more query rows than one call takes


def test_attention_workspace_grows_with_the_call():
    """One sized for the largest call serves the smaller ones."""
    q = bmx.load().bmx_attention_kv4_workspace_bytes
    for hq, hkv in ((32, 8), (6, 2), (300, 150)):
        for weigh in (0, 1):
            last = 0
            for M in (1, 2, 3, 8, 15, 64, 300, 1000, 5000):
                row = [q(hq, hkv, M, L, weigh) for L in (5000, 5001, 9000, 20000, 200000)]
                assert row == sorted(row) and row[0] >= last
                last = row[0]
            assert q(hq, hkv, 8, 9000, 1) > q(hq, hkv, 8, 9000, 0)


def test_evict_refusals():
    f = entry_points(kv4())["evict"]
    for n in ("w", "w_into", "kept"):
        assert f(**{n: None}) == bmx.BMX_E_ARG
        assert f(**{n: P + 4}) == bmx.BMX_E_ALIGN
    assert f(length=101) == bmx.BMX_E_KV_CAPACITY
    assert f(budget=51) == bmx.BMX_E_SHAPE  # more than there is
    assert f(budget=0) == bmx.BMX_E_SHAPE and f(budget=-3) == bmx.BMX_E_SHAPE
    assert f(sink=-1) == bmx.BMX_E_SHAPE and f(recent=-1) == bmx.BMX_E_SHAPE
    assert f(sink=10, recent=11) == bmx.BMX_E_SHAPE
    assert f(sink=2 ** 31 - 1, recent=2 ** 31 - 1) == bmx.BMX_E_SHAPE
    assert f(into=None) == bmx.BMX_E_ARG
    far = {n: (20 + i) * P for i, n in enumerate(("k", "k_scales", "k_biases", "v", "v_scales", "v_biases"))}
    other = kv4(**far)
    o = ctypes.pointer(other)
    assert f(into=o) == bmx.BMX_E_ARG  # another cache, the same weights
    assert f(w_into=8 * P) == bmx.BMX_E_ARG  # the same cache, other weights
    small = kv4(capacity=19, **far)
    assert f(into=ctypes.pointer(small), w_into=8 * P) == bmx.BMX_E_KV_CAPACITY
    heads = kv4(n_kv_heads=3, **far)
    assert f(into=ctypes.pointer(heads), w_into=8 * P) == bmx.BMX_E_SHAPE


def test_evict_workspace():
    q = bmx.load().bmx_kv4_evict_workspace_bytes
    assert q(8, 8192) == 0 and q(8, 8193) > 0 and q(0, 20000) == 0 and q(8, 0) == 0 and q(8, 16776961) == 0
    sizes = [q(8, n) for n in (8193, 40000, 131072, 1 << 20, 16776960)]
    assert sizes == sorted(sizes)
    f = entry_points(kv4(capacity=20000))["evict"]
    need = q(2, 20000)
    assert f(length=20000) == bmx.BMX_E_ARG and "workspace" in bmx.last_error()
    assert f(length=20000, ws=P, wsb=need - 1) == bmx.BMX_E_ARG
    assert f(length=20000, ws=P + 8, wsb=need) == bmx.BMX_E_ALIGN


def test_python_refusals_need_no_gpu():
    import torch

    t = [torch.zeros(2, 8, 16, dtype=torch.int32)] + [torch.zeros(2, 8, 2, dtype=torch.bfloat16)] * 2
    with pytest.raises(bmx.BmxError) as e:
        bmx.Kv4Cache(*t, *t)
    assert e.value.code == bmx.BMX_E_ARG and "GPU" in str(e.value)
    with pytest.raises(bmx.BmxError) as e:
        bmx.attention_kv4_workspace(4, 3, 1, 10)
    assert e.value.code == bmx.BMX_E_SHAPE


def test_attention_refuses_out_over_q():
    f = entry_points(kv4())["attention"]
    assert f(q=P, out=P) == bmx.BMX_E_ARG and f(q=P, out=P + 4096 - 16) == bmx.BMX_E_ARG
    assert "overlaps" in bmx.last_error()


@pytest.mark.parametrize("shared", ["k", "k_scales", "k_biases", "v", "v_scales", "v_biases"])
def test_evict_refuses_a_cache_over_itself(shared):
    """`into` that shares one array, or the end of one, with the cache."""
    far = dict(k=11 * P, k_scales=12 * P, k_biases=13 * P, v=14 * P, v_scales=15 * P, v_biases=16 * P)
    c = kv4()
    f = entry_points(c)["evict"]
    for at in (getattr(c, shared), getattr(c, shared) + 784):
        into = kv4(**{**far, shared: at})
        assert f(into=ctypes.pointer(into), w_into=17 * P) == bmx.BMX_E_ARG
        assert "overlaps" in bmx.last_error()
    into = kv4(**far)
    assert f(into=ctypes.pointer(into), w_into=7 * P + 784) == bmx.BMX_E_ARG


def test_rope_refuses_positions_past_fp32():
    """The rotation's angle takes the position as an fp32 number: beyond 2^24 neighbours would share one."""
    f = entry_points(kv4())["rope"]
    for position in (2 ** 24 - 2, 2 ** 24 + 1, 2 ** 31, 2 ** 40, 2 ** 63 - 1):
        assert f(position=position) == bmx.BMX_E_ARG and "position" in bmx.last_error()


def test_attention_row_range_does_not_wrap():
    f = entry_points(kv4())["attention"]
    assert f(M=2 ** 31 - 1, offset=100) == bmx.BMX_E_KV_CAPACITY
    assert f(M=2, offset=2 ** 31 - 1) == bmx.BMX_E_KV_CAPACITY
