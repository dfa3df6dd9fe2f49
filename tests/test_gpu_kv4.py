"""The 4-bit KV cache on the GPU: quantizing writes, read-back, attention,
accumulated weights and eviction, against plain implementations (float64 on
the CPU; the quantization itself, which is defined in float32, bit by bit in
numpy's IEEE float32)."""
import math

import numpy as np
import pytest
import torch

import bmx

pytestmark = pytest.mark.gpu

U8 = 2.0 ** -8    # largest relative rounding error of bf16
U24 = 2.0 ** -24  # of fp32
D = 128


# ---------------------------------------------------------------------------
# plain implementations
# ---------------------------------------------------------------------------
def ref_quantise(x):
    """bf16 [..., 128] -> words uint32 [..., 16], scales and biases (bf16 torch) by the documented formula."""
    y = x.float().cpu().numpy().reshape(*x.shape[:-1], 2, 64)
    with np.errstate(all="ignore"):
        lo, hi = y.min(-1), y.max(-1)  # NaN where the group holds one
        rng = (hi - lo).astype(np.float32)
        ok = np.isfinite(rng)
        s = torch.from_numpy(np.where(ok, rng / np.float32(15), np.float32(np.nan)).astype(np.float32)).to(torch.bfloat16)
        b = torch.from_numpy(np.where(ok, lo, np.float32(np.nan)).astype(np.float32)).to(torch.bfloat16)
        sf = s.float().numpy()[..., None]
        n = np.where(sf > 0, np.minimum(np.rint((y - lo[..., None]).astype(np.float32) / sf), 15), 0)
    n = np.nan_to_num(n).astype(np.uint64).reshape(*x.shape[:-1], 16, 8)
    return (n << (4 * np.arange(8, dtype=np.uint64))).sum(-1).astype(np.uint32), s, b


def ref_values(words, s, b):
    """float64 values of cache rows (words int32 torch, on any device)."""
    w = words.cpu().numpy().view(np.uint32)
    n = ((w[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).astype(np.float64).reshape(*w.shape[:-1], 2, 64)
    v = s.cpu().double().numpy()[..., None] * n + b.cpu().double().numpy()[..., None]
    return torch.from_numpy(v.reshape(*w.shape[:-1], D))


def random_cache(seed, heads, capacity, rows=None, stale=True):
    """A cache of random rows; rows past `rows` hold NaN scales and biases (a stale cache's garbage)."""
    g = torch.Generator().manual_seed(seed)
    t = []
    for mid in (0.5, 0.0):
        w = torch.randint(-2 ** 31, 2 ** 31, (heads, capacity, 16), generator=g, dtype=torch.int64).to(torch.int32)
        s = (0.05 + 0.4 * torch.rand(heads, capacity, 2, generator=g)).to(torch.bfloat16)
        b = (mid - 7.5 * s.float() + 0.3 * torch.randn(heads, capacity, 2, generator=g)).to(torch.bfloat16)
        if rows is not None and stale:
            s[:, rows:] = math.nan
            b[:, rows:] = math.inf
        t += [w.cuda(), s.cuda(), b.cuda()]
    return bmx.Kv4Cache(*t)


def ref_attention(q, cache, offset, scale):
    """(out [Hkv, rep, M, 128], P [Hkv, rep, M, L], (q, k, v, visible)) in float64."""
    Hq, M, _ = q.shape
    Hkv, L = cache.n_kv_heads, offset + M
    rep = Hq // Hkv
    k = ref_values(cache.k[:, :L], cache.k_scales[:, :L], cache.k_biases[:, :L])
    v = ref_values(cache.v[:, :L], cache.v_scales[:, :L], cache.v_biases[:, :L])
    qd = q.cpu().double().reshape(Hkv, rep, M, D)
    s = torch.matmul(qd, k[:, None].transpose(-1, -2)) * scale
    see = torch.arange(L)[None] <= offset + torch.arange(M)[:, None]
    s = torch.where(see, s, torch.tensor(-math.inf, dtype=torch.float64))
    p = torch.softmax(s, -1)
    p = torch.where(see, p, torch.zeros((), dtype=torch.float64))
    # a hidden row weighs nothing, whatever it holds
    out = torch.stack([torch.einsum("hrj,hjd->hrd", p[:, :, t, :offset + t + 1], v[:, :offset + t + 1])
                       for t in range(M)], 2)
    return out, p, (qd, k, v, see)


def out_bound(out, p, parts, cache, scale, L):
    """How far a bf16 output may be from `out`: its own rounding; P (times a
    scale) in bf16 against the centred nibbles and the middles, or P in bf16
    against values in bf16 (twice U8 of the weighted magnitudes); keys in bf16
    (a score off by e moves every weight by a factor within exp(2e)), and the
    fp32 arithmetic."""
    qd, k, v, _ = parts
    e = (U8 * scale * torch.matmul(qd.abs(), k.abs()[:, None].transpose(-1, -2))).amax(-1, keepdim=True)  # [.., M, 1]
    mass = torch.matmul(p, v.abs()[:, None].expand(-1, p.shape[1], -1, -1))
    vs = cache.v_scales[:, :L].cpu().double().repeat_interleave(64, -1)
    centred = 7.5 * torch.matmul(p, vs[:, None].expand(-1, p.shape[1], -1, -1))
    return U8 * out.abs() + 1.05 * (2 * e * mass + U8 * (2 * mass + centred)) + 2.0 ** -20 * (mass + centred) + 1e-30


def check_attention(q, cache, offset, scale=None, weights=None, ws=None, stream=None):
    Hq, M, _ = q.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    before = None if weights is None else weights.cpu().double()
    got = bmx.attention_kv4(q, cache, offset, scale=scale, weights=weights, workspace=ws, stream=stream)
    torch.cuda.synchronize()
    out, p, parts = ref_attention(q, cache, offset, scale)
    L, Hkv = offset + M, cache.n_kv_heads
    g = got.cpu().double().reshape(M, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
    bound = out_bound(out, p, parts, cache, scale, L)
    bad = (g - out).abs() > bound
    assert not bad.any() and torch.isfinite(g).all(), (
        f"Hq={Hq} Hkv={Hkv} M={M} offset={offset}: {int(bad.sum())} values off, first {bad.nonzero()[:3].tolist()}, "
        f"worst {float(((g - out).abs() / bound).max()):.3g} of the bound")
    # as a whole: the output's rounding (rms about U8 / 2.4), P's and V's alike
    rel = float((g - out).norm() / out.norm())
    assert rel < 5e-3, rel
    if weights is not None:
        w = weights.cpu().double()
        want = before[:, :L] + p.sum((1, 2))
        # a score's error: 130 fp32 additions of terms of up to |q| s 31 and
        # |q| |b|; the sum over rows and the exponential add a few units more
        qd = parts[0]
        s31 = torch.maximum(31 * cache.k_scales[:, :L].cpu().double().abs().amax(-1),
                            cache.k_biases[:, :L].cpu().double().abs().amax(-1))
        e = 140 * U24 * scale * qd.abs().sum(-1)[..., None] * s31[:, None, None]  # [Hkv, rep, M, L]
        tol = (p * (2 * e.amax(-1, keepdim=True) + 64 * U24)).sum((1, 2)) + 4 * U24 * (before[:, :L].abs() + want)
        assert ((w[:, :L] - want).abs() <= tol + 1e-30).all(), float(((w[:, :L] - want).abs() / tol).max())
        # as a whole: a weight is exp(S - log sum), and S and the logarithm are
        # fp32 numbers of their own size, each the end of a chain whose last
        # few roundings are at that size: a relative error of 2^-24 per unit of
        # |S| and rounding, four of them at most (group 0, group 1, bias, the
        # scale's product), on both sides.  Below |S| = 21 that is under 1e-5
        # together with the sums' own.
        big = float(torch.matmul(qd, parts[1][:, None].transpose(-1, -2)).abs().max()) * abs(scale)
        assert float((w[:, :L] - want).norm() / want.norm()) < max(1e-5, 8 * U24 * big)
        assert torch.equal(w[:, L:], before[:, L:])  # nothing past the last row
    return got


def queries(seed, Hq, M, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(Hq, M, D, generator=g)).to(torch.bfloat16).cuda()


# ---------------------------------------------------------------------------
# write and read
# ---------------------------------------------------------------------------
def check_rows(cache, lo, k, v):
    M = k.shape[1]
    for x, w, s, b in ((k, cache.k, cache.k_scales, cache.k_biases), (v, cache.v, cache.v_scales, cache.v_biases)):
        rw, rs, rb = ref_quantise(x)
        assert np.array_equal(w[:, lo:lo + M].cpu().numpy().view(np.uint32), rw)
        assert torch.equal(s[:, lo:lo + M].cpu().isnan(), rs.isnan()) and torch.equal(b[:, lo:lo + M].cpu().isnan(), rb.isnan())
        assert torch.equal(s[:, lo:lo + M].cpu().float().nan_to_num(9.0), rs.float().nan_to_num(9.0))
        assert torch.equal(b[:, lo:lo + M].cpu().float().nan_to_num(9.0), rb.float().nan_to_num(9.0))
    rk, rv = bmx.kv4_read(cache, lo, lo + M)
    for got, w, s, b in ((rk, cache.k, cache.k_scales, cache.k_biases), (rv, cache.v, cache.v_scales, cache.v_biases)):
        want = ref_values(w[:, lo:lo + M], s[:, lo:lo + M], b[:, lo:lo + M]).float().to(torch.bfloat16)
        assert torch.equal(got.cpu().float().nan_to_num(9.0), want.float().nan_to_num(9.0))
        # and the framework's dequantize agrees
        flat = bmx.dequantize(w[:, lo:lo + M].reshape(-1, 16).contiguous(), s[:, lo:lo + M].reshape(-1, 2).contiguous(),
                              b[:, lo:lo + M].reshape(-1, 2).contiguous()).reshape(got.shape)
        assert torch.equal(got.float().nan_to_num(9.0), flat.float().nan_to_num(9.0))


@pytest.mark.parametrize("heads,M,offset,cap", [(8, 1, 0, 1), (8, 1, 4095, 4352), (1, 3, 5, 8), (3, 17, 0, 17),
                                                (8, 333, 1001, 1500), (2, 1025, 7, 2000), (5, 64, 936, 1000)])
@pytest.mark.parametrize("layout", ["rows", "cache"])
def test_write_and_read(gpu, heads, M, offset, cap, layout):
    g = torch.Generator().manual_seed(M)
    std = torch.exp(3 * torch.randn(heads, M, 1, generator=g))
    k = (std * torch.randn(heads, M, D, generator=g) + torch.randn(heads, 1, D, generator=g)).to(torch.bfloat16).cuda()
    v = (torch.randn(heads, M, D, generator=g) / std).to(torch.bfloat16).cuda()
    if layout == "rows":
        ks, vs = (x.transpose(0, 1).contiguous().view(M, heads * D).view(M, heads, D).transpose(0, 1) for x in (k, v))
    else:  # a slice of a bf16 cache
        ks, vs = (torch.randn(heads, M + 9, D, device="cuda").to(torch.bfloat16) for _ in "kv")
        ks[:, 4:4 + M], vs[:, 4:4 + M] = k, v
        ks, vs = ks[:, 4:4 + M], vs[:, 4:4 + M]
    cache = random_cache(1, heads, cap)
    names = ("k", "k_scales", "k_biases", "v", "v_scales", "v_biases")
    before = [getattr(cache, n).clone() for n in names]
    bmx.kv4_write(ks, vs, cache, offset)
    check_rows(cache, offset, k, v)
    for n, b in zip(names, before):  # the rows around stay
        t = getattr(cache, n)
        assert torch.equal(t[:, :offset], b[:, :offset]) and torch.equal(t[:, offset + M:], b[:, offset + M:])


def test_write_special_values(gpu):
    """Constant and zero groups, ties, signed zeros, the range's ends, subnormals, NaN and infinities."""
    x = torch.zeros(1, 16, D)
    x[0, 1] = -3.25                                  # constant: scale 0
    x[0, 2, :64] = torch.arange(64) / 4.2            # many values per level
    x[0, 3, :16] = torch.arange(16)                  # scale 1 exactly, every level
    x[0, 3, 16:48] = torch.arange(32) / 2            # halves: ties to even
    x[0, 4, 5] = math.nan
    x[0, 5, 70] = math.inf
    x[0, 6, 3] = -math.inf
    x[0, 7, 0], x[0, 7, 1] = 3.3e38, -3.3e38         # the range overflows fp32
    x[0, 8, 0], x[0, 8, 1] = 1.7e38, -1.6e38         # the range just fits
    x[0, 9, :64] = 1e-40 * torch.arange(64)          # subnormal steps
    x[0, 10, 0] = 1e-39                              # a step that rounds to 0 or nearly
    x[0, 11] = torch.where(torch.arange(D) % 2 == 0, -0.0, 0.0)
    x[0, 12, 64:] = 1e30 + 1e28 * torch.arange(64)
    x[0, 13, 0], x[0, 13, 127] = 1.0, -1.0
    x[0, 14, :64] = math.nan
    x[0, 15, :] = torch.randn(D, generator=torch.Generator().manual_seed(3))
    x = x.to(torch.bfloat16).cuda()
    cache = bmx.Kv4Cache.empty(1, 16)
    bmx.kv4_write(x, x.flip(1).contiguous(), cache, 0)
    check_rows(cache, 0, x, x.flip(1))
    k, _ = bmx.kv4_read(cache, 0, 16)
    bad = k.isnan().view(16, 2, 64).all(-1).cpu()
    assert bad.nonzero().tolist() == [[4, 0], [5, 1], [6, 0], [7, 0], [14, 0]]
    assert k.isnan().sum() == 5 * 64  # whole groups and nothing else


def test_write_near_ties_match_division(gpu):
    """Values whose quotient lies at or next to a half step, for many scales."""
    g = torch.Generator().manual_seed(11)
    rows = 4096
    hi = torch.exp(2 * torch.randn(rows, 1, generator=g)).to(torch.bfloat16).float()
    s = (hi / 15).to(torch.bfloat16).float()
    at = torch.randint(0, 15, (rows, 126), generator=g) + 0.5
    x = (s * at).to(torch.bfloat16).float()
    x = torch.cat([torch.zeros(rows, 1), x[:, :62], hi, torch.zeros(rows, 1), x[:, 63:125], hi], 1)
    x = x.to(torch.bfloat16).reshape(1, rows, D).cuda()
    cache = bmx.Kv4Cache.empty(1, rows)
    bmx.kv4_write(x, x, cache, 0)
    check_rows(cache, 0, x, x)


@pytest.mark.parametrize("Hq,Hkv,M,offset,position", [(32, 8, 1, 4095, None), (16, 8, 5, 0, 17), (6, 2, 37, 11, 90000),
                                                      (64, 8, 9, 3, 0), (8, 8, 130, 20, 2000)])
def test_qk_norm_rope_kv4_is_the_two_calls(gpu, Hq, Hkv, M, offset, position):
    """Bit for bit: qk_norm_rope_kv into a bf16 cache, then kv4_write of its rows."""
    g = torch.Generator().manual_seed(Hq + M)
    q, k, v = ((torch.randn(M, h * D, generator=g)).to(torch.bfloat16).cuda() for h in (Hq, Hkv, Hkv))
    qn, kn = ((1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16).cuda() for _ in "qk")
    at = offset if position is None else position
    kc, vc = (torch.zeros(Hkv, at + M, D, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    want = bmx.qk_norm_rope_kv(q, k, v, qn, kn, kc, vc, at)
    a, b = random_cache(2, Hkv, offset + M + 3), random_cache(2, Hkv, offset + M + 3)
    bmx.kv4_write(kc[:, at:], vc[:, at:], a, offset)
    got = bmx.qk_norm_rope_kv4(q, k, v, qn, kn, b, offset, position=position)
    assert torch.equal(got, want)
    for n in ("k", "k_scales", "k_biases", "v", "v_scales", "v_biases"):
        assert torch.equal(getattr(a, n), getattr(b, n)), n


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
HEADS = [(8, 8), (16, 8), (32, 8), (64, 8), (6, 2), (10, 2), (16, 1), (3, 3)]


@pytest.mark.parametrize("Hq,Hkv", HEADS)
@pytest.mark.parametrize("past", [0, 1, 15, 16, 31, 32, 63, 127, 255, 256, 300])
def test_attention_one_token(gpu, Hq, Hkv, past):
    cache = random_cache(past, Hkv, past + 40, past + 1)
    check_attention(queries(past + 1, Hq, 1), cache, past)


@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (64, 8), (6, 2), (4, 4), (24, 1)])
@pytest.mark.parametrize("M,past", [(2, 0), (5, 1336), (8, 511), (9, 30), (16, 0), (17, 100), (33, 70), (65, 0), (130, 201)])
def test_attention_many_tokens(gpu, Hq, Hkv, M, past):
    cache = random_cache(M, Hkv, past + M + 5, past + M)
    check_attention(queries(M, Hq, M), cache, past)


@pytest.mark.parametrize("Hq,Hkv,M,past", [(32, 8, 1, 4095), (4, 1, 1, 20001), (8, 2, 3, 9999), (4, 1, 40, 5000)])
def test_attention_long(gpu, Hq, Hkv, M, past):
    cache = random_cache(past, Hkv, past + M, past + M)
    w = torch.zeros(Hkv, past + M, device="cuda")
    check_attention(queries(7, Hq, M), cache, past, weights=w)


@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (16, 8), (64, 8), (6, 2), (5, 5)])
@pytest.mark.parametrize("M,past", [(1, 0), (1, 40), (1, 700), (2, 31), (5, 250), (16, 3), (31, 0), (40, 100), (129, 60)])
def test_weights(gpu, Hq, Hkv, M, past):
    cache = random_cache(3 * M, Hkv, past + M + 7, past + M)
    g = torch.Generator().manual_seed(past)
    w = torch.rand(Hkv, past + M + 7, generator=g).cuda()
    got = check_attention(queries(M, Hq, M), cache, past, weights=w)
    # the outputs do not depend on whether weights were asked for
    assert torch.equal(got, bmx.attention_kv4(queries(M, Hq, M), cache, past))


def test_weights_accumulate(gpu):
    """Three steps of one token add up to rep * 3 per kv head."""
    cache = random_cache(5, 2, 64, 40)
    w = torch.zeros(2, 64, device="cuda")
    for i in range(3):
        bmx.attention_kv4(queries(i, 8, 1), cache, 37 + i, weights=w)
    assert torch.allclose(w.sum(1), torch.full((2,), 12.0, device="cuda"), rtol=2e-6)
    assert (w[:, 40:] == 0).all()


def test_attention_concentrated(gpu):
    """Scores of hundreds: one key takes everything, the rest underflow."""
    cache = random_cache(8, 2, 600, 600)
    check_attention(queries(1, 8, 1, std=60.0), cache, 599, weights=torch.zeros(2, 600, device="cuda"))
    check_attention(queries(1, 8, 3, std=60.0), cache, 500, weights=torch.zeros(2, 600, device="cuda"))


def test_attention_zero_scale_is_the_mean(gpu):
    cache = random_cache(9, 2, 300, 300)
    got = bmx.attention_kv4(queries(2, 4, 1), cache, 299, scale=0.0)
    v = ref_values(cache.v, cache.v_scales, cache.v_biases).mean(1)
    for h in range(4):
        want = v[h // 2]
        assert (got[0, h * D:(h + 1) * D].cpu().double() - want).abs().max() < U8 * (want.abs().max() + 8 * 0.45)


@pytest.mark.parametrize("M", [1, 3, 40])
def test_hidden_rows_weigh_nothing(gpu, M):
    """NaN and infinite scales behind the last row, and in rows that only later queries see."""
    past, Hq, Hkv = 70, 8, 2
    cache = random_cache(4, Hkv, 200, past + M)
    q = queries(3, Hq, M)
    clean = bmx.attention_kv4(q, cache, past)
    assert torch.isfinite(clean).all()
    if M > 1:
        cache.v_scales[:, past + M - 1] = math.nan
        cache.v_biases[:, past + M - 1] = math.inf
        cache.k_scales[:, past + M - 1] = math.nan
        w = torch.zeros(Hkv, 200, device="cuda")
        dirty = bmx.attention_kv4(q, cache, past, weights=w)
        assert torch.equal(dirty[:-1], clean[:-1])
        assert dirty[-1].isnan().all()


@pytest.mark.parametrize("M", [1, 40])
def test_bad_rows_poison_their_head_only(gpu, M):
    Hq, Hkv, past = 8, 4, 90
    cache = random_cache(4, Hkv, 200, past + M)
    cache.k_scales[1, 20, 0] = math.nan   # a key of kv head 1
    cache.v_biases[2, 33, 1] = math.nan   # values of kv head 2, second group
    w = torch.zeros(Hkv, 200, device="cuda")
    out = bmx.attention_kv4(queries(3, Hq, M), cache, past, weights=w).view(M, Hkv, 2, D)
    assert torch.isfinite(out[:, [0, 3]]).all() and out[:, 1].isnan().all()
    assert torch.isfinite(out[:, 2, :, :64]).all() and out[:, 2, :, 64:].isnan().all()
    assert torch.isfinite(w[[0, 2, 3]]).all() and w[1, :past + 1].isnan().all()


def test_equal_calls_equal_bits_and_workspace_reuse(gpu):
    """One workspace through calls of every kind and size, left ready each time."""
    cache = random_cache(6, 8, 3000, 3000)
    calls = [(32, 1, 2999, True), (32, 1, 5, False), (64, 5, 1000, True), (16, 300, 1200, True), (32, 1, 2999, True),
             (8, 40, 0, False), (64, 16, 2000, False)]
    ws = bmx.attention_kv4_workspace(64, 8, 300, 3000, weigh=True)
    for i, (Hq, M, past, weigh) in enumerate(calls):
        q = queries(i, Hq, M)
        outs = []
        for space in (ws, ws, None):
            w = torch.zeros(8, 3000, device="cuda") if weigh else None
            outs.append((bmx.attention_kv4(q, cache, past, weights=w, workspace=space), w))
            assert not ws[:bmx.KV4_COUNTER_BYTES].any()
        for o, w in outs[1:]:
            assert torch.equal(o, outs[0][0])
            assert w is None or torch.equal(w, outs[0][1])


def test_workspace_needs_no_more_than_it_says(gpu):
    """Nothing is written past the bytes the query names."""
    for Hq, Hkv, M, past, weigh in [(32, 8, 1, 4000, True), (16, 8, 5, 777, False), (12, 4, 64, 500, True), (4, 4, 200, 0, False)]:
        cache = random_cache(1, Hkv, past + M)
        n = bmx.load().bmx_attention_kv4_workspace_bytes(Hq, Hkv, M, past + M, int(weigh))
        ws = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
        ws[:bmx.KV4_COUNTER_BYTES] = 0
        w = torch.zeros(Hkv, past + M, device="cuda") if weigh else None
        q, out = queries(1, Hq, M), torch.empty(M, Hq * D, dtype=torch.bfloat16, device="cuda")
        rc = bmx.load().bmx_attention_gqa_kv4(q.data_ptr(), cache._ref, out.data_ptr(), None if w is None else w.data_ptr(),
                                              Hq, M, D, past, 0.1, ws.data_ptr(), n, None)
        torch.cuda.synchronize()
        assert rc == 0 and (ws[n:] == 0xA5).all()


def test_side_stream_and_graph(gpu):
    """A step -- write, attend with weights, evict in place -- captured and replayed, against the eager run."""
    Hkv, Hq, cap = 2, 8, 400
    q, k, v = queries(1, Hq, 1), queries(2, Hkv, 1), queries(3, Hkv, 1)
    ws = bmx.attention_kv4_workspace(Hq, Hkv, 1, 301, weigh=True)
    kept = torch.empty(Hkv, 200, dtype=torch.int32, device="cuda")

    def step(cache, w, out, stream):
        bmx.kv4_write(k, v, cache, 300, stream=stream)
        bmx.attention_kv4(q, cache, 300, weights=w, workspace=ws, out=out, stream=stream)
        bmx.kv4_evict(cache, w, 301, 200, sink=4, recent=20, kept=kept, stream=stream)

    def state():
        return random_cache(6, Hkv, cap, 300), torch.full((Hkv, cap), 0.01, device="cuda"), torch.empty(1, Hq * D, dtype=torch.bfloat16, device="cuda")

    want = state()
    results = []
    for _ in range(3):
        step(*want, None)
        results.append([want[0].k.clone(), want[0].v_scales.clone(), want[1].clone(), want[2].clone(), kept.clone()])
    side = torch.cuda.Stream()
    got = state()
    side.wait_stream(torch.cuda.current_stream())
    step(*got, side)  # eager on the side stream
    side.synchronize()
    for a, b in zip(results[0], [got[0].k, got[0].v_scales, got[1], got[2], kept]):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    got = state()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*got, None)
    for i in range(3):
        junk = torch.randn(1000, 1000, device="cuda").sum()  # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(junk)
        for a, b in zip(results[i], [got[0].k, got[0].v_scales, got[1], got[2], kept]):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), i


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------
def ref_kept(w, length, budget, sink, recent):
    keep = []
    for row in w[:, :length].cpu().double().tolist():
        order = sorted(range(sink, length - recent), key=lambda j: (row[j] == row[j], -row[j] if row[j] == row[j] else 0, j))
        keep.append(sorted([*range(sink), *order[:budget - sink - recent], *range(length - recent, length)]))
    return np.array(keep, np.int32).reshape(w.shape[0], budget)


NAMES = ("k", "k_scales", "k_biases", "v", "v_scales", "v_biases")


def check_evict(w, cache, length, budget, sink, recent, in_place):
    kept = ref_kept(w, length, budget, sink, recent)
    at = torch.from_numpy(kept).long().cuda()
    want = [torch.gather(getattr(cache, n), 1, at[..., None].expand(-1, -1, getattr(cache, n).shape[-1])) for n in NAMES]
    want_w = torch.gather(w, 1, at)
    if in_place:
        into, wi = cache, w
    else:
        into, wi = random_cache(99, cache.n_kv_heads, budget + 5), torch.full((cache.n_kv_heads, budget + 5), 7.0, device="cuda")
    tail = [getattr(into, n)[:, budget:].clone() for n in NAMES]
    src = [getattr(cache, n).clone() for n in NAMES]
    got = bmx.kv4_evict(cache, w, length, budget, sink=sink, recent=recent, **({} if in_place else dict(into=into, weights_into=wi)))
    torch.cuda.synchronize()
    assert np.array_equal(got.cpu().numpy(), kept)
    for n, x, t in zip(NAMES, want, tail):
        y = getattr(into, n)
        assert torch.equal(y[:, :budget].view(torch.int16), x.view(torch.int16)), n  # bits: NaN scales too
        assert torch.equal(y[:, budget:].view(torch.int16), t.view(torch.int16)), n  # the rows behind stay
    assert torch.equal(wi[:, :budget].view(torch.int32), want_w.view(torch.int32)) and (wi[:, budget:] == 0).all()
    if not in_place:
        for n, x in zip(NAMES, src):
            assert torch.equal(getattr(cache, n), x)


SIZES = [(1, 1, 0, 0), (2, 1, 0, 0), (2, 1, 0, 1), (5, 5, 2, 3), (5, 5, 0, 0), (9, 4, 4, 0), (9, 4, 0, 4), (65, 64, 4, 8),
         (300, 37, 4, 11), (1024, 1023, 0, 0), (1025, 512, 4, 256), (4352, 1024, 4, 256), (9000, 77, 0, 0), (5000, 4999, 1, 1),
         (16384, 4000, 4, 100), (16385, 4000, 4, 100), (16385, 16385, 0, 0), (40961, 2048, 4, 64), (40961, 30000, 0, 20000),
         (100003, 30001, 20000, 5), (131072, 4096, 0, 0)]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("length,budget,sink,recent", SIZES)
def test_evict(gpu, length, budget, sink, recent, in_place):
    heads = 3
    cache = random_cache(length, heads, length + 6)
    g = torch.Generator().manual_seed(budget)
    w = (torch.rand(heads, length + 6, generator=g) ** 6).cuda()
    check_evict(w, cache, length, budget, sink, recent, in_place)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few", "signed", "special", "rising", "falling", "subnormal"])
@pytest.mark.parametrize("length,budget", [(700, 300), (3000, 64), (9000, 2000), (20000, 9000), (50001, 700)])
def test_evict_ties_and_orders(gpu, kind, length, budget):
    heads = 2
    cache = random_cache(1, heads, length)
    g = torch.Generator().manual_seed(length)
    r = torch.rand(heads, length, generator=g)
    w = {"equal": torch.full((heads, length), 0.25), "zeros": torch.where(r < 0.5, -0.0, 0.0), "few": torch.round(3 * r),
         "signed": r - 0.5, "rising": torch.arange(length).float().expand(heads, -1) / 7,
         "falling": -torch.arange(length).float().expand(heads, -1) / 7, "subnormal": 1e-42 * torch.round(20 * r),
         "special": torch.where(r < 0.05, math.nan, torch.where(r < 0.1, math.inf, torch.where(r > 0.95, -math.inf, r)))}[kind]
    check_evict(w.contiguous().cuda(), cache, length, budget, 4, 16, True)


def test_evict_then_continue(gpu):
    """Decode with a bounded cache: prompt, weigh its last tokens, cut, then
    write / attend / cut as the text goes on; every step against float64."""
    Hq, Hkv, cap, budget = 8, 2, 260, 120
    g = torch.Generator().manual_seed(21)
    cache, w = bmx.Kv4Cache.empty(Hkv, cap), torch.zeros(Hkv, cap, device="cuda")
    qn, kn = (torch.ones(D, dtype=torch.bfloat16, device="cuda") for _ in "qk")
    ws = bmx.attention_kv4_workspace(Hq, Hkv, 200, cap, weigh=True)

    def project(M):
        return [torch.randn(M, h * D, generator=g).to(torch.bfloat16).cuda() for h in (Hq, Hkv, Hkv)]

    rows = position = 0
    for M in (200, 1, 1, 37, 1, 5, 1, 1, 60, 1):
        if rows + M > cap:
            bmx.kv4_evict(cache, w, rows, budget, sink=4, recent=32)
            rows = budget
        q = bmx.qk_norm_rope_kv4(*project(M), qn, kn, cache, rows, position=position)
        check_attention(q, cache, rows, weights=w, ws=ws)
        rows, position = rows + M, position + M
    assert position == 308 and rows < position


def test_gpu_python_refusals(gpu):
    cache = bmx.Kv4Cache.empty(2, 50)
    q = queries(1, 4, 1)
    w = torch.zeros(2, 50, device="cuda")
    k = queries(2, 2, 3)

    def code(f, *a, **kw):
        with pytest.raises(bmx.BmxError) as e:
            f(*a, **kw)
        return e.value.code

    assert code(bmx.attention_kv4, queries(1, 3, 1), cache, 0) == bmx.BMX_E_SHAPE
    assert code(bmx.attention_kv4, q.float(), cache, 0) == bmx.BMX_E_ARG
    assert code(bmx.attention_kv4, q, cache, 50) == bmx.BMX_E_KV_CAPACITY
    assert code(bmx.attention_kv4, q, cache, -1) == bmx.BMX_E_KV_CAPACITY
    assert code(bmx.attention_kv4, q, cache, 0, weights=w[:, :49].contiguous()) == bmx.BMX_E_SHAPE
    assert code(bmx.attention_kv4, q, cache, 0, weights=w.double()) == bmx.BMX_E_ARG
    assert code(bmx.attention_kv4, q, cache, 0, workspace=torch.zeros(100, device="cuda")) == bmx.BMX_E_ARG
    assert code(bmx.attention_kv4, q, cache, 0, out=torch.empty(7, dtype=torch.bfloat16, device="cuda")) == bmx.BMX_E_SHAPE
    assert code(bmx.attention_kv4, queries(1, 4, 4).transpose(0, 1), cache, 0) == bmx.BMX_E_ARG
    assert code(bmx.kv4_write, k, k[:, :2], cache, 0) == bmx.BMX_E_SHAPE
    assert code(bmx.kv4_write, k, k, cache, 48) == bmx.BMX_E_KV_CAPACITY
    assert code(bmx.kv4_write, k.transpose(1, 2).contiguous().transpose(1, 2), k, cache, 0) == bmx.BMX_E_ARG
    odd = torch.empty(2 * 3 * 129 + 1, dtype=torch.bfloat16, device="cuda")
    assert code(bmx.kv4_write, odd[:-1].view(2, 3, 129)[:, :, :128], k, cache, 0) == bmx.BMX_E_ALIGN
    assert code(bmx.kv4_read, cache, 0, 51) == bmx.BMX_E_KV_CAPACITY
    assert code(bmx.kv4_read, cache, 5, 4) == bmx.BMX_E_KV_CAPACITY
    assert bmx.kv4_read(cache, 7, 7)[0].shape == (2, 0, 128)
    assert code(bmx.kv4_evict, cache, w, 51, 20) == bmx.BMX_E_KV_CAPACITY
    assert code(bmx.kv4_evict, cache, w, 20, 21) == bmx.BMX_E_SHAPE
    assert code(bmx.kv4_evict, cache, w, 20, 0) == bmx.BMX_E_SHAPE
    assert code(bmx.kv4_evict, cache, w, 20, 10, into=bmx.Kv4Cache.empty(2, 10)) == bmx.BMX_E_ARG
    assert code(bmx.qk_norm_rope_kv4, *(torch.zeros(2, n * D, dtype=torch.bfloat16, device="cuda") for n in (4, 3, 2)),
                torch.ones(D, dtype=torch.bfloat16, device="cuda"), torch.ones(D, dtype=torch.bfloat16, device="cuda"), cache, 0) == bmx.BMX_E_SHAPE
