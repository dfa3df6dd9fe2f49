"""Attention over the 4-bit KV cache where its kernels for many rows, long
contexts and unusual values run: against float64 on the same device, one kv
head at a time."""
import math

import pytest
import torch

import bmx
from test_gpu_kv4 import D, U24, U8, check_evict, queries, random_cache

pytestmark = pytest.mark.gpu


def values(words, s, b):
    n = (words.to(torch.int64)[..., None] >> (4 * torch.arange(8, device=words.device))) & 15
    wide = lambda x: x.double().repeat_interleave(64, -1)
    return n.reshape(*words.shape[:-1], D).double() * wide(s) + wide(b)


def check(q, cache, past, scale=None, weigh=True):
    """Outputs [M, Hq, 128] and weights of a call, each held to its bound:
    U8 of the output for its rounding; P and V off by U8 each at most, against
    the weighted magnitudes or against the centred nibbles and the middles
    (U8 (2 mass + centred)); a score off by e moves its weight by a factor
    within exp(2 e)."""
    Hq, M, _ = q.shape
    Hkv, L = cache.n_kv_heads, past + M
    rep, scale = Hq // Hkv, 1 / math.sqrt(D) if scale is None else scale
    w = torch.full((Hkv, cache.capacity), 0.5, device="cuda") if weigh else None
    got = bmx.attention_kv4(q, cache, past, scale=scale, weights=w)
    if weigh:  # the outputs are the same bits without
        assert torch.equal(got, bmx.attention_kv4(q, cache, past, scale=scale))
        assert (w[:, L:] == 0.5).all()
    see = torch.arange(L, device="cuda") <= past + torch.arange(M, device="cuda")[:, None]
    see = see.repeat(rep, 1)
    diff = ref = 0.0
    for h in range(Hkv):
        k = values(cache.k[h, :L], cache.k_scales[h, :L], cache.k_biases[h, :L])
        v = values(cache.v[h, :L], cache.v_scales[h, :L], cache.v_biases[h, :L])
        qd = q[h * rep:(h + 1) * rep].double().reshape(rep * M, D)
        s = torch.mm(qd, k.t().contiguous()) * scale
        p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
        out = torch.mm(p, v)
        mass = torch.mm(p, v.abs())
        centred = 7.5 * torch.mm(p, cache.v_scales[h, :L].double().abs().repeat_interleave(64, -1))
        e = 140 * U24 * abs(scale) * qd.abs().sum(-1, keepdim=True) * torch.maximum(
            31 * cache.k_scales[h, :L].double().abs().amax(-1), cache.k_biases[h, :L].double().abs().amax(-1))
        es = e.amax(-1, keepdim=True)
        bound = U8 * out.abs() + 1.05 * (2 * es * mass + U8 * (2 * mass + centred)) + 2.0 ** -20 * (mass + centred) + 1e-30
        g = got.view(M, Hq, D)[:, h * rep:(h + 1) * rep].transpose(0, 1).reshape(rep * M, D).double()
        off = ((g - out).abs() / bound).max()
        assert off < 1, f"kv head {h}: {float(off):.3g} of the bound"
        diff, ref = diff + float((g - out).square().sum()), ref + float(out.square().sum())
        if weigh:
            want = 0.5 + p.sum(0)
            tol = (p * (2 * es + 64 * U24)).sum(0) + 4 * U24 * (0.5 + want)
            d = (w[h, :L].double() - want).abs()
            assert (d <= tol).all(), f"kv head {h}: {float((d / tol).max()):.3g} of the weights' tolerance"
    assert diff ** 0.5 < 3e-3 * ref ** 0.5, (diff / ref) ** 0.5
    return got


WIDE = [(32, 8, 512, 0), (32, 8, 511, 2001), (64, 8, 130, 70), (64, 8, 65, 3001), (16, 1, 777, 0), (64, 8, 40, 20000),
        (16, 2, 700, 0), (64, 64, 30, 100), (6, 2, 1000, 0), (5, 5, 700, 33), (24, 3, 200, 1000), (12, 2, 333, 4100),
        (16, 1, 64, 20001), (32, 8, 1024, 0),
        (32, 8, 140, 16001), (64, 8, 32, 16000), (64, 64, 200, 0), (8, 1, 1500, 700), (32, 8, 1, 12000), (64, 8, 1, 5001), (3, 3, 1, 300001), (8, 1, 1, 300001), (64, 8, 16, 9000)]


@pytest.mark.parametrize("Hq,Hkv,M,past", WIDE)
def test_wide(gpu, Hq, Hkv, M, past):
    cache = random_cache(M + past, Hkv, past + M + 3, past + M)
    check(queries(M, Hq, M), cache, past)


# a call for each kernel: few rows, more, tiles of 64, of 256
KERNELS = [(8, 2, 1, 700), (8, 2, 40, 70), (64, 8, 130, 70), (32, 8, 1024, 0)]


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS)
@pytest.mark.parametrize("scale", [-0.07, 1e-4, 0.6])
def test_scales(gpu, Hq, Hkv, M, past, scale):
    cache = random_cache(1, Hkv, past + M, past + M)
    check(queries(M, Hq, M), cache, past, scale=scale)


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS)
@pytest.mark.parametrize("kind", ["tiny", "huge", "ends", "rows", "rising", "groups", "negative"])
def test_value_magnitudes(gpu, Hq, Hkv, M, past, kind):
    """Values of 2^-60, 2^100 and 2^117 as a whole, of 2^-20 .. 2^20 from row to row,
    rising along the context, of 2^12 between a row's groups, and negative scales."""
    cache = random_cache(2, Hkv, past + M, past + M)
    g = torch.Generator().manual_seed(5)
    n = past + M
    f = {"tiny": torch.full((n, 2), 2.0 ** -60), "huge": torch.full((n, 2), 2.0 ** 100),
         "ends": torch.full((n, 2), 2.0 ** 117),
         "rows": 2.0 ** torch.randint(-20, 21, (n, 1), generator=g).float().expand(n, 2),
         "rising": 2.0 ** torch.linspace(-30, 30, n).round()[:, None].expand(n, 2),
         "groups": torch.tensor([[2.0 ** -12, 1.0]]).expand(n, 2),
         "negative": torch.where(torch.rand(n, 2, generator=g) < 0.5, -1.0, 1.0)}[kind].cuda()
    cache.v_scales.mul_(f)
    cache.v_biases.mul_(f)
    check(queries(M, Hq, M), cache, past, weigh=False)


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS[1:])
@pytest.mark.parametrize("kind", ["largest", "lowest", "nan"])
def test_what_a_query_does_not_see(gpu, Hq, Hkv, M, past, kind):
    """The last rows hold bf16's ends or NaN: the queries before keep their bits."""
    cache = random_cache(3, Hkv, past + M + 9, past + M)
    q = queries(M, Hq, M)
    clean = bmx.attention_kv4(q, cache, past)
    last = slice(past + M - 5, past + M)
    most = torch.finfo(torch.bfloat16).max
    value = {"largest": most, "lowest": -most, "nan": math.nan}[kind]
    cache.v_biases[:, last] = value
    cache.v_scales[:, last] = 0.0 if kind != "nan" else math.inf
    cache.k_biases[:, last] = value
    dirty = bmx.attention_kv4(q, cache, past)
    assert torch.equal(dirty[:-5], clean[:-5])


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS)
def test_bad_rows_stay_in_their_group(gpu, Hq, Hkv, M, past):
    """A NaN key takes its kv head's rows that see it, an infinite value its group of 64."""
    cache = random_cache(4, Hkv, past + M, past + M)
    at = past + M // 2
    cache.v[1, at, 8:] = 0x77777777  # (0 times infinity is no infinity)
    cache.k_scales[0, at, 1] = math.nan
    cache.v_scales[1, at, 1] = math.inf
    w = torch.zeros(Hkv, past + M, device="cuda")
    out = bmx.attention_kv4(queries(M, Hq, M), cache, past, weights=w).view(M, Hkv, Hq // Hkv, D)
    sees = M // 2
    assert out[sees:, 0].isnan().all() and torch.isfinite(out[:sees]).all()
    assert not torch.isfinite(out[sees:, 1, :, 64:]).any() and torch.isfinite(out[:, 1, :, :64]).all()
    assert torch.isfinite(out[:, 2:]).all()
    assert w[0, :at + 1].isnan().all() and torch.isfinite(w[1:]).all()


def test_steps_share_a_workspace_between_graphs(gpu):
    """Two captured calls of different kernels, one workspace, replayed in turns."""
    cache = random_cache(6, 8, 3000, 3000)
    ws = bmx.attention_kv4_workspace(32, 8, 300, 3000, weigh=True)
    calls = [(queries(1, 32, 1), 2999), (queries(2, 32, 300), 2500), (queries(3, 32, 5), 700)]
    want, graphs = [], []
    for q, past in calls:
        w = torch.zeros(8, 3000, device="cuda")
        want.append((bmx.attention_kv4(q, cache, past, weights=w, workspace=ws).clone(), w))
    torch.cuda.synchronize()
    for q, past in calls:
        w, out = torch.zeros(8, 3000, device="cuda"), torch.empty(q.shape[1], 32 * D, dtype=torch.bfloat16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.zero_()
            bmx.attention_kv4(q, cache, past, weights=w, workspace=ws, out=out)
        graphs.append((graph, out, w))
    for turn in range(3):
        for i in (turn, (turn + 1) % 3, (turn + 2) % 3):
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for (graph, out, w), (o, ww) in zip(graphs, want):
            assert torch.equal(out, o) and torch.equal(w, ww)
            out.zero_()


def test_no_tokens(gpu):
    """Calls of no tokens at all leave the cache as it is."""
    cache = random_cache(7, 2, 20)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scales.view(torch.int16))]
    none = torch.empty(2, 0, D, dtype=torch.bfloat16, device="cuda")
    bmx.kv4_write(none, none, cache, 20)
    rows = [torch.empty(0, n * D, dtype=torch.bfloat16, device="cuda") for n in (4, 2, 2)]
    unit = torch.ones(D, dtype=torch.bfloat16, device="cuda")
    assert bmx.qk_norm_rope_kv4(*rows, unit, unit, cache, 20).shape == (4, 0, D)
    assert bmx.attention_kv4(queries(1, 4, 1)[:, :0].contiguous(), cache, 20).shape == (0, 4 * D)
    for f in (lambda: bmx.kv4_write(none, none, cache, 21), lambda: bmx.qk_norm_rope_kv4(*rows, unit, unit, cache, 21)):
        with pytest.raises(bmx.BmxError):
            f()
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scales.view(torch.int16))))


@pytest.mark.parametrize("Hq,Hkv,M,past", KERNELS)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_query_stays_alone(gpu, Hq, Hkv, M, past, bad):
    """A NaN or infinity in one query: every other row keeps its bits."""
    cache = random_cache(8, Hkv, past + M, past + M)
    q = queries(M, Hq, M)
    want = bmx.attention_kv4(q, cache, past).view(M, Hq, D)
    h, t = Hq // 2, M // 2
    q[h, t, 70] = bad
    got = bmx.attention_kv4(q, cache, past).view(M, Hq, D)
    same = torch.ones(M, Hq, dtype=torch.bool, device="cuda")
    same[t, h] = False
    assert torch.equal(got[same], want[same]) and not torch.isfinite(got[t, h]).all()


def test_two_streams_at_once(gpu):
    """Calls on two streams with a workspace each, queued without waiting."""
    cache = random_cache(9, 8, 5000, 5000)
    calls = [(queries(i, 32, M), past) for i, (M, past) in enumerate([(1, 4999), (5, 3000), (300, 100), (1, 10)])]
    want = [bmx.attention_kv4(q, cache, past) for q, past in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    spaces = [bmx.attention_kv4_workspace(32, 8, 300, 5000) for _ in streams]
    torch.cuda.synchronize()
    got = [[], []]
    for turn in range(10):
        for i, (s, ws) in enumerate(zip(streams, spaces)):
            q, past = calls[(turn + i) % 4]
            got[i].append(bmx.attention_kv4(q, cache, past, workspace=ws, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        for turn in range(10):
            assert torch.equal(got[i][turn], want[(turn + i) % 4]), (i, turn)


def test_past_four_gib(gpu):
    """Heads whose rows lie more than 2^32 bytes into the cache: written, read,
    attended over, weighed and cut.  All rows but the last ten are zeros, which
    score 0 and add nothing."""
    Hkv, Hq, cap, new = 8, 16, 9_000_000, 10
    past = cap - new
    cache, w = bmx.Kv4Cache.empty(Hkv, cap), torch.zeros(Hkv, cap, device="cuda")
    g = torch.Generator().manual_seed(1)
    k, v = ((4 * torch.randn(Hkv, new, D, generator=g)).to(torch.bfloat16).cuda() for _ in "kv")
    bmx.kv4_write(k, v, cache, past)
    rk, rv = bmx.kv4_read(cache, past - 1, cap)
    assert not rk[:, 0].any() and not rv[:, 0].any()
    kd, vd = (values(*(getattr(cache, n + s)[:, past:] for s in ("", "_scales", "_biases"))) for n in "kv")
    assert torch.equal(rk[:, 1:], kd.float().to(torch.bfloat16)) and torch.equal(rv[:, 1:], vd.float().to(torch.bfloat16))
    for M in (1, new):  # few rows, more
        lo = cap - M
        q = queries(3 + M, Hq, M, std=4.0)
        w.zero_()
        got = bmx.attention_kv4(q, cache, lo, weights=w).view(M, Hkv, 2, D)
        s = torch.matmul(q.double().view(Hkv, 2 * M, D), kd.transpose(1, 2).contiguous()) / math.sqrt(D)
        see = (torch.arange(new, device="cuda") - (new - M) <= torch.arange(M, device="cuda")[:, None]).repeat(2, 1)
        x = torch.where(see, s.exp(), 0.0)
        p = x / (past + x.sum(-1, keepdim=True))
        out = torch.matmul(p, vd).view(Hkv, 2, M, D).permute(2, 0, 1, 3)
        # outputs as above: U8 for the rounding, U8 (2 mass + centred) for P and V
        size = 3 * vd.abs() + 7.5 * cache.v_scales[:, past:].double().abs().repeat_interleave(64, -1)
        size = torch.matmul(p, size).view(Hkv, 2, M, D).permute(2, 0, 1, 3)
        assert ((got.double() - out).abs() <= 1.05 * U8 * size + 1e-12).all()
        # weights: a sum of 9 million equal terms is off by far less than 1e-4
        tol = 1e-4 * p.sum(1) + 1e-12
        assert ((w[:, past:].double() - p.sum(1)).abs() <= tol).all()
        zero = (1 / (past + x.sum(-1))).sum(-1, keepdim=True)
        assert ((w[:, ::1000003].double() - zero).abs() <= 1e-4 * zero).all()
    r = torch.rand(Hkv, cap, generator=g)
    w.copy_(r)
    into, wi = bmx.Kv4Cache.empty(Hkv, 1000), torch.empty(Hkv, 1000, device="cuda")
    kept = bmx.kv4_evict(cache, w, cap, 1000, sink=4, recent=new, into=into, weights_into=wi)
    order = torch.sort(w[:, 4:past], dim=1, descending=True, stable=True)[1][:, :1000 - 4 - new] + 4
    assert torch.equal(kept[:, 4:-new].long(), order.sort(1)[0])
    assert torch.equal(into.v[:, -new:], cache.v[:, past:]) and torch.equal(wi, torch.gather(w, 1, kept.long()))
    assert bmx.kv4_evict(cache, w, cap, 1000, sink=4, recent=new).equal(kept)
    assert torch.equal(cache.k[:, :1000], into.k) and torch.equal(cache.v_biases[:, :1000], into.v_biases)


def test_a_cache_keeps_its_tensors(gpu):
    """Other tensors in a cache's place would leave the library with the old addresses."""
    cache = random_cache(1, 2, 8)
    cache.v_scales *= 2  # the same tensor
    for name in ("k", "v_biases", "capacity"):
        with pytest.raises(bmx.BmxError):
            setattr(cache, name, torch.zeros(1))
    assert cache.capacity == 8


@pytest.mark.parametrize("kind", ["random", "equal", "few", "narrow"])
@pytest.mark.parametrize("heads,length,budget", [(60, 17000, 500), (2, 33000, 9000)])
def test_evict_slices(gpu, kind, heads, length, budget):
    """Both sizes of a long head's slices; weights that agree in all their bits, or in the first eleven."""
    g = torch.Generator().manual_seed(heads)
    r = torch.rand(heads, length, generator=g)
    w = {"random": r ** 5, "equal": torch.full_like(r, 0.5), "few": torch.round(2 * r), "narrow": 0.5 + 0.01 * r}[kind]
    check_evict(w.cuda(), random_cache(2, heads, length), length, budget, 4, 100, False)


def test_evict_workspace_serves_shorter_lengths():
    q = bmx.load().bmx_kv4_evict_workspace_bytes
    for heads in (1, 8, 16, 17, 64):
        sizes = [q(heads, n) for n in range(8193, 600000, 991)]
        assert sizes == sorted(sizes)
