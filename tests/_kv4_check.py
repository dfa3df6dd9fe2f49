"""Attention over the 4-bit KV cache against its definition in float64, one kv
head at a time, with bounds that a wrong row or group cannot hide under.  Plain
torch on any device."""
import math

import torch

U8 = 2.0 ** -8    # largest relative rounding error of bf16
U24 = 2.0 ** -24  # of fp32
D = 128


def values(words, s, b):
    """float64 values of cache rows."""
    n = (words.to(torch.int64)[..., None] >> (4 * torch.arange(8, device=words.device))) & 15
    wide = lambda x: x.double().repeat_interleave(64, -1)
    return n.reshape(*words.shape[:-1], D).double() * wide(s) + wide(b)


def visible(rep, M, past, device):
    see = torch.arange(past + M, device=device) <= past + torch.arange(M, device=device)[:, None]
    return see.repeat(rep, 1)


def head_reference(q, cache, h, past, scale):
    """Of kv head h: outputs [rep * M, 128], weights p [rep * M, L], how far a right
    output and a right sum of weights may be off, and the largest |S|.

    An output is off by its own rounding, U8 |out|.  Of the keys' parts, weight
    and values are rounded to no fewer than 8 bits each, against the centred
    nibble n - 7.5 and the middle 7.5 s + b of its group: a relative error of at
    most U8 in p |s| |n - 7.5| and in p |7.5 s + b|, independent from key to
    key.  A sum of independent errors within +-u has a standard deviation of
    at most u / sqrt(3) each; six of them are not passed in 10^9 values.

    A score's error: up to 140 fp32 additions, each off by U24 of the partial sum
    it makes.  With 16 Q to take off (Q the group's sum of q) and nibbles that
    do not depend on q, a partial sum of q (16 + n) stays within 16 |Q| +
    3 |q| 31; it is multiplied by s.  The biases' part is a few roundings of
    |b Q|, the score's end a few of |S|.  A weight moves by that and by its row's
    common factor (twice e), and from key to key independently.  The rest is
    fp32 sums."""
    Hq, M, _ = q.shape
    rep, L = Hq // cache.n_kv_heads, past + M
    k = values(cache.k[h, :L], cache.k_scales[h, :L], cache.k_biases[h, :L])
    v = values(cache.v[h, :L], cache.v_scales[h, :L], cache.v_biases[h, :L])
    qd = q[h * rep:(h + 1) * rep].double().reshape(rep * M, D)
    s = torch.mm(qd, k.t().contiguous()) * scale
    see = visible(rep, M, past, q.device)
    p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
    out = torch.mm(p, v)
    vs = cache.v_scales[h, :L].double().repeat_interleave(64, -1)
    middle = 7.5 * vs + cache.v_biases[h, :L].double().repeat_interleave(64, -1)
    spread = torch.mm(p.square(), (v - middle).square() + middle.square()).sqrt()
    mass = torch.mm(p, v.abs()) + 7.5 * torch.mm(p, vs.abs())
    groups = qd.reshape(rep * M, 2, 64)
    sums = groups.sum(-1).abs()
    partial = 16 * sums + 93 * groups.norm(dim=-1)
    e = U24 * abs(scale) * (140 * torch.mm(partial, cache.k_scales[h, :L].double().abs().t().contiguous())
                            + 8 * torch.mm(sums, cache.k_biases[h, :L].double().abs().t().contiguous())) + 4 * U24 * s.abs()
    e = torch.where(see, e, 0.0)
    score = 2 * torch.mm((p * e).square(), v.square()).sqrt()
    bound = U8 * out.abs() + 6 / math.sqrt(3) * U8 * spread + score + 2.0 ** -20 * mass + 1e-30
    weigh = (p * (2 * e.amax(-1, keepdim=True) + 64 * U24)).sum(0)
    big = float(torch.where(see, s.abs(), 0.0).max())
    return out, p, bound, weigh, big


def hold(got, out, bound, what=""):
    """Every element within its bound, and every row's half (a group of 64) close as a whole."""
    off = (got - out).abs() / bound
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    assert float(off.max()) < 1, f"{what}: {float(off.max()):.3g} of the bound"
    # a group's norm: U8 of it for the outputs' rounding, and half of what its
    # elements' six deviations add up to for the keys' parts
    err = (got - out).reshape(-1, 2, 64).norm(dim=-1)
    lim = U8 * out.reshape(-1, 2, 64).norm(dim=-1) + 0.5 * (bound - U8 * out.abs()).reshape(-1, 2, 64).norm(dim=-1)
    assert bool((err <= lim).all()), f"{what}: a row's group is off by {float((err / lim).max()):.3g} of its norm's bound"


def check(call, q, cache, past, scale=None, weigh=True):
    """`call` (bmx.attention_kv4's arguments) against the definition; returns outputs [M, Hq * 128]."""
    Hq, M, _ = q.shape
    Hkv, L = cache.n_kv_heads, past + M
    rep, scale = Hq // Hkv, 1 / math.sqrt(D) if scale is None else scale
    w = torch.full((Hkv, cache.capacity), 0.5, device=q.device) if weigh else None
    got = call(q, cache, past, scale=scale, weights=w)
    for h in range(Hkv):
        out, p, bound, tol, big = head_reference(q, cache, h, past, scale)
        g = got.view(M, Hq, D)[:, h * rep:(h + 1) * rep].transpose(0, 1).reshape(rep * M, D).double()
        hold(g, out, bound, f"kv head {h}")
        if weigh:
            want = 0.5 + p.sum(0)
            d = (w[h, :L].double() - want).abs() / (tol + 4 * U24 * (0.5 + want))
            assert float(d.max()) <= 1, f"kv head {h}: {float(d.max()):.3g} of the weights' tolerance"
            # as a whole: S and the logarithm of the sum are fp32 numbers, each
            # the end of a chain whose last few roundings (four at most) are at
            # its own size, on both sides
            off = float((w[h, :L].double() - want).norm() / want.norm())
            assert off < max(1e-5, 8 * U24 * big), f"kv head {h}: weights off by {off:.3g}"
    return got
