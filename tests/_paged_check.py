"""A paged cache and a batch on any device, and the operators over them from
their definitions in float64."""
import math

import torch

D = 128
U8 = 2.0 ** -8    # largest relative rounding error of bf16
U24 = 2.0 ** -24  # of fp32


def normal(seed, *shape, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device, dtype=torch.float32)


def layout(seed, new, lens, page, spare=3, common=0, width=None):
    """Page lists in random order, `common` first pages the same for all;
    (lists, pages there are)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    n_pages = common + sum(max(n - common, 0) for n in need) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    lists, at = [], common
    for n in need:
        lists.append((order[:common] + order[at:at + max(n - common, 0)])[:max(n, common)])
        at += max(n - common, 0)
    if width:
        lists = [x + [-1] * (width - len(x)) for x in lists]
    return lists, n_pages


def rows_of(x, table, L):
    """Rows 0 .. L - 1 of a sequence whose page list is `table`, [n_kv_heads, L, 128];
    None in the place of pages that do not exist, as zeros, and which rows do."""
    n, H, page, _ = x.shape
    pages = table[:-(-L // page)] if L > 0 else []
    real = torch.tensor([0 <= p < n for p in pages], dtype=torch.bool, device=x.device)
    at = torch.tensor([p if 0 <= p < n else 0 for p in pages], dtype=torch.long, device=x.device)
    got = x[at].transpose(0, 1).reshape(H, -1, D)[:, :max(L, 0)]
    return got, real.repeat_interleave(page)[:max(L, 0)]


def attention_reference(q, k, v, new, lens, tables, scale, shared=0, cap=None, half=True):
    """out [T, Hq, 128] float64, and how far a right bf16 output may be off.

    An output is off by its own rounding, U8 |out|.  A score is 128 fp32
    additions of products that are exact, and three more roundings of the score
    itself: off by e, which moves a weight and its row's sum by exp(e) each.
    Weights are held in two bf16 pieces, each off by U8 of itself: U8^2 in all;
    or (half: prompts, shared rows) in fp16, off by 2^-11 at most, 2^-32 below
    the largest weight (2^7 of 2^-25 fp16's smallest step, halved), and with them
    the values: exactly from 2^-25 on, below that off by less than 2^-32, where the 8
    values about it reach 2^-20.
    The exponential (2 units), sums over keys and the parts' joining: fp32,
    fewer than 2^5 roundings on a chain at a weight's size for the lengths here
    beyond the random walk of the sum, which 2^-18 of the mass covers."""
    Hq, T, _ = q.shape
    Hkv, dev = k.shape[1], q.device
    rep = Hq // Hkv
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=dev)
    bound = torch.full_like(out, 1e-37)
    row = 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        L = min(lens[b], cap) if cap else lens[b]
        table = (tables[0][:shared // k.shape[2]] + tables[b][shared // k.shape[2]:]) if shared else tables[b]
        kr, real = rows_of(k, table, L)
        vr, _ = rows_of(v, table, L)
        pos = lens[b] - n + torch.arange(n, device=dev)
        see = (torch.arange(max(L, 0), device=dev)[None] <= pos[:, None]) & real[None]
        see = see[:, None].expand(n, rep, max(L, 0)).reshape(n * rep, -1)
        any_ = see.any(0) if L > 0 else None
        for h in range(Hkv if L > 0 else 0):
            kd = torch.where(any_[:, None], kr[h].double(), 0.0)
            vd = vr[h].double()
            rows = q[h * rep:(h + 1) * rep, row:row + n].transpose(0, 1).reshape(n * rep, D).double()
            s = torch.mm(rows, kd.t().contiguous()) * scale
            s = torch.where(see, s, -math.inf)
            some = see.any(1, keepdim=True)
            top = torch.where(some, s.amax(1, keepdim=True), 0.0)
            e = torch.exp(s - top)
            p = torch.where(some, e / e.sum(1, keepdim=True).clamp(min=1e-300), 0.0)
            clean = torch.where(torch.isfinite(vd) & any_[:, None], vd, 0.0)
            o = torch.mm(p, clean)
            mass = torch.mm(p, clean.abs())
            odd = (~torch.isfinite(vd)) & any_[:, None]
            if odd.any():  # what such values do to the rows that see them
                hit = torch.mm(see.double(), odd.double()) > 0
                o = torch.where(hit, math.nan, o)
            mag = torch.mm(rows.abs(), kd.abs().t().contiguous()) * abs(scale)
            err = U24 * (130 * mag + 4 * s.abs())
            err = torch.where(see & torch.isfinite(err), err, 0.0).amax(1, keepdim=True)
            w = U8 * o.abs() + (torch.expm1(2 * err) + (2.0 ** -11 if half else U8 * U8) + 2.0 ** -18) * mass + 1e-37
            if half:
                w = w + 2.0 ** -32 + 2.0 ** -32 * torch.mm(see.double(), clean.abs())
            out[row:row + n, h * rep:(h + 1) * rep] = o.reshape(n, rep, D)
            bound[row:row + n, h * rep:(h + 1) * rep] = w.reshape(n, rep, D)
        row += n
    return out, bound


def hold(got, out, bound, what=""):
    """Every output within its bound; not finite exactly where the definition's is not."""
    got = got.double().reshape(out.shape)
    nan = torch.isnan(out)
    assert not torch.isfinite(got[nan]).any(), f"{what}: finite where a visible value is not"
    off = torch.where(nan, 0.0, (got - torch.nan_to_num(out)).abs() / torch.where(nan, 1.0, bound))
    bad = ~(off <= 1)
    assert not bad.any(), (f"{what}: {int(bad.sum())} values off, first {bad.nonzero()[:3].tolist()}, worst "
                           f"{float(torch.nan_to_num(off, nan=math.inf).max()):.3g} of the bound")
    # as a whole: an output's rounding is uniform within +-U8 of a power of two
    # below it, so its square's mean is at most (U8 out)^2 / 3 and that square's
    # deviation 0.9 of it; the sum over the outputs, weighted by out^2, has a
    # relative deviation of 0.9 / sqrt(n), n = (sum out^2)^2 / sum out^4 the number
    # of outputs that count.  Six of them from n = 1000 on: 17 %, 8.3 % of the norm.
    # (Few outputs that count may all be off by U8.)  The rest is far smaller.
    out = torch.nan_to_num(out)
    two = out.square().sum()
    if float(two ** 2) < 1000 * float(out.pow(4).sum()):
        return
    rel = float((torch.where(nan, 0.0, got) - out).norm() / two.sqrt())
    assert rel < 1.083 * U8 / math.sqrt(3), f"{what}: off by {rel:.3g} of the norm"


def rotated(x, w, pos, eps, theta):
    """x [n, heads, 128] normed and rotated in float64, and how far a right result
    may be off: its rounding, and fp32 arithmetic -- the mean of 128 squares and
    the root 8 roundings, two products, cos and sin two units each and two
    products and a sum of the pair: 2^-19 of the pair's magnitudes."""
    y = x.double()
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    ang = pos.double()[:, None, None] * float(theta) ** (-torch.arange(64, dtype=torch.float64, device=x.device) / 64)
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = y[..., :64], y[..., 64:]
    out = torch.cat([a * c - b * s, b * c + a * s], -1)
    mag = (a.abs() + b.abs()).repeat(1, 1, 2)
    return out, U8 * out.abs() + 2.0 ** -19 * mag + 1e-37
