"""The operators of a KV cache held in 4 bits, as cases that can be timed and
compared: rows quantised into the cache and read back, attention over it
(single tokens, draft verification, prompt chunks), attention that also
gathers the weight every cached position drew, and the eviction of the
positions that drew least.

The cache of a layer is MLX affine 4-bit with groups of 64, the format of the
framework's weights: k and v [n_kv_heads, capacity, 16] words of eight
nibbles, and [n_kv_heads, capacity, 2] bf16 scales s and biases b, a value
being s * nibble + b.

`run` in its plain form is float32 torch; with `own` it makes the package's
calls.  `exact` repeats each case in float64.
"""
import math
import os
import sys

import torch

own = False

D = 128      # head_dim
GROUP = 64   # values that share a scale and a bias
SINK = 4     # first positions that eviction always keeps

# (q heads, kv heads): the shapes the package names, and generic ones with
# one q head per kv head and with counts that are no power of two
HEADS = {"0.6b": (16, 8), "4b": (32, 8), "8b": (32, 8), "32b": (64, 8), "mha": (8, 8), "by3": (6, 2), "by5": (10, 2)}
MOST_SCORES = 32 * 2048 * 4096  # of an attention case: the largest listed one
MOST_BYTES = 131072 * 8 * 144   # of cache an attention case reads


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # a decode step's new row, into a cache that is nearly full
        {"name": "write_decode", "op": "write", "heads": "4b", "M": 1, "offset": 4095, "rows": False},
        # a bf16 prompt cache turned into a 4-bit one, an odd number of rows
        {"name": "write_cache_8191", "op": "write", "heads": "8b", "M": 8191, "offset": 0, "rows": False},
        # a prompt chunk from projection rows [M, n_kv_heads * 128], at a row inside the cache
        {"name": "write_chunk_333", "op": "write", "heads": "mha", "M": 333, "offset": 1001, "rows": True},
        # one token of a chat at the context the benchmark decodes at
        {"name": "attn_4b_decode", "op": "attn", "heads": "4b", "M": 1, "past": 4096},
        # one token of a long document, where the cache is all the traffic
        {"name": "attn_8b_decode_128k", "op": "attn", "heads": "8b", "M": 1, "past": 131071},
        # four drafts and their leader verified, 40 query rows per kv head
        {"name": "attn_32b_verify5", "op": "attn", "heads": "32b", "M": 5, "past": 1336},
        # the second half of a prompt
        {"name": "attn_4b_prefill2048", "op": "attn", "heads": "4b", "M": 2048, "past": 2048},
        # a decode step that keeps the positions' weights for a later eviction
        {"name": "weigh_4b_decode", "op": "weigh", "heads": "4b", "M": 1, "past": 8191},
        # the last tokens of a long prompt weigh its positions before it is cut down
        {"name": "weigh_8b_window32", "op": "weigh", "heads": "8b", "M": 32, "past": 16352},
        # a ragged prompt chunk, every position weighed
        {"name": "weigh_0.6b_chunk509", "op": "weigh", "heads": "0.6b", "M": 509, "past": 1000},
        # a full chat cache cut to a quarter
        {"name": "evict_chat", "op": "evict", "heads": "4b", "length": 4352, "budget": 1024, "recent": 256},
        # a long prompt cut to what a decode cache holds
        {"name": "evict_128k", "op": "evict", "heads": "8b", "length": 131001, "budget": 4096, "recent": 512},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "attn", "attn", "weigh", "evict"])
    heads = rng.choice(sorted(HEADS))
    if op == "write":
        return {"op": op, "heads": heads, "M": _log_int(rng, 1, 8191), "offset": rng.choice([0, rng.randint(1, 4096)]),
                "rows": rng.random() < 0.5}
    if op == "evict":
        length = _log_int(rng, 24, 131072)
        budget = rng.randint(16, max(16, min(length, 8192)))
        return {"op": op, "heads": heads, "length": length, "budget": budget, "recent": rng.randint(0, budget - 8)}
    hq, hkv = HEADS[heads]
    M = _log_int(rng, 1, 2048 if op == "attn" else 512)
    most = min(131072, MOST_SCORES // (hq * M) - M, MOST_BYTES // (hkv * 144) - M)
    return {"op": op, "heads": heads, "M": M, "past": _log_int(rng, 1, max(1, most)) - 1}


def _visible(c):
    """Sum over the tokens of the positions each sees."""
    return c["M"] * c["past"] + c["M"] * (c["M"] + 1) // 2


def work(case):
    hq, hkv = HEADS[case["heads"]]
    if case["op"] == "write":
        # bf16 rows in, packed rows out; packed rows in, bf16 rows out; k and v
        return {"bytes": 2 * case["M"] * hkv * (256 + 72) * 2, "flops": 2 * case["M"] * hkv * D * 6}
    if case["op"] == "evict":
        rows = min(case["budget"], case["length"])
        # weights in; kept rows in and out, read back as bf16; their weights and indices out
        return {"bytes": hkv * (4 * case["length"] + rows * (3 * 144 + 2 * 256 + 8)), "flops": hkv * case["length"]}
    L = case["past"] + case["M"]
    cache = hkv * L * 144 + 2 * hq * case["M"] * 256
    more = hkv * L * 8 if case["op"] == "weigh" else 0
    return {"bytes": cache + more, "flops": 4 * D * hq * _visible(case)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows_like(g, heads, rows, kind):
    """Keys: a few channels of every head are larger and off zero, as after
    the rotation of trained keys; values: plain."""
    x = _normal(g, heads, rows, D)
    if kind == "k":
        x = x * (0.5 + torch.rand(heads, 1, D, generator=g, device="cuda")) + 0.7 * _normal(g, heads, 1, D)
    return x.to(torch.bfloat16)


def _quantise(x):
    """bf16 rows [..., 128] -> words [..., 16], scales and biases [..., 2]."""
    y = x.float().reshape(*x.shape[:-1], D // GROUP, GROUP)
    lo, hi = y.amin(-1), y.amax(-1)
    s = ((hi - lo) / 15).to(torch.bfloat16)
    step = s.float()[..., None]
    n = torch.where(step == 0, torch.zeros_like(y), torch.round((y - lo[..., None]) / step).clamp(0, 15))
    n = n.to(torch.int64).reshape(*x.shape[:-1], D // 8, 8)
    words = (n << (4 * torch.arange(8, device=x.device))).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return words, s, lo.to(torch.bfloat16)


def _filled(g, heads, capacity, rows):
    """A cache whose first `rows` rows hold keys and values."""
    c = {}
    for kind in ("k", "v"):
        w = torch.zeros(heads, capacity, D // 8, dtype=torch.int32, device="cuda")
        s = torch.zeros(heads, capacity, 2, dtype=torch.bfloat16, device="cuda")
        b = torch.zeros(heads, capacity, 2, dtype=torch.bfloat16, device="cuda")
        for a in range(0, rows, 32768):
            z = min(rows, a + 32768)
            w[:, a:z], s[:, a:z], b[:, a:z] = _quantise(_rows_like(g, heads, z - a, kind))
        c[kind], c[kind + "_scales"], c[kind + "_biases"] = w, s, b
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hq, hkv = HEADS[case["heads"]]
    st = {"case": case}
    if case["op"] == "write":
        M, off = case["M"], case["offset"]
        st["cache"] = _filled(g, hkv, off + M, 0)
        if case["rows"]:
            k = _rows_like(g, hkv, M, "k").transpose(0, 1).reshape(M, hkv * D).contiguous()
            v = _rows_like(g, hkv, M, "v").transpose(0, 1).reshape(M, hkv * D).contiguous()
            st["k"], st["v"] = (x.view(M, hkv, D).transpose(0, 1) for x in (k, v))
        else:
            st["k"], st["v"] = _rows_like(g, hkv, M, "k"), _rows_like(g, hkv, M, "v")
        return st
    if case["op"] == "evict":
        L = case["length"]
        st["cache"] = _filled(g, hkv, L, L)
        st["into"] = _filled(g, hkv, case["budget"] + 256, 0)
        # few positions draw much, most next to nothing, some exactly as much as others
        w = 30.0 * torch.rand(hkv, L, generator=g, device="cuda") ** 8
        st["weights"] = torch.where(w < 0.01, torch.round(w * 4096) / 4096, w)
        st["weights_into"] = torch.zeros(hkv, case["budget"] + 256, device="cuda")
        return st
    L = case["past"] + case["M"]
    st["cache"] = _filled(g, hkv, L, L)
    st["q"] = (1.5 * _normal(g, hq, case["M"], D)).to(torch.bfloat16)
    if case["op"] == "weigh":
        # what as many tokens before these would have left
        st["weights"] = torch.rand(hkv, L, generator=g, device="cuda") * (2.0 * hq // hkv * case["M"] / L)
    return st


# ---------------------------------------------------------------------------
# the operators
# ---------------------------------------------------------------------------
_spaces = {}  # attention workspaces, one per size, as a program keeps them


def _bmx():
    if "bmx" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "base-mlx_amd"))
    import bmx

    return bmx


def _values(words, scales, biases):
    """float32 [..., 128] that the rows stand for."""
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32)
    n = ((words[..., None] >> shift) & 15).float().reshape(*words.shape[:-1], 2, GROUP)
    return (scales.float()[..., None] * n + biases.float()[..., None]).reshape(*words.shape[:-1], D)


def _plain_attention(q, c, L, past):
    """Softmax weights [n_kv_heads, rep * M, L] and outputs [M, n_heads * 128]."""
    hq, M, _ = q.shape
    k = _values(c["k"][:, :L], c["k_scales"][:, :L], c["k_biases"][:, :L])
    v = _values(c["v"][:, :L], c["v_scales"][:, :L], c["v_biases"][:, :L])
    hkv = k.shape[0]
    rows = q.float().reshape(hkv, hq // hkv * M, D)
    s = torch.matmul(rows, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
    if M > 1:
        j = torch.arange(L, device=q.device)
        t = torch.arange(M, device=q.device) + past
        hidden = (j[None] > t[:, None]).repeat(hq // hkv, 1)
        s.masked_fill_(hidden, -math.inf)
    s -= s.amax(-1, keepdim=True)
    p = torch.exp_(s)
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).reshape(hq, M, D).transpose(0, 1).reshape(M, hq * D)
    return p, out.to(torch.bfloat16)


def _own_cache(st, name="cache"):
    key = "own_" + name
    if key not in st:
        c = st[name]
        st[key] = _bmx().Kv4Cache(c["k"], c["k_scales"], c["k_biases"], c["v"], c["v_scales"], c["v_biases"])
    return st[key]


def run(state):
    case = state["case"]
    op = case["op"]
    if op == "write":
        lo, hi = case["offset"], case["offset"] + case["M"]
        if own:
            cache = _own_cache(state)
            _bmx().kv4_write(state["k"], state["v"], cache, lo)
            return _bmx().kv4_read(cache, lo, hi)
        c, back = state["cache"], []
        for kind in ("k", "v"):
            w, s, b = _quantise(state[kind])
            c[kind][:, lo:hi], c[kind + "_scales"][:, lo:hi], c[kind + "_biases"][:, lo:hi] = w, s, b
            back.append(_values(c[kind][:, lo:hi], c[kind + "_scales"][:, lo:hi],
                                c[kind + "_biases"][:, lo:hi]).to(torch.bfloat16))
        return tuple(back)
    if op == "evict":
        length, budget, recent = case["length"], case["budget"], case["recent"]
        if own:
            into = _own_cache(state, "into")
            kept = _bmx().kv4_evict(_own_cache(state), state["weights"], length, budget, sink=SINK, recent=recent,
                                    into=into, weights_into=state["weights_into"])
            k, v = _bmx().kv4_read(into, 0, budget)
            return kept, k, v, state["weights_into"]
        w = state["weights"]
        mid = w[:, SINK:length - recent]
        best = torch.sort(mid, dim=1, descending=True, stable=True).indices[:, :budget - SINK - recent] + SINK
        j = torch.arange(length, device=w.device)
        ends = torch.cat([j[:SINK], j[length - recent:]]).expand(w.shape[0], -1)
        kept = torch.sort(torch.cat([best, ends], 1), dim=1).values
        src, dst = state["cache"], state["into"]
        for name in src:
            dst[name][:, :budget] = torch.gather(src[name], 1, kept[..., None].expand(-1, -1, src[name].shape[-1]))
        wi = state["weights_into"]
        wi.zero_()
        wi[:, :budget] = torch.gather(w, 1, kept)
        back = [_values(dst[x][:, :budget], dst[x + "_scales"][:, :budget],
                        dst[x + "_biases"][:, :budget]).to(torch.bfloat16) for x in ("k", "v")]
        return kept.to(torch.int32), back[0], back[1], wi
    q, L = state["q"], case["past"] + case["M"]
    if own:
        b, c = _bmx(), _own_cache(state)
        key = (q.shape[0], c.n_kv_heads, case["M"], L, op)
        if key not in _spaces:
            _spaces.clear()
            _spaces[key] = b.attention_kv4_workspace(q.shape[0], c.n_kv_heads, case["M"], L, weigh=op == "weigh")
        if op == "attn":
            return b.attention_kv4(q, c, case["past"], workspace=_spaces[key])
        return b.attention_kv4(q, c, case["past"], weights=state["weights"], workspace=_spaces[key]), state["weights"]
    p, out = _plain_attention(q, state["cache"], L, case["past"])
    if op == "attn":
        return out
    state["weights"] += p.sum(1)
    return out, state["weights"]


# ---------------------------------------------------------------------------
# the same in float64, from the definitions
# ---------------------------------------------------------------------------
def _exact_values(c, kind, rows):
    w = c[kind][:, :rows].to(torch.int64) & 0xFFFFFFFF
    out = torch.empty(*w.shape[:-1], D, dtype=torch.float64, device=w.device)
    for d in range(D):
        n = (w[..., d // 8] // 16 ** (d % 8)) % 16
        out[..., d] = c[kind + "_scales"][:, :rows, d // GROUP].double() * n + c[kind + "_biases"][:, :rows, d // GROUP].double()
    return out


def _exact_write(x):
    """Every value by its group's 16 levels, the nearest (of two, the even one)."""
    y = x.double().unflatten(-1, (2, GROUP))
    lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    step = ((hi - lo) / 15).float().to(torch.bfloat16).double()
    at = torch.where(step > 0, (y - lo) / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(y))
    return (lo + step * torch.round(at).clamp(max=15)).flatten(-2)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(st["k"]), _exact_write(st["v"])
    if case["op"] == "evict":
        length, budget, recent = case["length"], case["budget"], case["recent"]
        w, n = st["weights"].double().cpu(), case["budget"] - SINK - case["recent"]
        k, v = (_exact_values(st["cache"], x, length) for x in ("k", "v"))
        kept, wi = [], torch.zeros(w.shape[0], budget + 256, dtype=torch.float64)
        for h in range(w.shape[0]):
            order = sorted(range(SINK, length - recent), key=lambda j, row=w[h].tolist(): (-row[j], j))
            keep = sorted([*range(SINK), *order[:n], *range(length - recent, length)])
            kept.append(keep)
            wi[h, :budget] = w[h, keep]
        at = torch.tensor(kept, device=k.device)[..., None].expand(-1, -1, D)
        return None, torch.gather(k, 1, at), torch.gather(v, 1, at), wi
    q, past, M = st["q"].double(), case["past"], case["M"]
    L = past + M
    k, v = (_exact_values(st["cache"], x, L) for x in ("k", "v"))
    hq, hkv = q.shape[0], k.shape[0]
    out = torch.empty(M, hq, D, dtype=torch.float64, device=q.device)
    weights = st["weights"].double() if case["op"] == "weigh" else None
    see = torch.arange(L, device=q.device)[None] <= past + torch.arange(M, device=q.device)[:, None]
    for h in range(hq):
        e = torch.where(see, torch.exp(q[h] @ k[h * hkv // hq].T / math.sqrt(D)), torch.zeros((), dtype=torch.float64, device=q.device))
        e = e / e.sum(1, keepdim=True)
        out[:, h] = e @ v[h * hkv // hq]
        if weights is not None:
            weights[h * hkv // hq] += e.sum(0)
    out = out.reshape(M, hq * D)
    return out if weights is None else (out, weights)
