"""The operators of a paged KV cache that many sequences share, as cases that
can be timed and compared: the packed rows of a batch normed, rotated and
appended to their sequences' pages; attention of packed sequences of different
lengths over their pages (single tokens, draft verification, prompts and
chunks of prompts); and attention of a batch whose sequences begin with the
same pages, read once for all.

A layer's cache is k and v [n_pages, n_kv_heads, page_size, 128] bf16; a
sequence's row j lies on page pages[b, j / page_size].  The batch's new tokens
are packed: those of sequence b are rows starts[b] .. starts[b + 1] - 1 and the
last of its lens[b] cached rows.

`run` in its plain form is float32 torch; with `own` it makes the package's
calls.  `exact` repeats each case in float64.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128  # head_dim
EPS, THETA = 1e-6, 1e6

# (q heads, kv heads): the shapes the package names, and generic ones with
# one q head per kv head and with counts that are no power of two
HEADS = {"0.6b": (16, 8), "4b": (32, 8), "8b": (32, 8), "32b": (64, 8), "mha": (8, 8), "by3": (6, 2), "by5": (10, 2)}
PAGES = (16, 32, 64, 128, 256)
MOST_ROWS = 64 * 8192 * 8        # rows x kv heads an attention case caches: the largest listed one
MOST_SCORES = 32 * 4096 * 2049   # visible (query, key) pairs x q heads
MOST_PLAIN = 131072 * 64 * 64    # q heads x keys of one sequence's plain scores, with its tokens
MOST_GATHERED = 160 * 33068 * 8  # rows x kv heads the plain form of a shared prefix gathers


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# A batch: `seqs` sequences with new_lo .. new_hi new tokens each after past_lo
# .. past_hi cached ones (spread over the logarithm, drawn from `mix`), the
# first of them with new_first tokens and past_first cached ones where these
# are not negative; `shared` rows before all of that are common to them.
def _case(op, heads, page, seqs, new=(1, 1), past=(0, 0), first=(-1, -1), shared=0, mix=0, name=None):
    c = {"op": op, "heads": heads, "page": page, "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0],
         "past_hi": past[1], "new_first": first[0], "past_first": first[1], "shared": shared, "mix": mix}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one chat's new token
        _case("append", "4b", 64, 1, past=(4095, 4095), name="append_1"),
        # a decode step of a server's batch
        _case("append", "4b", 16, 64, past=(100, 1500), mix=1, name="append_decode_64"),
        # four ragged prompts packed into one forward
        _case("append", "8b", 64, 4, new=(900, 3500), mix=2, name="append_prompts"),
        # one chat's decode step, where latency counts
        _case("attn", "4b", 64, 1, past=(4096, 4096), name="attn_decode_1"),
        # a server's batch: chats of every length
        _case("attn", "8b", 64, 64, past=(500, 8191), mix=3, name="attn_decode_64"),
        # a long document beside short chats
        _case("attn", "8b", 256, 8, past=(60, 900), first=(1, 131000), mix=4, name="attn_decode_long"),
        # drafts verified for a batch: 5 tokens each, 40 query rows per kv head
        _case("attn", "32b", 16, 16, new=(5, 5), past=(300, 3000), mix=5, name="attn_verify5_16"),
        # packed prompts of different lengths, one of them a single token
        _case("attn", "4b", 64, 6, new=(1, 1500), first=(2049, 0), mix=6, name="attn_prompts"),
        # a prompt's chunk beside a batch's decode steps
        _case("attn", "4b", 32, 32, past=(200, 4000), first=(509, 1503), mix=7, name="attn_chunk_decode"),
        # a whole prompt
        _case("attn", "4b", 64, 1, new=(4096, 4096), name="attn_prompt_4096"),
        # a batch of chats behind one system prompt
        _case("attn", "4b", 64, 64, past=(10, 500), shared=4096, mix=8, name="shared_decode_64"),
        # questions about one long document, answered together
        _case("attn", "8b", 128, 160, past=(20, 300), shared=32768, mix=9, name="shared_document_160"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "verify", "prompts", "shared", "shared_prompts"])
    heads, page, mix = rng.choice(sorted(HEADS)), rng.choice(PAGES), rng.randrange(1 << 30)
    hq, hkv = HEADS[heads]
    while True:
        seqs = _log_int(rng, 1, 160)
        if op == "append":
            if rng.random() < 0.5:
                c = _case("append", heads, page, seqs, past=(_log_int(rng, 1, 100), 1500), mix=mix)
            else:
                c = _case("append", heads, page, min(seqs, 16), new=(1, _log_int(rng, 2, 3500)), past=(0, 50), mix=mix)
        elif op == "decode":
            first = (1, _log_int(rng, 1000, 131000)) if rng.random() < 0.3 else (-1, -1)
            c = _case("attn", heads, page, seqs, past=(rng.randint(0, 500), _log_int(rng, 501, 8191)), first=first, mix=mix)
        elif op == "verify":
            c = _case("attn", heads, page, seqs, new=(rng.randint(1, 3), rng.randint(4, 8)), past=(5, _log_int(rng, 10, 3000)),
                      mix=mix)
        elif op == "prompts":
            first = (_log_int(rng, 1, 4096), rng.choice([0, _log_int(rng, 1, 3000)]))
            c = _case("attn", heads, page, min(seqs, 32), new=(1, _log_int(rng, 1, 1500)), past=(0, rng.choice([0, 700])),
                      first=first, mix=mix)
        elif op == "shared":
            c = _case("attn", heads, page, seqs, past=(0, _log_int(rng, 1, 500)), shared=page * _log_int(rng, 1, 32768 // page),
                      mix=mix)
        else:
            c = _case("attn", heads, page, min(seqs, 32), new=(1, _log_int(rng, 2, 200)), past=(0, 30),
                      shared=page * _log_int(rng, 1, 8192 // page), mix=mix)
        new, past = _lengths(c)
        rows = sum(p + n for p, n in zip(past, new)) + c["shared"]
        if (rows * hkv <= (MOST_ROWS if c["op"] == "attn" else MOST_ROWS // 4) and sum(new) * (hq + hkv) <= 9000 * 40
                and (c["op"] == "append" or (
                    _visible(c) * hq <= MOST_SCORES
                    and max(n * (p + n + c["shared"]) for n, p in zip(new, past)) * hq <= MOST_PLAIN
                    and (not c["shared"] or sum(p + n + c["shared"] for n, p in zip(new, past)) * hkv <= MOST_GATHERED)))):
            return c


def _lengths(c):
    """Per sequence: new tokens, and its own rows before them (past the shared ones)."""
    rng = random.Random(c["mix"])
    new = [_log_int(rng, c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    past = [_log_int(rng, 1 + c["past_lo"], 1 + c["past_hi"]) - 1 for _ in range(c["seqs"])]
    if c["new_first"] >= 0:
        new[0], past[0] = c["new_first"], c["past_first"]
    return new, past


def _visible(c):
    """Sum over the tokens of the positions each sees."""
    return sum(n * (p + c["shared"]) + n * (n + 1) // 2 for n, p in zip(*_lengths(c)))


def work(case):
    hq, hkv = HEADS[case["heads"]]
    new, past = _lengths(case)
    T = sum(new)
    if case["op"] == "append":
        # projection rows in; queries, keys and values out; the norms' and the rotation's arithmetic
        return {"bytes": T * 256 * (2 * hq + 4 * hkv), "flops": T * D * 7 * (hq + hkv)}
    rows = case["shared"] + sum(n + p for n, p in zip(new, past))
    return {"bytes": rows * hkv * 512 + 2 * T * hq * 256, "flops": 4 * D * hq * _visible(case)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    hq, hkv = HEADS[case["heads"]]
    page, shared = case["page"], case["shared"]
    new, past = _lengths(case)
    T = sum(new)
    lens = [shared + p + n for n, p in zip(new, past)]
    need = [-(-n // page) for n in lens]
    common = shared // page
    n_pages = common + sum(n - common for n in need) + 3  # (some pages belong to nobody)
    order = list(range(n_pages))
    rng.shuffle(order)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = common
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[:common] + order[at:at + n - common], dtype=torch.int32)
        at += n - common
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st = {"case": case, "new": new, "lens_host": lens, "pages": table.cuda(), "T": T,
          "starts": torch.tensor(starts, dtype=torch.int32).cuda(), "lens": torch.tensor(lens, dtype=torch.int32).cuda()}
    # keys: a few channels of every head are larger and off zero, as after the
    # rotation of trained keys; values: plain; pages in use or not hold rows
    st["k"] = torch.empty(n_pages, hkv, page, D, dtype=torch.bfloat16, device="cuda")
    st["v"] = torch.empty_like(st["k"])
    wide, off = 0.5 + torch.rand(hkv, 1, D, generator=g, device="cuda"), 0.7 * _normal(g, hkv, 1, D)
    step = max(1, (1 << 27) // (hkv * page * D))
    for a in range(0, n_pages, step):
        z = min(n_pages, a + step)
        st["k"][a:z] = (_normal(g, z - a, hkv, page, D) * wide + off).to(torch.bfloat16)
        st["v"][a:z] = _normal(g, z - a, hkv, page, D).to(torch.bfloat16)
    if case["op"] == "append":
        std = 0.3 + torch.rand(1, hq + 2 * hkv, 1, generator=g, device="cuda")
        x = (_normal(g, T, hq + 2 * hkv, D) * std).to(torch.bfloat16)
        st["q"], st["kn"], st["vn"] = (t.reshape(T, -1).contiguous() for t in x.split([hq, hkv, hkv], 1))
        st["q_norm"], st["k_norm"] = ((1 + 0.2 * _normal(g, D)).to(torch.bfloat16) for _ in "qk")
    else:
        st["q"] = (1.5 * _normal(g, hq, T, D)).to(torch.bfloat16)
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


def _sequences(st):
    """(sequence, first packed row, rows, first position) of those with new tokens."""
    at = 0
    for b, n in enumerate(st["new"]):
        if n:
            yield b, at, n, st["lens_host"][b] - n
        at += n


def _norm_rope(x, w, pos):
    """x [T, heads, 128] normed and rotated, float32; angles in 64 bits."""
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
    freq = THETA ** (-torch.arange(D // 2, dtype=torch.float64, device=x.device) / (D // 2))
    ang = pos.double()[:, None, None] * freq
    c, s = torch.cos(ang).float(), torch.sin(ang).float()
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _positions(st):
    """Of the packed rows: their positions, pages and rows on these."""
    pos, seq = [], []
    for b, _, n, p in _sequences(st):
        pos.append(torch.arange(p, p + n, device="cuda"))
        seq.append(torch.full((n,), b, device="cuda"))
    pos, seq, size = torch.cat(pos), torch.cat(seq), st["case"]["page"]
    return pos, st["pages"].long()[seq, pos // size], pos % size


def _rows_of(st, b, what, rows):
    """The first `rows` rows of sequence b, [n_kv_heads, rows, 128]."""
    size = st["case"]["page"]
    x = st[what][st["pages"][b, :-(-rows // size)].long()]
    return x.transpose(0, 1).reshape(x.shape[1], -1, D)[:, :rows]


def _own_objects(st):
    if "own" not in st:
        b, T = _bmx(), st["T"]
        st["own"] = (b.PagedKvCache(st["k"], st["v"]),
                     b.PagedBatch(st["starts"], st["lens"], st["pages"], T, max_new=max(st["new"])))
    return st["own"]


def run(state):
    case, st = state["case"], state
    hq, hkv = HEADS[case["heads"]]
    T = st["T"]
    if case["op"] == "append":
        if own:
            cache, batch = _own_objects(st)
            q = _bmx().qk_norm_rope_paged(st["q"], st["kn"], st["vn"], st["q_norm"], st["k_norm"], cache, batch, eps=EPS,
                                          theta=THETA)
            return q, st["k"], st["v"]
        pos, page, row = _positions(st)
        q = _norm_rope(st["q"].view(T, hq, D), st["q_norm"], pos).to(torch.bfloat16).transpose(0, 1).contiguous()
        st["k"][page, :, row] = _norm_rope(st["kn"].view(T, hkv, D), st["k_norm"], pos).to(torch.bfloat16)
        st["v"][page, :, row] = st["vn"].view(T, hkv, D)
        return q, st["k"], st["v"]
    if own:
        b = _bmx()
        cache, batch = _own_objects(st)
        key = (hq, hkv, T, case["seqs"], max(st["new"]), case["shared"])
        if key not in _spaces:
            _spaces.clear()
            _spaces[key] = b.attention_paged_workspace(hq, hkv, batch, shared=case["shared"])
        return b.attention_paged(st["q"], cache, batch, shared=case["shared"], workspace=_spaces[key])
    out = torch.empty(T, hq, D, dtype=torch.bfloat16, device="cuda")
    for b, at, n, past in _sequences(st):
        L = past + n
        k, v = (_rows_of(st, b, x, L).float() for x in "kv")
        rows = st["q"][:, at:at + n].float().reshape(hkv, hq // hkv * n, D)
        s = torch.matmul(rows, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(D))
        if n > 1:
            hidden = torch.arange(L, device="cuda")[None] > (past + torch.arange(n, device="cuda"))[:, None]
            s.masked_fill_(hidden.repeat(hq // hkv, 1), -math.inf)
        s -= s.amax(-1, keepdim=True)
        p = torch.exp_(s)
        p /= p.sum(-1, keepdim=True)
        out[at:at + n] = torch.matmul(p, v).reshape(hq, n, D).transpose(0, 1).to(torch.bfloat16)
    return out.view(T, hq * D)


# ---------------------------------------------------------------------------
# the same in float64, from the definitions
# ---------------------------------------------------------------------------
def _exact_rotated(x, w, pos):
    """x [heads, n, 128] by complex numbers."""
    y = x.double()
    y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + EPS) * w.double()
    i = torch.arange(D // 2, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       pos.double()[:, None] * torch.exp(-i / (D // 2) * math.log(THETA)))
    z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
    return torch.cat([z.real, z.imag], -1)


def exact(case, seed):
    st = prepare(case, seed)
    hq, hkv = HEADS[case["heads"]]
    T, size, pages = st["T"], case["page"], st["pages"].tolist()
    if case["op"] == "append":
        q = torch.empty(hq, T, D, dtype=torch.float64, device="cuda")
        k, v = st["k"].double(), st["v"].double()
        for b, at, n, past in _sequences(st):
            pos = torch.arange(past, past + n, device="cuda")
            q[:, at:at + n] = _exact_rotated(st["q"][at:at + n].view(n, hq, D).transpose(0, 1), st["q_norm"], pos)
            kn = _exact_rotated(st["kn"][at:at + n].view(n, hkv, D).transpose(0, 1), st["k_norm"], pos)
            vn = st["vn"][at:at + n].view(n, hkv, D).transpose(0, 1).double()
            j = past
            while j < past + n:  # a page at a time
                end = min(past + n, (j // size + 1) * size)
                on = slice(j % size, j % size + end - j)
                k[pages[b][j // size], :, on] = kn[:, j - past:end - past]
                v[pages[b][j // size], :, on] = vn[:, j - past:end - past]
                j = end
        return q, k, v
    if _visible(case) * hq > 32 * 4096 * 4096:
        return None
    out = torch.empty(T, hq, D, dtype=torch.float64, device="cuda")
    for b, at, n, past in _sequences(st):
        L = past + n
        mine = torch.tensor(pages[b][:-(-L // size)], device="cuda")
        see = torch.arange(L, device="cuda")[None] <= past + torch.arange(n, device="cuda")[:, None]
        for h in range(hkv):
            k, v = (st[x][mine, h].reshape(-1, D)[:L].double() for x in "kv")
            for r in range(h * hq // hkv, (h + 1) * hq // hkv):
                s = torch.mm(st["q"][r, at:at + n].double(), k.t().contiguous()) / math.sqrt(D)
                e = torch.where(see, torch.exp(s - torch.where(see, s, -math.inf).amax(1, keepdim=True)), 0.0)
                out[at:at + n, r] = torch.mm(e / e.sum(1, keepdim=True), v)
    return out.view(T, hq * D)
