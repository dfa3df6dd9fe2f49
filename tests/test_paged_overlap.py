"""The paged KV cache's entry points refuse buffers that they write over others
that they read or write (no GPU work is issued by any call here)."""
import bmx
from test_paged import P, append, attend, batch, kv

CACHE = 10 * 2 * 16 * 256        # bytes of kv()'s keys
Q, KV = 6 * 4 * 256, 6 * 2 * 256  # of the batch's packed rows, 4 heads over 2


def refused(rc):
    return rc == bmx.BMX_E_ARG and "overlap" in bmx.last_error()


def test_append_to_keys_over_values():
    for v in (P, P + 16, P + CACHE - 16, P - CACHE + 16):
        assert refused(append(kv(v=v), batch())), hex(v)


def test_append_over_what_it_reads_or_writes():
    for c in (P, 2 * P):
        for n, size in (("q", Q), ("kp", KV), ("vp", KV), ("qn", 256), ("kn", 256), ("out", Q)):
            for at in (c, c + CACHE - 16, c - size + 16):
                assert refused(append(kv(), batch(), **{n: at})), (n, hex(at))
        for n, size in (("starts", 16), ("lens", 12), ("pages", 48)):
            for at in (c, c + CACHE - 4, c - size + 4):
                assert refused(append(kv(), batch(**{n: at}))), (n, hex(at))
    for n, size in (("qn", 256), ("kn", 256)):
        for out in (0, size - 16, 16 - Q):
            assert refused(append(kv(), batch(), out={"qn": 9, "kn": 10}[n] * P + out))
    for at, size in ((3 * P, 16), (4 * P, 12), (5 * P, 48)):
        assert refused(append(kv(), batch(), out=at)) and refused(append(kv(), batch(), out=at - Q + 16))


def test_attention_over_what_it_reads():
    need = bmx.load().bmx_attention_paged_workspace_bytes(4, 2, 6, 3, 3, 0)
    reads = {"k": (P, CACHE), "v": (2 * P, CACHE), "starts": (3 * P, 16), "lens": (4 * P, 16), "pages": (5 * P, 48), "q": (6 * P, Q)}
    for n, (at, size) in reads.items():
        for to in (at, at + size - 16, at - Q + 16):
            assert refused(attend(kv(), batch(), out=to)), (n, "out")
        for to in (at, at + size - 16, at - need + 16):
            assert refused(attend(kv(), batch(), ws=to, wsb=need)), (n, "workspace")
    for to in (11 * P, 11 * P + Q - 16, 11 * P - need + 16):
        assert refused(attend(kv(), batch(), ws=to, wsb=need))
