"""Outputs whose rows overlap, which no order of writing makes right, are refused by the C entry points. On the host: nothing is launched."""
import ctypes as C

from tests.test_kv8_abi import append_args, attention_args, p  # noqa: F401  (p: the fixture)


def apart(n0, s0, n1, s1, dim):
    seen = set()
    for i in range(n0):
        for j in range(n1):
            row = range((i * s0 + j * s1) // 8, (i * s0 + j * s1 + dim) // 8)
            if not seen.isdisjoint(row):
                return False
            seen.update(row)
    return True


def test_attention(hip_lib, p):  # noqa: F811
    """All small strides: those that overlap are refused, the others come as far as the next check."""
    ptr, _ = p
    for tokens in (1, 2, 3, 5):
        for heads in (1, 2, 6):
            for st in range(0, 500, 24):
                for sh in range(0, 500, 24):
                    rc = hip_lib.lq_kv8_attention(*attention_args(ptr, batch=1, tokens=tokens, most=tokens, heads=heads, kv=1, ot=st, oh=sh, ws_bytes=-1))
                    want = b"workspace" if apart(tokens, st, heads, sh, 64) else b"rows of the output overlap"
                    assert rc == -1 and want in hip_lib.lq_last_error(), (tokens, heads, st, sh, hip_lib.lq_last_error())


def test_append(hip_lib, p):  # noqa: F811
    ptr, _ = p
    for change in (dict(ot=64, oh=64), dict(ot=0, oh=64), dict(ot=128, oh=0), dict(ot=96, oh=64), dict(ot=64, oh=192), dict(ot=1 << 62, oh=8)):
        args = append_args(ptr, q=ptr, qt=128, qh=64, qo=ptr, cos=ptr, sin=ptr, positions=4, rot=64, **change)
        assert hip_lib.lq_kv8_append(*args) == -1 and b"rows of q_out overlap" in hip_lib.lq_last_error(), change
