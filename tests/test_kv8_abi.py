"""The C entry points of the paged 8-bit cache on the host: refusals, and the plan of attention. Nothing is launched."""
import ctypes as C

import pytest


@pytest.fixture
def p():
    buf = (C.c_char * 4096)()
    at = C.addressof(buf)
    yield C.c_void_p(at + (-at) % 16), buf


def append_args(p, **change):
    a = dict(k=p, kt=128, kh=64, v=p, vt=128, vh=64, q=None, qt=0, qh=0, qo=None, ot=0, oh=0, cos=None, sin=None, positions=0, rot=0, kc=p, vc=p, ks=p, vs=p,
             blocks=4, table=p, width=2, lens=p, cu=None, batch=2, tokens=4, most=2, heads=2, kv=2, dim=64, dtype=0, stream=None)
    a.update(change)
    return list(a.values())


def attention_args(p, **change):
    a = dict(q=p, qt=128, qh=64, kc=p, vc=p, ks=p, vs=p, blocks=4, table=p, width=2, lens=p, cu=None, batch=2, tokens=4, most=2, len=100, heads=2, kv=2, dim=64,
             dtype=0, scale=1.0, causal=1, window=0, out=p, ot=128, oh=64, lse=None, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, message", [
    (dict(k=None), b"null pointer"), (dict(lens=None), b"null pointer"), (dict(dim=80), b"64, 96, 128 or 256"), (dict(dtype=2), b"dtype"), (dict(kv=0), b"kv head"),
    (dict(tokens=-1), b"negative"), (dict(tokens=3), b"same number of tokens"), (dict(kt=130), b"multiples of 8"), (dict(vh=-8), b"multiples of 8"), (dict(blocks=0), b"pool of blocks"),
    (dict(width=0), b"block table"), (dict(width=1 << 26), b"block table"), (dict(sin=1), b"go together"), (dict(q=1), b"go together"), (dict(q="p", qo="p"), b"needs cos and sin"),
    (dict(cos="p", sin="p", positions=4, rot=24), b"multiple of 16"), (dict(cos="p", sin="p", positions=4, rot=80), b"multiple of 16"),
    (dict(cos="p", sin="p", positions=0, rot=16), b"at least one position"), (dict(v="odd"), b"16-byte aligned"), (dict(kc="odd"), b"16-byte aligned"),
    (dict(kv=40000), b"too many heads"), (dict(tokens=1 << 32, batch=1 << 31), b"too many")])
def test_append_refuses(hip_lib, p, change, message):
    ptr, _ = p
    change = {k: ptr if v == "p" else C.c_void_p(ptr.value + 4) if v == "odd" else v for k, v in change.items()}
    assert hip_lib.lq_kv8_append(*append_args(ptr, **change)) == -1
    assert message in hip_lib.lq_last_error(), hip_lib.lq_last_error()


@pytest.mark.parametrize("change, message", [
    (dict(q=None), b"null pointer"), (dict(out=None), b"null pointer"), (dict(dim=32), b"64, 96, 128 or 256"), (dict(dtype=2), b"dtype"), (dict(heads=3), b"multiple of kv heads"),
    (dict(heads=0), b"multiple of kv heads"), (dict(window=-1), b"window"), (dict(scale=0.0), b"positive"), (dict(scale=-1.0), b"positive"), (dict(scale=float("nan")), b"positive"),
    (dict(scale=float("inf")), b"positive"), (dict(most=0), b"max_tokens"), (dict(tokens=5), b"same number of tokens"), (dict(ot=4), b"multiples of 8"), (dict(out="odd"), b"16-byte aligned"),
    (dict(ws="odd"), b"16-byte aligned"), (dict(ws_bytes=-1), b"workspace"), (dict(blocks=1 << 31), b"pool of blocks"), (dict(len=-1), b"negative"),
    (dict(tokens=1 << 31, batch=1), b"too many")])
def test_attention_refuses(hip_lib, p, change, message):
    ptr, _ = p
    change = {k: C.c_void_p(ptr.value + 4) if v == "odd" else v for k, v in change.items()}
    assert hip_lib.lq_kv8_attention(*attention_args(ptr, **change)) == -1
    assert message in hip_lib.lq_last_error(), hip_lib.lq_last_error()


def test_read_refuses(hip_lib, p):
    ptr, _ = p
    good = [ptr, ptr, ptr, ptr, 4, ptr, 2, 2, 64, 0, ptr, ptr, None]
    for at, value, message in ((0, None, b"null"), (4, 0, b"pool"), (6, -1, b"negative"), (7, 0, b"kv head"), (8, 72, b"64, 96"), (9, 3, b"dtype"), (10, C.c_void_p(ptr.value + 8), b"aligned")):
        args = list(good)
        args[at] = value
        assert hip_lib.lq_kv8_read(*args) == -1 and message in hip_lib.lq_last_error(), hip_lib.lq_last_error()


def test_calls_without_work_launch_nothing(hip_lib, p):
    ptr, _ = p
    assert hip_lib.lq_kv8_append(*append_args(ptr, tokens=0)) == 0
    assert hip_lib.lq_kv8_append(*append_args(ptr, batch=0, tokens=0)) == 0
    assert hip_lib.lq_kv8_attention(*attention_args(ptr, tokens=0)) == 0
    assert hip_lib.lq_kv8_read(ptr, ptr, ptr, ptr, 4, ptr, 0, 2, 64, 0, ptr, ptr, None) == 0


def test_plan_of_attention(hip_lib):
    from latentq_llm_amd import ops
    from latentq_llm_amd._C import LatentQError

    def plan(batch, most, length, heads, kv_heads, dim=128, **more):
        return ops.kv8_attention_plan(batch, batch * most, most, length, heads, kv_heads, dim, compute_units=256, **more)

    # rows of a kv head: tokens times the query heads that share it
    assert plan(1, 1, 1019, 32, 32)[0] == plan(1, 16, 1019, 32, 32)[0] == plan(1, 4, 1019, 32, 8)[0] == plan(1, 16, 64, 8, 8, 256)[0] == "few"
    assert plan(1, 32, 8192, 32, 32)[0] == plan(1, 64, 8192, 32, 32, 64)[0] == "few"
    assert plan(1, 17, 64, 32, 32)[0] == plan(1, 33, 8192, 32, 32)[0] == plan(1, 17, 8192, 8, 8, 256)[0] == plan(1, 65, 8192, 32, 32, 64)[0] == "prompt"
    # enough workgroups, or few keys: nothing to join, no workspace
    assert plan(64, 1, 2048, 32, 32)[1:] == plan(1, 1, 64, 32, 32)[1:] == (0, 0) and plan(1, 8192, 8192, 32, 32)[1:] == (1, 0)
    # few rows on many keys: shares, whose partial results fit the workspace
    for case in ((1, 1, 131072, 32, 8), (2, 5, 4096, 8, 8), (64, 1, 8192, 32, 8)):
        kernel, parts, needed = plan(*case)
        assert parts > 1 and needed == 2 * parts * case[1] * case[3] // case[4] * 129 * 4 <= ops.WORKSPACE_MAX_BYTES
        assert plan(*case, workspace_bytes=0)[1:] == (0, 0)
        assert plan(*case, workspace_bytes=needed // parts * 2)[1] == 2
    # a piece of a prompt: slices
    kernel, parts, needed = plan(1, 512, 16384, 32, 8)
    assert parts > 1 and needed == parts * 512 * 32 * 129 * 4 <= ops.WORKSPACE_MAX_BYTES
    assert plan(1, 512, 16384, 32, 8, workspace_bytes=0)[1:] == (1, 0)
    # a window bounds the keys
    assert plan(1, 1, 131072, 32, 8, window=128)[1] == 0
    assert plan(0, 0, 0, 8, 8) == ("few", 0, 0)
    with pytest.raises(LatentQError, match="multiple of kv heads"):
        plan(1, 1, 100, 8, 3)
