"""The C entry points of the cache's bookkeeping and of draft verification on the host: refusals and the plan. Nothing is launched."""
import ctypes as C

import pytest


@pytest.fixture
def p():
    buf = (C.c_char * 4096)()
    at = C.addressof(buf)
    yield C.c_void_p(at + (-at) % 16), buf


def at(p, offset):
    return C.c_void_p(p.value + offset)


def resize_args(p, **change):
    a = dict(table=p, width=4, lens=at(p, 256), free=at(p, 512), capacity=8, count=at(p, 768), change=at(p, 1024), batch=3, shared=0, rows=5, cu=at(p, 1280), positions=at(p, 1536),
             slots=at(p, 1792), status=at(p, 2048), stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, message", [
    (dict(table=None), b"null pointer"), (dict(lens=None), b"null pointer"), (dict(free=None), b"null pointer"), (dict(count=None), b"null pointer"), (dict(change=None), b"null pointer"),
    (dict(cu=None), b"null pointer"), (dict(status=None), b"null pointer"), (dict(positions=None), b"null pointer"), (dict(slots=None), b"null pointer"), (dict(batch=-1), b"sequences"),
    (dict(batch=4097), b"4096"), (dict(width=0), b"columns"), (dict(width=1 << 26), b"columns"), (dict(capacity=-1), b"list"), (dict(capacity=1 << 31), b"list"), (dict(shared=-1), b"shared"),
    (dict(shared=5), b"shared"), (dict(rows=1 << 31), b"rows"), (dict(lens=0), b"overlap"), (dict(change=256 + 8), b"overlap"), (dict(free=44), b"overlap"), (dict(count=512 + 28), b"overlap")])
def test_resize_refuses(hip_lib, p, change, message):
    ptr, _ = p
    change = {k: at(ptr, v) if isinstance(v, int) and k in ("lens", "change", "free", "count") else v for k, v in change.items()}
    assert hip_lib.lq_kv8_resize(*resize_args(ptr, **change)) == -1
    assert message in hip_lib.lq_last_error(), hip_lib.lq_last_error()


def verify_args(p, **change):
    a = dict(logits=p, stride=100, draft=p, draft_stride=100, tokens=p, cu=None, batch=2, rows=6, vocab=100, most=3, dtype=0, temperature=1.0, accept=p, sample=p, out=p, accepted=p, change=None, ws=p,
             ws_bytes=1 << 20, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, message", [
    (dict(logits=None), b"null pointer"), (dict(tokens=None), b"null pointer"), (dict(out=None), b"null pointer"), (dict(accepted=None), b"null pointer"), (dict(sample=None), b"sample_draws"),
    (dict(accept=None), b"accept_draws"), (dict(batch=-1), b"rows"), (dict(rows=65536), b"65535 rows"), (dict(rows=-1), b"rows"), (dict(vocab=0), b"logit"), (dict(vocab=1 << 31), b"logit"),
    (dict(dtype=3), b"dtype"), (dict(temperature=-0.5), b"temperature"), (dict(temperature=float("nan")), b"temperature"), (dict(temperature=float("inf")), b"temperature"),
    (dict(temperature=1e-30), b"temperature"), (dict(most=-1), b"max_tokens"), (dict(most=0), b"max_tokens"), (dict(batch=4), b"same number of rows"), (dict(stride=-100), b"strides"),
    (dict(draft_stride=-1), b"strides"), (dict(ws=None), b"workspace"), (dict(ws_bytes=16), b"workspace of"), (dict(ws="odd"), b"aligned"), (dict(cu="p", batch=65536), b"65535 sequences")])
def test_verify_refuses(hip_lib, p, change, message):
    ptr, _ = p
    change = {k: ptr if v == "p" else at(ptr, 8) if v == "odd" else v for k, v in change.items()}
    assert hip_lib.lq_verify_drafts(*verify_args(ptr, **change)) == -1
    assert message in hip_lib.lq_last_error(), hip_lib.lq_last_error()


def test_verify_does_nothing_for_no_sequences(hip_lib, p):
    assert hip_lib.lq_verify_drafts(*verify_args(p[0], batch=0, rows=0)) == 0


@pytest.mark.parametrize("rows, vocab, greedy, draft", [(1, 1, 0, 0), (1, 32000, 0, 0), (40, 32000, 0, 1), (384, 32000, 0, 1), (384, 32000, 1, 0), (65535, 100003, 0, 1), (3, 2 ** 31 - 70000, 0, 0)])
def test_verify_plan(hip_lib, rows, vocab, greedy, draft):
    slices, needed = C.c_int(), C.c_int64()
    assert hip_lib.lq_verify_drafts_plan(rows, rows, vocab, greedy, draft, 256, C.addressof(slices), C.addressof(needed)) == 0
    assert 1 <= slices.value <= -(-vocab // 2048)
    assert needed.value >= rows * slices.value * 16  # a maximum and a sum of every slice


def shared_args(p, **change):
    a = dict(q=p, qt=128, qh=64, kc=p, vc=p, ks=p, vs=p, blocks=4, table=p, width=2, lens=p, cu=None, batch=2, tokens=4, most=2, len=100, shared=1, heads=2, kv=2, dim=64,
             dtype=0, scale=1.0, causal=1, out=p, ot=128, oh=64, lse=None, ws=None, ws_bytes=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, message", [
    (dict(q=None), b"null pointer"), (dict(out=None), b"null pointer"), (dict(table=None), b"null pointer"), (dict(dim=32), b"64, 96, 128 or 256"), (dict(dtype=2), b"dtype"),
    (dict(heads=3), b"multiple of kv heads"), (dict(scale=0.0), b"positive"), (dict(most=0), b"max_tokens"), (dict(tokens=5), b"same number of tokens"), (dict(ot=4), b"multiples of 8"),
    (dict(out="odd"), b"16-byte aligned"), (dict(ws="odd"), b"16-byte aligned"), (dict(ws_bytes=-1), b"workspace"), (dict(blocks=0), b"pool of blocks"), (dict(len=-1), b"negative"),
    (dict(shared=-1), b"shared"), (dict(shared=3), b"shared"), (dict(tokens=1 << 31, batch=1), b"too many"), (dict(oh=32), b"overlap")])
def test_shared_attention_refuses(hip_lib, p, change, message):
    ptr, _ = p
    change = {k: at(ptr, 4) if v == "odd" else v for k, v in change.items()}
    assert hip_lib.lq_kv8_attention_shared(*shared_args(ptr, **change)) == -1
    assert message in hip_lib.lq_last_error(), hip_lib.lq_last_error()


def test_shared_attention_does_nothing_for_no_tokens(hip_lib, p):
    assert hip_lib.lq_kv8_attention_shared(*shared_args(p[0], tokens=0)) == 0
    assert hip_lib.lq_kv8_attention_shared(*shared_args(p[0], tokens=0, batch=0)) == 0


def test_shared_attention_plan_stays_within_its_workspace(hip_lib):
    """Slices that cover the keys, and the bytes they take, over the sizes; with little workspace fewer slices, then none."""
    from latentq_llm_amd import ops
    for batch, most, group, dim, shared, own in [(2, 1, 1, 64, 2, 1), (64, 1, 4, 128, 128, 512), (16, 1, 4, 128, 2048, 257), (8, 5, 1, 64, 64, 640), (500, 1, 8, 256, 9, 3000), (3, 8, 8, 96, 1, 8)]:
        for kv_heads in (1, 8, 32):
            slot = batch * most * group * kv_heads * (dim + 1) * 4
            before = None
            for room in sorted((64 << 20, 9 * slot, 4 * slot, 2 * slot, 2 * slot - 1, 0), reverse=True):
                prefix, own_slices, needed = ops.kv8_attention_shared_plan(batch, batch * most, most, shared * 64 + own, group * kv_heads, kv_heads, dim, shared, room, 256)
                assert needed <= max(room, 0)
                if prefix:
                    assert 1 <= prefix <= shared and 1 <= own_slices <= -(-own // 64) and needed == (prefix + own_slices) * slot
                    assert ops.kv8_attention_shared_plan(batch, batch * most, most, shared * 64 + own, group * kv_heads, kv_heads, dim, shared, needed, 256) == (prefix, own_slices, needed)
                assert before is None or prefix + own_slices <= before
                before = prefix + own_slices
