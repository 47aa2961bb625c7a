"""Sizes at the ends of 64 bits at the C entry points of the 8-bit cache. On the host: nothing is launched."""
import pytest

from latentq_llm_amd import ops
from tests.test_kv8_abi import attention_args, p  # noqa: F401  (p: the fixture)


@pytest.mark.parametrize("change", [dict(tokens=1 << 62, batch=1, heads=4, kv=1), dict(tokens=1 << 62, batch=1 << 62, heads=4, kv=4), dict(tokens=1 << 31, batch=1),
                                    dict(tokens=1 << 61, batch=1, heads=8, kv=8), dict(tokens=4, batch=1 << 62, heads=4, kv=4)])
def test_products_of_sizes_do_not_wrap(hip_lib, p, change):  # noqa: F811
    # (the output's strides would be refused next, were these sizes taken)
    assert hip_lib.lq_kv8_attention(*attention_args(p[0], ot=0, oh=0, **change)) == -1
    assert b"too many tokens or sequences" in hip_lib.lq_last_error(), hip_lib.lq_last_error()


def test_blocks_to_read(hip_lib, p):  # noqa: F811
    ptr = p[0]
    # 2^62 blocks of 4 heads; outputs that are not aligned are refused next
    import ctypes as C
    args = [ptr, ptr, ptr, ptr, 4, ptr, 1 << 62, 4, 64, 0, C.c_void_p(ptr.value + 4), ptr, None]
    assert hip_lib.lq_kv8_read(*args) == -1 and b"too many blocks" in hip_lib.lq_last_error()


def test_lengths_and_windows_of_any_size_have_a_plan(hip_lib):
    def plan(length, window=0, tokens=1):
        return ops.kv8_attention_plan(1, tokens, tokens, length, 32, 8, 128, window, compute_units=256)

    top = (1 << 63) - 1
    for tokens in (1, 512):
        assert plan(top, tokens=tokens) == plan((1 << 31) - 1, tokens=tokens)
        for window in ((1 << 31) - 1, 1 << 31, 1 << 40, top - 64, top):
            assert plan(16384, window, tokens) == plan(16384, 0, tokens), window


def test_launches_that_are_too_large_are_refused_with_the_reason(hip_lib, p):  # noqa: F811
    """Many sequences whose number of new tokens is not given: every one may have them all. (A null stream and host pointers: nothing may be
    launched here.)"""
    from tests.test_kv8_abi import append_args
    ptr = p[0]
    assert hip_lib.lq_kv8_attention(*attention_args(ptr, cu=ptr, batch=512, tokens=1 << 17, most=1 << 17, len=512, heads=32, kv=8, width=8, ot=32 * 64)) == -1
    assert b"max_tokens" in hip_lib.lq_last_error() and b"512 sequences" in hip_lib.lq_last_error(), hip_lib.lq_last_error()
    assert hip_lib.lq_kv8_append(*append_args(ptr, cu=ptr, batch=4096, tokens=1 << 20, most=1 << 20)) == -1
    assert b"max_tokens" in hip_lib.lq_last_error(), hip_lib.lq_last_error()
    import ctypes as C
    assert hip_lib.lq_kv8_read(ptr, ptr, ptr, ptr, 4, ptr, 1 << 22, 8, 64, 0, ptr, C.c_void_p(ptr.value), None) == -1 and b"too many blocks" in hip_lib.lq_last_error()
