"""Arguments of the 8-bit cache's operators that are not what the native binding converts: the wrappers take or refuse them."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


@pytest.fixture
def call():
    lens = [200, 150]
    cache = ref.Cache(8, 2, 64, seed=1)
    tensors, table = cache.tensors(), i32(ref.blocks_of(lens, 8))
    q = torch.randn((6, 4, 64), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()

    def attend(**more):
        from latentq_llm_amd import ops
        return ops.kv8_attention(q, *tensors, table, i32(lens), **more)
    attend.tensors, attend.table, attend.q = tensors, table, q
    return attend


def test_numbers_that_are_whole(hip_lib, call):
    for name, value, same in (("window", 70.0, 70), ("window", np.float32(70), 70), ("max_len", 200.0, 200), ("max_tokens", 3.0, 3), ("window", None, 0),
                              ("scale", np.float32(0.125), 0.125), ("scale", 1, 1.0), ("causal", 0, False), ("causal", np.bool_(False), False)):
        assert torch.equal(call(**{name: value}), call(**{name: same})), name
    assert torch.equal(call(cu_tokens=i32([0, 3, 6]), max_tokens=3.0), call())


def test_what_cannot_be_converted(hip_lib, call):
    from latentq_llm_amd import ops
    for kind, more in ((ValueError, dict(window="x")), (ValueError, dict(max_len="x")), ((TypeError, ValueError), dict(max_tokens="x")), (ValueError, dict(scale="x")),
                       (RuntimeError, dict(causal=torch.ones(2))), (TypeError, dict(window=[70]))):
        with pytest.raises(kind):
            call(**more)
    k = call.q[:, :2].contiguous()
    with pytest.raises((TypeError, ValueError)):
        ops.kv8_append(k, k, *call.tensors, call.table, i32([3, 3]), max_tokens="x")
    before = [t.clone() for t in call.tensors]
    ops.kv8_append(k, k, *call.tensors, call.table, i32([3, 3]), max_tokens=3.0)
    after, tensors = [t.clone() for t in call.tensors], call.tensors
    for t, b in zip(tensors, before):
        t.copy_(b)
    ops.kv8_append(k, k, *tensors, call.table, i32([3, 3]), max_tokens=3)
    assert all(torch.equal(a, t) for a, t in zip(after, tensors))


def test_sizes_of_a_layer_that_are_not_integers(hip_lib):
    """The same of the other calls of the binding: the wrapper's checks speak, not the interpreter."""
    from latentq_llm_amd import ops
    x = torch.zeros((2, 256), dtype=BF16, device="cuda")
    codes, s = torch.zeros(128 * 128, dtype=torch.uint8, device="cuda"), torch.zeros(256, dtype=BF16, device="cuda")
    with pytest.raises(Exception) as e:
        ops.a16w4_forward(x, codes, s, s, (128.0, 256))
    assert not isinstance(e.value, SystemError)


def test_windows_of_any_size(hip_lib, call):
    """Beyond every position: as none, also for sequences with fewer tokens than new ones."""
    from latentq_llm_amd import ops
    want = call()
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1, 2 ** 63, 2 ** 64 + 5, 2 ** 70):
        assert torch.equal(call(window=window), want), window
    q = call.q.repeat(20, 1, 1)
    short = dict(cu_tokens=i32([0, 100, 120]), max_tokens=100)
    lens = i32([40, 20])
    want = ops.kv8_attention(q, *call.tensors, call.table, lens, **short)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 63 - 1):
        assert torch.equal(ops.kv8_attention(q, *call.tensors, call.table, lens, window=window, **short), want), window
