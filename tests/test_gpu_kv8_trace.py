"""A trace cannot hold the 8-bit cache's operators, which work through pointers: it is refused, where it would have kept their results as
constants."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("grad", [False, True])
def test_a_trace_is_refused(hip_lib, grad):
    from latentq_llm_amd import ops
    i32 = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()  # noqa: E731
    t, table, n = ref.Cache(3, 2, 64, seed=1).tensors(), i32([[1]]), i32([3])
    before = [x.clone() for x in t]
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    k = q[:, :2].contiguous()
    with torch.set_grad_enabled(grad):
        for call, x in ((lambda x: ops.kv8_attention(x, *t, table, n), q), (lambda x: ops.kv8_append(x, x, *t, table, n) or x * 1, k),
                        (lambda x: ops.kv8_read(*t, x)[0], i32([1]))):
            with pytest.raises(RuntimeError, match="cannot be recorded in a trace"):
                torch.jit.trace(call, x, check_trace=False)
            call(x)
        assert not all(torch.equal(a, b) for a, b in zip(t, before))  # (the last calls append)
