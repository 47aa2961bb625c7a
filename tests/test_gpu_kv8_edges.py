"""The 8-bit cache's operators at the ends of what they take: lengths near 2^31, scales of zero, outputs whose rows overlap."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


@pytest.mark.parametrize("back", [0, 1, 63, 64, 70])
@pytest.mark.parametrize("tokens", [2, 70])
def test_appending_at_the_largest_lengths(hip_lib, tokens, back):
    """A sequence length near 2^31 - 1 on the device: the tokens lie beyond the table and are not stored, the queries take the tables'
    last row, and nothing outside the operands is touched."""
    from latentq_llm_amd import ops
    dim, heads, lens = 64, 4, [2 ** 31 - 1 - back]
    cache = ref.Cache(3, 2, dim, seed=1)
    tensors, table = cache.tensors(), np.array([[2, 1]], np.int32)
    k, q = rows((tokens, 2, dim), BF16, 2), rows((tokens + 200, heads, dim), BF16, 3)
    cos, sin = ref.tables(90, dim)
    room = torch.full_like(q, 7.0).cuda()  # the output's rows in the middle of others
    out = room[100:100 + tokens]
    got = ops.kv8_append(k.cuda(), k.cuda(), *tensors, i32(table), i32(lens), q=q[100:100 + tokens].cuda(), cos=torch.from_numpy(cos).cuda(),
                         sin=torch.from_numpy(sin).cuda(), q_out=out)
    want = torch.from_numpy(ref.rotated(q[100:100 + tokens].float().numpy(), cos[[89] * tokens], sin[[89] * tokens])).to(BF16)
    assert got is out and torch.equal(out.cpu(), want) and (room[:100] == 7).all() and (room[100 + tokens:] == 7).all()
    codes = ref.from_layout(*tensors[:2])
    assert all(np.array_equal(a, b) for a, b in zip(codes, cache.codes))
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(tensors[2:], cache.scale))
