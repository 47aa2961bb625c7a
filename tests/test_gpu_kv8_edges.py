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


def call(tensors, q, table, lens, news, **more):
    from latentq_llm_amd import ops
    cu = None if len(set(news)) == 1 else i32(np.concatenate([[0], np.cumsum(news)]))
    return ops.kv8_attention(q.cuda(), *tensors, i32(table), i32(lens), cu_tokens=cu, **more)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("lens, tokens", [([400], 1), ([1900], 3), ([400], 90), ([700], 500), ([8300], 70)])
def test_value_scales_of_zero(hip_lib, lens, tokens, dim):
    """Blocks whose value scale is 0, negative zero, subnormal or under 2^-97, as of blocks of zeros: their keys have their weight, their values
    add nothing. One workgroup to a row, shares, one tile, two sides and slices of the keys."""
    pool = -(-lens[0] // 64) + 2
    table = ref.blocks_of(lens, pool, seed=1)
    q = rows((tokens, 4, dim), BF16, 6)
    for seed, scales in ((0, [0.0]), (1, [0.0, -0.0, 1e-40, 2.0 ** -126, 2.0 ** -98]), (2, [2.0 ** -97])):
        cache = ref.Cache(pool, 2, dim, seed=5 + seed)
        rng = np.random.default_rng(seed)
        for h in range(2):
            for b in range(pool):
                if rng.random() < 0.5:
                    cache.scale[1][b, h] = np.float32(rng.choice(scales))
        cache.scale[1][table[0, 0]] = scales[0]  # among them the first tile
        want, (want_lse, lse_bound), bound = ref.attention(cache, q, table, lens, [tokens])
        out, lse = call(cache.tensors(), q, table, lens, [tokens], return_lse=True)
        got, off = out.cpu().double().numpy(), np.abs(out.cpu().double().numpy() - want)
        assert np.isfinite(got).all() and (off <= bound + 127 * 2.0 ** -97).all(), (seed, float((off / bound).max()))
        assert (np.abs(lse.cpu().double().numpy() - want_lse) <= lse_bound).all()


@pytest.mark.parametrize("tokens", [1, 90])
def test_value_scales_that_are_all_zero(hip_lib, tokens):
    cache = ref.Cache(6, 2, 64, seed=5)
    cache.scale[1][:] = 0
    table = ref.blocks_of([300], 6)
    assert not call(cache.tensors(), rows((tokens, 4, 64), BF16, 6), table, [300], [tokens]).any()


def test_outputs_whose_rows_overlap(hip_lib):
    """Refused in every entry; rows that lie apart in unusual strides are not."""
    from latentq_llm_amd import ops
    dim, lens = 64, [70]
    cache = ref.Cache(3, 2, dim)
    t, table, n = cache.tensors(), i32(ref.blocks_of(lens, 3)), i32(lens)
    q, k = rows((6, 4, dim), BF16, 1).cuda(), rows((6, 2, dim), BF16, 2).cuda()
    cos, sin = (torch.from_numpy(x).cuda() for x in ref.tables(70, dim))
    room = torch.zeros(20000, dtype=BF16, device="cuda")
    want = ops.kv8_attention(q, *t, table, n)
    turned = ops.kv8_append(k, k, *ref.Cache(3, 2, dim).tensors(), table, n, q=q, cos=cos, sin=sin)
    for strides, apart in (((64, 64), False), ((128, 64), False), ((64, 128), False), ((0, 64), False), ((256, 64), True), ((64, 384), True), ((192, 128), False),
                           ((192, 64), False), ((512, 64), True), ((320, 1600), False), ((96, 576), True), ((192, 704), True)):
        out = room.as_strided((6, 4, dim), (*strides, 1))
        if apart:
            assert torch.equal(ops.kv8_attention(q, *t, table, n, out=out), want), strides
            assert torch.equal(ops.kv8_append(k, k, *ref.Cache(3, 2, dim).tensors(), table, n, q=q, cos=cos, sin=sin, q_out=out), turned), strides
        else:
            with pytest.raises(ValueError, match="heads of their own"):
                ops.kv8_attention(q, *t, table, n, out=out)
            with pytest.raises(ValueError, match="heads of their own"):
                ops.kv8_append(k, k, *t, table, n, q=q, cos=cos, sin=sin, q_out=out)
