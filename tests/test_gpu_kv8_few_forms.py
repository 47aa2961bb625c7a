"""Every form of the few-rows kernel of lq_kv8_attention: 1, 2 and 4 tiles of 16 rows, whole units and equal shares, both ways of joining. Each
case asserts the plan that takes it there. Bounds are those of tests/kv8_ref.py."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


class Case:
    def __init__(self, lens, news, heads, kv_heads, dim, dtype, seed=0):
        self.lens, self.news, self.heads, self.kv_heads, self.dim = lens, news, heads, kv_heads, dim
        pool = sum(-(-n // 64) for n in lens) + 1
        self.cache, self.table = ref.Cache(pool, kv_heads, dim, seed=seed), ref.blocks_of(lens, pool, seed=seed)
        self.q = torch.randn((sum(news), heads, dim), generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
        self.device = self.q.cuda(), *self.cache.tensors(), i32(self.table), i32(lens)
        self.cu = None if len(set(news)) == 1 else i32(np.concatenate([[0], np.cumsum(news)]))

    def plan(self, workspace, window=0):
        from latentq_llm_amd import ops
        return ops.kv8_attention_plan(len(self.lens), sum(self.news), max(self.news), max(self.lens), self.heads, self.kv_heads, self.dim, window, workspace)

    def shared(self, **how):
        from latentq_llm_amd import ops
        kernel, parts, _ = self.plan(ops.WORKSPACE_MAX_BYTES, how.get("window", 0))
        assert kernel == "few" and parts > 1
        return parts, ops.kv8_attention(*self.device, cu_tokens=self.cu, max_tokens=max(self.news), max_len=max(self.lens), return_lse=True, **how)

    def whole(self, causal=True, window=0):
        """Without a workspace there is nothing to share the keys through."""
        from latentq_llm_amd import _C
        assert self.plan(0, window)[:2] == ("few", 0)
        q, kc, vc, ks, vs, table, lens = self.device
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        _C.call("lq_kv8_attention", q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), kc.shape[0], table.data_ptr(),
                table.shape[1], lens.data_ptr(), None if self.cu is None else self.cu.data_ptr(), len(self.lens), q.shape[0], max(self.news), max(self.lens), self.heads,
                self.kv_heads, self.dim, int(q.dtype == F16), self.dim ** -0.5, int(causal), window, out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(), None, 0,
                torch.cuda.current_stream().cuda_stream)
        return out, lse

    def check(self, got, **how):
        want, (want_lse, lse_bound), bound = ref.attention(self.cache, self.q, self.table, self.lens, self.news, **how)
        for out, lse in got:
            off = np.abs(out.cpu().double().numpy() - want)
            assert (off <= bound).all(), np.argwhere(~(off <= bound))[:4].tolist()
            lse, seen = lse.cpu().double().numpy(), np.isfinite(want_lse)
            assert np.array_equal(np.isfinite(lse), seen) and (np.abs(lse[seen] - want_lse[seen]) <= lse_bound[seen]).all()


ROWS = {17: (17, 1), 32: (8, 4), 33: (11, 3), 63: (9, 7), 64: (16, 4)}  # rows of a kv head: (tokens, query heads that share it)
LONG = {64: 3100, 96: 2100, 128: 2100}  # keys from which equal shares are taken, and some
FORMS = [(d, r) for d in (64, 96) for r in ROWS] + [(128, 17), (128, 32)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim, rows", FORMS)
def test_rows_beyond_one_tile(hip_lib, dim, rows, dtype):
    tokens, group = ROWS[rows]
    c = Case([LONG[dim], LONG[dim] - 51], [tokens] * 2, 2 * group, 2, dim, dtype, seed=rows)
    c.check([c.shared()[1], c.whole()])


@pytest.mark.parametrize("causal, windowed", [(True, False), (False, False), (True, True), (False, True)])
@pytest.mark.parametrize("dim, rows", FORMS)
def test_sequences_of_different_lengths(hip_lib, dim, rows, causal, windowed):
    """All, some, one and none of a sequence's rows new, more new tokens than tokens, a sequence without any."""
    tokens, group = ROWS[rows]
    how = {"causal": causal, "window": LONG[dim] - 50 if windowed else 0}
    c = Case([LONG[dim], 130, 0, LONG[dim] + 100, tokens - 2, 64], [tokens, 1, 3, tokens - 1, tokens, 0], group, 1, dim, BF16, seed=rows)
    c.check([c.shared(**how)[1], c.whole(**how)], **how)


@pytest.mark.parametrize("tokens, group", [(1, 1), (3, 5), (16, 1)])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("units", ["few", "many"])
def test_both_ways_of_joining(hip_lib, units, dim, tokens, group):
    """A unit in many pieces, which several threads of a row join, and in few."""
    lens = [3200] if units == "few" else [3100 + 7 * i for i in range(18)]
    c = Case(lens, [tokens] * len(lens), 4 * group if units == "many" else group, 4 if units == "many" else 1, dim, F16, seed=tokens)
    parts, got = c.shared()
    assert (parts > 8 * len(lens) * c.kv_heads) == (units == "few")
    if units == "many" and tokens * group > 1:  # the reference takes its time: the shortest, the longest and one between
        c.lens, c.news = c.lens[:3], c.news[:3]
        n = 3 * tokens
        c.table, c.q, got = c.table[:3], c.q[:n], tuple(x[:n] for x in got)
    c.check([got])


@pytest.mark.parametrize("rows", [33, 64])
@pytest.mark.parametrize("dim", [64, 96])
def test_many_rows_joined_in_few_pieces(hip_lib, dim, rows):
    tokens, group = ROWS[rows]
    c = Case([3000 + 64 * i for i in range(20)], [tokens] * 20, 4 * group, 4, dim, BF16, seed=dim)
    parts, got = c.shared()
    assert parts <= 8 * 20 * 4
    c.lens, c.news, c.table, c.q = c.lens[:2], c.news[:2], c.table[:2], c.q[:2 * tokens]
    c.check([tuple(x[:2 * tokens] for x in got)])


@pytest.mark.parametrize("tokens, length, heads, kv_heads, dim", [(31, 9619, 32, 8, 96), (195, 13664, 12, 12, 64), (17, 4000, 4, 4, 96)])
def test_a_captured_call_gives_the_bits_of_an_eager_one(hip_lib, tokens, length, heads, kv_heads, dim):
    """It gets no more workspace than its plan names, an eager one the whole buffer."""
    from latentq_llm_amd import ops
    c = Case([length], [tokens], heads, kv_heads, dim, BF16, seed=tokens)
    assert c.plan(ops.WORKSPACE_MAX_BYTES)[1] > 1
    more = dict(max_tokens=tokens, max_len=length)
    q, rest = c.device[0], c.device[1:]
    given = [q.clone(), torch.randn_like(q), torch.randn_like(q)]
    want = [ops.kv8_attention(x, *rest, **more) for x in given]
    q, graph = q.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.kv8_attention(q, *rest, **more)
    for i in (1, 2, 0, 1):
        q.copy_(given[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
