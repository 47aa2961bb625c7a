"""lq_kv8_attention_shared of sequences that have different numbers of new tokens, in batches that one look by 64 lanes covers and in larger ones, with the bound of their number exact and far above:
every call takes the shared form, by the plan of just its arguments, and is compared with attention in 64 bits (bounds: tests/test_gpu_kv8_shared.py). Rows go through matrix tiles of 16 or 32."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref
from tests.test_gpu_kv8_shared import holds, i32, rows, table_of

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def check(shared, lens, news, heads, kv_heads, dim, dtype, seed, max_tokens, behind=0, causal=True):
    """behind: rows that no sequence has, which stay as they are."""
    from latentq_llm_amd import ops
    pool = shared + sum(max(0, -(-n // 64) - shared) for n in lens) + 2
    cache = ref.Cache(pool, kv_heads, dim, seed=seed)
    table, total = table_of(lens, shared, pool, seed), sum(news)
    q = rows((total + behind, heads, dim), dtype, seed + 1)
    bound = total + behind if max_tokens is None else max_tokens
    plan = ops.kv8_attention_shared_plan(len(lens), total + behind, min(bound, total + behind), table.shape[1] * 64, heads, kv_heads, dim, shared)
    assert plan[0] > 0, plan
    out = torch.full((total + behind, heads, dim), 7.0, dtype=dtype, device="cuda")
    cu = np.concatenate([[0], np.cumsum(news)])
    got, lse = ops.kv8_attention_shared(q.cuda(), *cache.tensors(), i32(table), i32(lens), shared, cu_tokens=i32(cu), max_tokens=max_tokens, causal=causal, out=out, return_lse=True)
    want, (want_lse, lse_bound), limit = ref.attention(cache, q[:total], table, lens, news, causal=causal)
    assert (got[total:] == 7).all()
    seen = np.ones(total, dtype=bool)
    if max_tokens is not None:  # rows of a sequence beyond it stay as they are, too
        for i, n in enumerate(news):
            seen[cu[i] + max_tokens:cu[i] + n] = False
    assert (got[:total][torch.from_numpy(~seen)] == 7).all()
    at = torch.from_numpy(seen).nonzero()[:, 0]
    holds(got[:total][at.cuda()], want[seen], (limit + (max(lens) / 32 + 4) * 2.0 ** -24 * 255 * cache.scale[1].max())[seen])
    lse, want_lse, lse_bound = lse[:total].cpu().double().numpy()[seen], want_lse[seen], lse_bound[seen]
    assert np.array_equal(np.isinf(lse), np.isinf(want_lse))
    fine = np.isfinite(want_lse)
    assert (np.abs(lse[fine] - want_lse[fine]) <= lse_bound[fine]).all()


def ragged(batch, seed, most=5, longest=1500):
    """Numbers of new tokens from none to `most`, lengths from nothing to more than is shared; rows before position 0 among them."""
    rng = np.random.default_rng(seed)
    news, lens = [int(n) for n in rng.integers(0, most + 1, batch)], [int(n) for n in rng.integers(0, longest, batch)]
    news[0], lens[0], news[1], lens[1], news[-1], lens[-1] = most, 14 * 64, 3, 0, 2, 14 * 64 + 1
    return news, lens


@pytest.mark.parametrize("bound", ["exact", "all"])
@pytest.mark.parametrize("batch", [3, 63, 64, 65, 130, 200])
def test_batches_of_different_numbers(hip_lib, batch, bound):
    news, lens = ragged(batch, batch)
    for heads, kv_heads, dim, dtype in ((8, 2, 64, BF16), (3, 3, 128, F16)):
        check(14, lens, news, heads, kv_heads, dim, dtype, batch, max(news) if bound == "exact" else None, behind=batch % 7)
    check(14, lens, news, 8, 2, 64, BF16, batch, max(news) if bound == "exact" else None, causal=False)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("batch, long, heads, kv_heads", [(30, 40, 4, 2), (9, 17, 16, 2), (70, 33, 4, 1), (25, 100, 3, 3), (129, 300, 2, 1)])
def test_one_sequence_with_many(hip_lib, batch, long, heads, kv_heads, dim, dtype):
    """Many rows of one sequence, first, in the middle or last, among single tokens and sequences without any: those beyond the rows that a sequence is taken to have."""
    for at in (0, batch // 2, batch - 1):
        news = [1 if i % 9 else 0 for i in range(batch)]
        news[at] = long
        lens = [14 * 64 + 1 + 37 * i % 200 for i in range(batch)]
        lens[at] = 14 * 64 + long - 3
        check(14, lens, news, heads, kv_heads, dim, dtype, batch + at, long if at else None, behind=2)


@pytest.mark.parametrize("batch", [20, 64, 100])
def test_several_with_many(hip_lib, batch):
    """Numbers around the tiles of 16 and 32 rows, next to each other and apart."""
    news = [1] * batch
    for i, n in zip((0, 1, 2, 7, 8, batch - 3, batch - 1), (33, 31, 1, 17, 48, 16, 65)):
        news[i] = n
    lens = [14 * 64 + n + 5 * i for i, n in enumerate(news)]
    for heads, kv_heads, dim in ((2, 2, 64), (4, 1, 128)):
        for bound in (None, 65, 40):  # (40: rows beyond it are left as they are)
            check(14, lens, news, heads, kv_heads, dim, BF16, batch, bound)


def test_more_sequences_than_one_look_covers_twice(hip_lib):
    """More than 64 x 64 sequences: three looks."""
    news = [1 if i % 3 else 0 for i in range(4200)]
    news[4100], news[7] = 30, 21
    lens = [14 * 64 + (n + i % 5 if n else 0) for i, n in enumerate(news)]
    check(14, lens, news, 1, 1, 64, BF16, 1, None, behind=3)


def test_equal_numbers_by_the_c_entry_with_a_bound_above(hip_lib):
    """Without first rows max_tokens may be a bound, too."""
    from latentq_llm_amd import _C, ops
    batch, tokens, shared, heads = 30, 2, 14, 4
    lens = [14 * 64 + 2 + i for i in range(batch)]
    cache = ref.Cache(80, 2, 64, seed=3)
    table, q = table_of(lens, shared, 80, 3), rows((batch * tokens, heads, 64), F16, 4)
    want, _, bound = ref.attention(cache, q, table, lens, [tokens] * batch)
    t, tab, length, x = cache.tensors(), i32(table), i32(lens), q.cuda()
    width = tab.shape[1]
    exact = ops.kv8_attention_shared_plan(batch, batch * tokens, tokens, width * 64, heads, 2, 64, shared)
    for most in (tokens, 7, batch * tokens, 10 ** 6):
        plan = ops.kv8_attention_shared_plan(batch, batch * tokens, most, width * 64, heads, 2, 64, shared)
        assert plan == exact and plan[0] > 0
        ws, out = torch.empty(plan[2], dtype=torch.uint8, device="cuda"), torch.zeros_like(x)
        _C.call("lq_kv8_attention_shared", x.data_ptr(), x.stride(0), x.stride(1), *(c.data_ptr() for c in t), 80, tab.data_ptr(), width, length.data_ptr(), None, batch, batch * tokens, most,
                width * 64, shared, heads, 2, 64, 1, 0.125, 1, out.data_ptr(), out.stride(0), out.stride(1), None, ws.data_ptr(), plan[2], torch.cuda.current_stream().cuda_stream)
        holds(out, want, bound + (max(lens) / 32 + 4) * 2.0 ** -24 * 255 * cache.scale[1].max())


def test_first_rows_that_are_none(hip_lib):
    """Broken first rows of many sequences: other values, nothing outside the output, and an end."""
    from latentq_llm_amd import ops
    batch, shared = 70, 14
    cache = ref.Cache(30, 2, 64, seed=5)
    table = i32(np.tile(np.arange(16, dtype=np.int32), (batch, 1)))
    q = rows((90, 4, 64), BF16, 6).cuda()
    assert ops.kv8_attention_shared_plan(batch, 90, 90, 1024, 4, 2, 64, shared)[0] > 0
    rng = np.random.default_rng(7)
    for n in range(8):
        cu = rng.integers(-5, 95, batch + 1) if n < 4 else rng.integers(-2 ** 31, 2 ** 31, batch + 1)
        if n % 2:
            cu = np.sort(cu)[::-1] if n > 5 else np.sort(cu)
        out = torch.full((100, 4, 64), 7.0, dtype=BF16, device="cuda")
        ops.kv8_attention_shared(q, *cache.tensors(), table, i32([1000] * batch), shared, cu_tokens=i32(cu.astype(np.int64)), out=out[5:95])
        torch.cuda.synchronize()
        assert (out[:5] == 7).all() and (out[95:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("own", [(1, 2), (64, 3000), (255, 256), (257, 1), (700, 0, 1400), (4000, 4001, 5, 130, 1025)])
def test_own_keys_by_many_workgroups(hip_lib, own, dim, dtype):
    """Few sequences, whose own keys are shared among workgroups, four tiles each in turn; bounds of the lengths that are right, too small, too large, and none."""
    from latentq_llm_amd import ops
    shared, heads, kv_heads = 14, 4, 2
    lens = [64 * shared + n for n in own]
    pool = shared + sum(-(-n // 64) for n in own) + 2
    cache = ref.Cache(pool, kv_heads, dim, seed=dim)
    table, q = table_of(lens, shared, pool, dim, width=shared + 70), rows((len(own), heads, dim), dtype, 3)
    want, _, bound = ref.attention(cache, q, table, lens, [1] * len(own))
    bound = bound + (max(lens) / 32 + 4) * 2.0 ** -24 * 255 * cache.scale[1].max()
    tensors, tab, length, x = cache.tensors(), i32(table), i32(lens), q.cuda()
    for max_len in (max(lens), 64 * shared + 1, tab.shape[1] * 64, 1 << 40, None):
        plan = ops.kv8_attention_shared_plan(len(own), len(own), 1, 1 << 31 if max_len is None else max_len, heads, kv_heads, dim, shared)
        assert plan[0] > 0 and (max_len is not None or plan[1] > 4)
        holds(ops.kv8_attention_shared(x, *tensors, tab, length, shared, max_len=max_len), want, bound)


def test_sequences_on_the_device_share_by_default(hip_lib):
    """A pass described with no bound but its rows is cut as one with the bound that its sequences keep, and gives the same bits."""
    from latentq_llm_amd import ops
    from latentq_llm_amd.kv_cache import DeviceSequences, KVCache8
    batch, shared, heads, kv_heads, dim = 40, 14, 8, 2, 64
    cache, gen = KVCache8(120, kv_heads, dim), torch.Generator().manual_seed(1)
    seqs = DeviceSequences(120, batch, 64 * shared + 100, shared)
    results = []
    kv = torch.randn((64 * shared, kv_heads, dim), generator=gen).to(BF16).cuda()
    cache.append(kv, kv.flip(0), seqs.prompt())
    x = torch.randn((2 * batch, heads, dim), generator=gen).to(BF16).cuda()
    for bounds in ({}, {"max_tokens": 2}, {"max_tokens": 2 * batch}):
        step = seqs.extend(torch.full((batch,), 2, dtype=torch.int32, device="cuda"), 2 * batch, **bounds)
        assert ops.kv8_attention_shared_plan(batch, 2 * batch, step.max_tokens, 1 << 31, heads, kv_heads, dim, shared)[0] > 0
        cache.append(x[:, :kv_heads], x[:, kv_heads:2 * kv_heads], step)
        results.append(cache.attend(x, step))
        seqs.give_back(torch.full((batch,), 2, dtype=torch.int32, device="cuda"))
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


def test_a_captured_call_with_a_bound_above(hip_lib):
    """Replays with other first rows than those that it was captured with."""
    from latentq_llm_amd import ops
    batch, shared = 40, 14
    cache = ref.Cache(120, 2, 64, seed=8)
    lens = [14 * 64 + 40] * batch
    t, table, length = cache.tensors(), i32(table_of(lens, shared, 120, 8)), i32(lens)
    q, held = rows((70, 4, 64), BF16, 9).cuda(), i32(np.arange(batch + 1))

    def call():
        return ops.kv8_attention_shared(q, *t, table, length, shared, cu_tokens=held, out=torch.zeros_like(q))

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in range(6):
        news = np.random.default_rng(n).integers(0, 2, batch)
        news[n % batch] += 30 - n
        held.copy_(i32(np.concatenate([[0], np.cumsum(news)])))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n


def test_bounds_that_are_no_numbers(hip_lib):
    """What the binding cannot convert is the wrapper's to refuse, or to take where it is a whole number."""
    from latentq_llm_amd import ops
    shared, lens = 14, [14 * 64 + 3, 14 * 64 + 70]
    cache = ref.Cache(20, 2, 64, seed=1)
    t, table, length, q = cache.tensors(), i32(table_of(lens, shared, 20, 1)), i32(lens), rows((2, 4, 64), BF16, 2).cuda()
    for name in ("max_len", "scale"):
        with pytest.raises(ValueError):
            ops.kv8_attention_shared(q, *t, table, length, shared, **{name: "x"})
    with pytest.raises(ValueError, match="max_len must not be negative"):
        ops.kv8_attention_shared(q, *t, table, length, shared, max_len=-1)
    want = ops.kv8_attention_shared(q, *t, table, length, shared, max_len=966)
    for max_len in (966.0, np.float32(966)):
        assert torch.equal(ops.kv8_attention_shared(q, *t, table, length, shared, max_len=max_len), want)
    want = ops.kv8_attention_shared(q, *t, table, length, shared)
    for max_len in (1e9, 1 << 40):  # as one that is not known
        assert torch.equal(ops.kv8_attention_shared(q, *t, table, length, shared, max_len=max_len), want)
