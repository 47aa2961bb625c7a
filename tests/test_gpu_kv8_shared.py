"""lq_kv8_attention_shared: attention of sequences that begin with the same blocks, against attention in 64 bits. The bounds are those of
tests/kv8_ref.py, derived from what the kernels round, and what this kernel adds to them: codes go into the products as u = 1 .. 255, so the sums that 128 times
the queries, or the weights, come off are up to 255 sum |q| and 255 max(v_scale), in steps of 32 terms that round to 24 bits each. For a score these are
(dim / 32 + 2) 2^-24 255 sum |q| k_scale, less than (dim + 8) 2^-24 sum |q k| while codes are 14 from 128 on average (they are 27 here); for an output (keys / 32 + 4) 2^-24 255
max(v_scale), added below."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def holds(got, want, bound):
    got = got.cpu().double().numpy()
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= bound).all(), (float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(off > bound)[:4].tolist())


def table_of(lens, shared, pool, seed, width=None):
    """Block tables whose first `shared` entries are the same, also those of sequences that do not reach there."""
    order = [int(b) for b in np.random.default_rng(seed).permutation(pool)]
    common, at = order[:shared], shared
    table = np.full((len(lens), width or max(shared, max(-(-n // 64) for n in lens), 1)), -1, dtype=np.int32)
    table[:, :shared] = common
    for i, n in enumerate(lens):
        more = max(0, -(-n // 64) - shared)
        table[i, shared:shared + more] = order[at:at + more]
        at += more
    assert at <= pool
    return table


def call(tensors, q, table, lens, news, shared, **more):
    from latentq_llm_amd import ops
    cu = None if len(set(news)) == 1 else i32(np.concatenate([[0], np.cumsum(news)]))
    return ops.kv8_attention_shared(q.cuda(), *tensors, i32(table), i32(lens), shared, **{"cu_tokens": cu, **more})


def run(shared, own, news, heads, kv_heads, dim, dtype, seed=0, split=True, lens=None, cache=None, width=None, **how):
    from latentq_llm_amd import ops
    lens = [64 * shared + n for n in own] if lens is None else lens
    pool = shared + sum(max(0, -(-n // 64) - shared) for n in lens) + 2
    cache = cache(pool) if cache else ref.Cache(pool, kv_heads, dim, seed=seed)
    table = table_of(lens, shared, pool, seed, width)
    q = rows((sum(news), heads, dim), dtype, seed + 1)
    took = ops.kv8_attention_shared_plan(len(lens), sum(news), max(news), how.get("max_len", table.shape[1] * 64), heads, kv_heads, dim, shared)
    assert (took[0] > 0) == split, took  # (a plan that leaves the call to kv8_attention)
    out, lse = call(cache.tensors(), q, table, lens, news, shared, return_lse=True, **how)
    want, (want_lse, lse_bound), bound = ref.attention(cache, q, table, lens, news, **{k: how[k] for k in ("scale", "causal") if k in how})
    holds(out, want, bound + (max(lens) / 32 + 4) * 2.0 ** -24 * 255 * cache.scale[1].max())
    lse = lse.cpu().double().numpy()
    assert np.array_equal(np.isinf(lse), np.isinf(want_lse))
    fine = np.isfinite(want_lse)
    assert (np.abs(lse[fine] - want_lse[fine]) <= lse_bound[fine]).all()
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads, kv_heads, batch", [(4, 4, 5), (8, 2, 4), (9, 3, 7), (16, 1, 3), (6, 2, 17), (16, 2, 40), (64, 1, 2), (40, 1, 2)])
def test_one_token(hip_lib, heads, kv_heads, batch, dim, dtype):
    """Rows of the prefix for every form of the kernel (to 16, to 64, more), own keys around the tiles of 64."""
    own = ([1, 2, 63, 64, 65, 127, 300] * 6)[:batch]
    run(14, own, [1] * batch, heads, kv_heads, dim, dtype, seed=dim + heads)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("tokens, group, batch", [(2, 1, 3), (5, 3, 2), (8, 2, 9), (3, 4, 30), (8, 8, 2), (33, 1, 2), (64, 1, 3)])
def test_few_tokens(hip_lib, tokens, group, batch, dim, dtype):
    run(15, ([tokens, tokens + 1, 64 + tokens, 257] * 8)[:batch], [tokens] * batch, 2 * group, 2, dim, dtype, seed=tokens)


@pytest.mark.parametrize("how", [{}, {"causal": False}, {"scale": 0.3}])
@pytest.mark.parametrize("batch", [2, 3, 64, 65, 130])
def test_sequences_of_all_lengths(hip_lib, batch, how):
    """Different numbers of new tokens, none among them; sequences shorter than what they share, to nothing at all, and rows before position 0."""
    rng = np.random.default_rng(batch)
    news = [int(n) for n in rng.integers(0, 6, batch)]
    lens = [int(n) for n in rng.integers(0, 1500, batch)]
    news[0], lens[0] = 5, 14 * 64
    news[1], lens[1] = 3, 0
    if batch > 2:
        news[2], lens[2] = 4, 2
        news[-1], lens[-1] = 2, 14 * 64 + 1
    run(14, None, news, 8, 2, 64, BF16, seed=batch, lens=lens, **how)
    run(14, None, news, 3, 3, 128, F16, seed=batch, lens=lens, **how)


@pytest.mark.parametrize("shared, width", [(14, 20), (15, 16), (16, 19), (63, 70), (64, 66), (65, 66), (300, 301)])
@pytest.mark.parametrize("dim, batch", [(128, 3), (64, 30), (96, 70)])
def test_shared_lengths(hip_lib, shared, width, dim, batch):
    run(shared, [1 + i % 60 for i in range(batch)], [1] * batch, 4, 2, dim, BF16, seed=shared, width=width)


def test_nothing_of_their_own(hip_lib):
    """Rows that are in the shared blocks themselves, and a table with no other columns."""
    run(14, None, [3, 3, 3], 4, 2, 64, BF16, lens=[896, 700, 3])
    run(14, None, [1, 2], 4, 2, 128, F16, lens=[896, 2])


@pytest.mark.parametrize("shared, batch, tokens, heads", [(0, 3, 1, 4), (5, 1, 3, 4), (5, 2, 17, 8), (5, 4, 1, 4)])
def test_left_to_ordinary_attention(hip_lib, shared, batch, tokens, heads):
    """Nothing shared, nobody to share with, rows enough in every sequence, and little to be shared: as kv8_attention gives it, bit for bit."""
    from latentq_llm_amd import ops
    lens = [400] * batch
    cache = ref.Cache(40, 2, 64, seed=3)
    table = table_of(lens, shared, 40, 3)
    q = rows((batch * tokens, heads * 2, 64), BF16, 4).cuda()
    assert ops.kv8_attention_shared_plan(batch, batch * tokens, tokens, 448, heads * 2, 2, 64, shared)[:2] == (0, 0)
    t = cache.tensors()
    assert torch.equal(ops.kv8_attention_shared(q, *t, i32(table), i32(lens), shared), ops.kv8_attention(q, *t, i32(table), i32(lens)))


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("batch", [3, 20, 50])
def test_scales_far_apart(hip_lib, dim, batch):
    """Blocks without values (scale 0 and under 2^-97), keys of zero, and values of very different sizes."""
    def cache(pool):
        c, rng = ref.Cache(pool, 2, dim, seed=dim), np.random.default_rng(dim)
        c.scale[1] = np.exp2(rng.integers(-60, 1, c.scale[1].shape)).astype(np.float32)
        c.scale[1][rng.random(c.scale[1].shape) < 0.2] = 0.0
        c.scale[1][rng.random(c.scale[1].shape) < 0.1] = 1e-35
        c.scale[0][rng.random(c.scale[0].shape) < 0.2] = 0.0
        c.scale[0][0] *= 8
        return c
    run(14, [1 + 37 * (i % 5) for i in range(batch)], [1] * batch, 4, 2, dim, BF16, seed=dim + batch, cache=cache)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("batch, tokens", [(4, 1), (30, 1), (6, 5)])
@pytest.mark.parametrize("kind", [0, 1])
def test_blocks_that_a_sequence_does_not_see(hip_lib, kind, batch, tokens, dim):
    """Scales that are no numbers, of shared blocks behind a sequence's end and of own blocks behind a token's last key, are nothing to it."""
    lens = [64 * 16 + 70 if i % 3 == 0 else 64 * 14 + i - 1 for i in range(batch)]
    cache = ref.Cache(18 + 2 * batch, 2, dim, seed=dim)
    table = table_of(lens, 16, 18 + 2 * batch, 1)
    q = rows((batch * tokens, 4, dim), BF16, 2)
    want, (want_lse, lse_bound), bound = ref.attention(cache, q, table, lens, [tokens] * batch)
    bound = bound + (max(lens) / 32 + 4) * 2.0 ** -24 * 255 * cache.scale[1].max()
    short = [i * tokens + j for i in range(batch) if lens[i] <= 64 * 15 for j in range(tokens)]
    for bad in (float("nan"), float("inf"), -float("inf")):
        tensors = cache.tensors()
        tensors[2 + kind][i32(table[0, 15:16]).long()] = bad
        out, lse = call(tensors, q, table, lens, [tokens] * batch, 16, return_lse=True)
        holds(out[short], want[short], bound[short])
        assert (np.abs(lse.cpu().double().numpy() - want_lse)[short] <= lse_bound[short]).all()
    # five tokens of which the last one alone sees the third own block
    lens = [64 * 18 + 1] * batch
    table = table_of(lens, 15, 18 + 4 * batch, 1)
    cache = ref.Cache(18 + 4 * batch, 2, dim, seed=dim)
    q = rows((batch * 5, 4, dim), BF16, 2)
    want, _, bound = ref.attention(cache, q, table, lens, [5] * batch)
    bound = bound + (max(lens) / 32 + 4) * 2.0 ** -24 * 255 * cache.scale[1].max()
    tensors = cache.tensors()
    tensors[2 + kind][i32(table[:, 18]).long()] = float("nan")
    out = call(tensors, q, table, lens, [5] * batch, 15)
    seen = [i for i in range(5 * batch) if i % 5 < 4]
    holds(out[seen], want[seen], bound[seen])


def test_scores_far_apart(hip_lib):
    """Scores to some hundreds: the largest ones in the prefix for some rows, among their own keys for others."""
    def cache(pool):
        c = ref.Cache(pool, 1, 128, seed=3)
        c.scale[0] *= np.float32(30) * np.random.default_rng(3).random(c.scale[0].shape).astype(np.float32)
        return c
    for batch in (3, 40, 90):
        run(14, [1 + 11 * i for i in range(batch)], [1] * batch, 2, 1, 128, F16, seed=5, cache=cache)


@pytest.mark.parametrize("size, scale", [(1e30, 1e-30), (3e34, 1e-35), (1e-30, 1e30), (1.0, 1e3), (1.0, 1e5), (1e-30, 1.0), (1e-38, 1.0), (0.0, 1.0)])
def test_queries_of_any_size(hip_lib, size, scale):
    """As ordinary attention gives them, queries and their factor at the ends of 32 bits; scores of 1e6 pick a key (from some 2^26 on a step of 32 bits is an exponent's range,
    and there neither kernel has a result), small ones average."""
    from latentq_llm_amd import ops
    lens, shared = [1000, 1300, 960, 900], 14
    cache = ref.Cache(40, 2, 64, seed=21)
    t, table, length = cache.tensors(), i32(table_of(lens, shared, 40, 21)), i32(lens)
    q = (rows((4, 4, 64), BF16, 22).float() * size).to(BF16).cuda()
    got = ops.kv8_attention_shared(q, *t, table, length, shared, scale=scale)
    assert ops.kv8_attention_shared_plan(4, 4, 1, table.shape[1] * 64, 4, 2, 64, shared)[0] > 0
    want = ops.kv8_attention(q, *t, table, length, scale=scale)
    assert torch.isfinite(got).all()
    # each is within its bound of the value: ulp and weights (2^-11 |o| + 2^-11 sum p |v|, |v| <= 127 v_scale), and one step of bf16 of either
    slack = (2.0 ** -10 + 2.0 ** -12) * 127 * float(cache.scale[1].max()) * 2 + 2.0 ** -7 * want.float().abs()
    assert ((got.float() - want.float()).abs() <= slack).all()


def test_strides_and_a_given_output(hip_lib):
    lens, shared, heads, dim = [1160, 960, 900], 14, 4, 128
    cache = ref.Cache(30, 2, dim, seed=9)
    table = table_of(lens, shared, 30, 9)
    q = rows((6, heads, dim), BF16, 10)
    want, _, bound = ref.attention(cache, q, table, lens, [2, 2, 2])
    wide = torch.zeros((6, heads, 3 * dim), dtype=BF16, device="cuda")
    wide[:, :, dim:2 * dim] = q.cuda()
    turned = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(6 * heads * dim + 3, dtype=BF16, device="cuda")[3:].view(6, heads, dim)
    odd.copy_(q)
    from latentq_llm_amd import ops
    for x in (wide[:, :, dim:2 * dim], turned, odd):
        out = torch.full((6, heads, 2 * dim), 7.0, dtype=BF16, device="cuda")
        got = ops.kv8_attention_shared(x, *cache.tensors(), i32(table), i32(lens), shared, out=out[:, :, :dim])
        assert got.data_ptr() == out.data_ptr() and (out[:, :, dim:] == 7).all()
        holds(got, want, bound)


def test_rows_that_no_sequence_has(hip_lib):
    """Rows behind the last sequence, and beyond max_tokens of one, are left as they were."""
    lens, news, shared = [1276, 976, 906], [2, 0, 3], 14
    cache = ref.Cache(30, 2, 64, seed=11)
    table, q = table_of(lens, shared, 30, 11), rows((9, 4, 64), BF16, 12)
    want, _, bound = ref.attention(cache, q[:5], table, lens, news)
    out = torch.full((9, 4, 64), 7.0, dtype=BF16, device="cuda")
    got = call(cache.tensors(), q, table, lens, news, shared, cu_tokens=i32([0, 2, 2, 5]), out=out)
    holds(got[:5], want, bound)
    assert (out[5:] == 7).all()
    out.fill_(7.0)
    got = call(cache.tensors(), q, table, lens, news, shared, cu_tokens=i32([0, 2, 2, 5]), max_tokens=2, out=out)
    holds(got[:4], want[:4], bound[:4])
    assert (out[4:] == 7).all()


def test_bounds_that_are_too_small(hip_lib):
    """A max_len below the sequences' lengths costs time, not correctness: below their shared blocks, too."""
    for max_len in (1, 64, 890, 896, 900, 1000):
        run(14, [300, 100, 20, 64], [1] * 4, 4, 2, 64, BF16, seed=13, max_len=max_len, split=max_len > 832)


def test_what_the_device_holds_is_kept_inside(hip_lib):
    """Blocks outside the pool, lengths beyond the table, broken first rows: other values, and no fault."""
    cache = ref.Cache(12, 2, 64, seed=14)
    q = rows((8, 4, 64), BF16, 15)
    t = cache.tensors()
    table = table_of([1104] * 4, 14, 40, 14)
    table[:, 1], table[2, 16], table[3, 15] = 1 << 30, -5, 99
    for lens in ([1104] * 4, [2 ** 31 - 1, -2 ** 31, 1153, -1]):
        for cu in (None, [0, 2, 4, 6, 8], [-9, 1 << 30, 3, 2, 8], [8, 0, 8, 0, 8]):
            out = call(t, q, table, lens, [2] * 4, 14, cu_tokens=None if cu is None else i32(cu))
            assert out.shape == q.shape


def test_another_stream_and_graphs(hip_lib):
    from latentq_llm_amd import ops
    lens, shared = [1156, 1456, 956, 897, 906], 14
    cache = ref.Cache(60, 4, 128, seed=16)
    t, table = cache.tensors(), i32(table_of(lens, shared, 60, 16))
    length = i32(lens)
    qs = [rows((5, 8, 128), BF16, 20 + i).cuda() for i in range(3)]
    want = [ops.kv8_attention_shared(q, *t, table, length, shared).clone() for q in qs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.kv8_attention_shared(qs[1], *t, table, length, shared)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want[1])
    held = qs[0].clone()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.kv8_attention_shared(held, *t, table, length, shared)
        graphs.append((graph, out))
    for n in range(6):
        held.copy_(qs[n % 3])
        for graph, _ in graphs:
            graph.replay()
        assert torch.equal(ops.kv8_attention_shared(qs[2], *t, table, length, shared), want[2])
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[n % 3]) for _, out in graphs), n


def test_little_workspace(hip_lib):
    """By the C entry, with every amount of workspace from none to what it takes: fewer slices, then ordinary attention."""
    from latentq_llm_amd import _C, ops
    lens, shared, news = [5000, 4500, 4300], 60, [1, 1, 1]
    cache = ref.Cache(120, 2, 64, seed=17)
    table, q = table_of(lens, shared, 120, 17), rows((3, 4, 64), F16, 18)
    want, _, bound = ref.attention(cache, q, table, lens, news)
    t, tab, length, x = cache.tensors(), i32(table), i32(lens), q.cuda()
    full = ops.kv8_attention_shared_plan(3, 3, 1, 5056, 4, 2, 64, shared)
    slot = 3 * 4 * 65 * 4
    assert full[2] == (full[0] + full[1]) * slot and full[0] > 4
    seen = set()
    for size in (0, 16, slot, 2 * slot, 2 * slot + 16, 3 * slot, 5 * slot, full[2] - 16, full[2], 2 * full[2]):
        plan = ops.kv8_attention_shared_plan(3, 3, 1, 5056, 4, 2, 64, shared, workspace_bytes=size)
        assert plan[2] <= size
        seen.add(plan[0])
        guard = torch.full((size + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(x)
        _C.call("lq_kv8_attention_shared", x.data_ptr(), x.stride(0), x.stride(1), *(c.data_ptr() for c in t), 120, tab.data_ptr(), tab.shape[1], length.data_ptr(), None, 3, 3, 1, 5056,
                shared, 4, 2, 64, 1, 0.125, 1, out.data_ptr(), out.stride(0), out.stride(1), None, guard.data_ptr() if size else None, size, torch.cuda.current_stream().cuda_stream)
        holds(out, want, bound)
        assert (guard[size:] == 0xAB).all()
    assert 0 in seen and len(seen) > 3


def test_refusals(hip_lib):
    from latentq_llm_amd import ops
    lens = [400, 300]
    cache = ref.Cache(20, 2, 64, seed=1)
    t, table, n, q = cache.tensors(), i32(table_of(lens, 3, 20, 1)), i32(lens), rows((4, 4, 64), BF16, 2).cuda()
    ops.kv8_attention_shared(q, *t, table, n, 3)
    for kind, args, more in ((ValueError, (q, *t, table, n, -1), {}), (ValueError, (q, *t, table, n, table.shape[1] + 1), {}), (ValueError, (q[:3], *t, table, n, 3), {}),
                             (TypeError, (q.float(), *t, table, n, 3), {}), (ValueError, (q, *t, table, n, 3), dict(scale=0.0)), (ValueError, (q, *t, table, n, 3), dict(max_len=-1)),
                             (ValueError, (q, *t, table, n, 3), dict(out=torch.empty((4, 4, 65), dtype=BF16, device="cuda")[:, :, :64])), (TypeError, (q, *t, table.long(), n, 3), {}),
                             (ValueError, (q, *t, table, n[:1], 3), {}), (RuntimeError, (q.clone().requires_grad_(), *t, table, n, 3), {}), (ValueError, (q[:, :3], *t, table, n, 3), {})):
        with pytest.raises(kind):
            ops.kv8_attention_shared(*args, **more)
    with pytest.raises(RuntimeError, match="cannot be recorded in a trace"):
        torch.jit.trace(lambda x: ops.kv8_attention_shared(x, *t, table, n, 3), q, check_trace=False)
