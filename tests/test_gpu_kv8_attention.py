"""lq_kv8_attention against attention in 64 bits over the values that the codes stand for. The bounds are those of
tests/kv8_ref.py, derived from what the kernels round."""
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


def call(tensors, q, table, lens, news, **more):
    from latentq_llm_amd import ops
    cu = None if len(set(news)) == 1 else i32(np.concatenate([[0], np.cumsum(news)]))
    return ops.kv8_attention(q.cuda(), *tensors, i32(table), i32(lens), cu_tokens=cu, **more)


def holds(got, want, bound):
    got = got.cpu().double().numpy()
    off = np.abs(got - want)
    assert np.isfinite(got).all() and (off <= bound).all(), (float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(off > bound)[:4].tolist())


def run(lens, news, heads, kv_heads, dim, dtype, seed=0, width=None, std=1.0, **how):
    pool = sum(-(-n // 64) for n in lens) + 2
    cache = ref.Cache(pool, kv_heads, dim, seed=seed)
    table = ref.blocks_of(lens, pool, seed=seed, width=width)
    q = rows((sum(news), heads, dim), dtype, seed + 1, std)
    out, lse = call(cache.tensors(), q, table, lens, news, return_lse=True, **how)
    want, (want_lse, lse_bound), bound = ref.attention(cache, q, table, lens, news, **{k: how[k] for k in ("scale", "causal", "window") if k in how})
    holds(out, want, bound)
    lse = lse.cpu().double().numpy()
    assert np.array_equal(np.isinf(lse), np.isinf(want_lse))
    fine = np.isfinite(want_lse)
    assert (np.abs(lse - want_lse)[fine] <= lse_bound[fine]).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads, kv_heads", [(4, 4), (8, 2), (9, 3), (16, 1), (20, 1)])
def test_one_token(hip_lib, heads, kv_heads, dim, dtype):
    """Lengths around the tiles of 64, one to a few slices, one sequence that is empty but for its new token."""
    lens = [1, 2, 63, 64, 65, 127, 300, 1019]
    run(lens, [1] * len(lens), heads, kv_heads, dim, dtype, seed=dim + heads)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("tokens, group", [(2, 1), (5, 3), (8, 4), (16, 2), (7, 9), (33, 1), (64, 1), (4, 16)])
def test_few_tokens(hip_lib, tokens, group, dim, dtype):
    lens = [tokens, tokens + 1, 64 + tokens, 257, 130]
    run(lens, [tokens] * len(lens), 2 * group, 2, dim, dtype, seed=tokens)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("lens, news, heads, kv_heads", [
    ([65], [65], 2, 2), ([127, 300], [127, 200], 2, 1), ([128, 64, 1], [128, 64, 1], 6, 2), ([200, 5, 129], [100, 0, 129], 2, 2), ([515], [70], 4, 1)])
def test_prompts(hip_lib, lens, news, heads, kv_heads, dim, dtype):
    run(lens, news, heads, kv_heads, dim, dtype, seed=lens[0])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("lens, news, how", [
    ([449], [449], {}), ([512, 70, 0], [130, 70, 3], {}), ([640], [60], {"causal": False}), ([577, 420], [90, 420], {"window": 400}), ([700], [100], {"window": 30})])
def test_prompts_of_a_few_sequences(hip_lib, lens, news, how, dim, dtype):
    """Few workgroups with many keys each: even and odd numbers of tiles, also for some rows only, rows without any."""
    run(lens, news, 4, 2, dim, dtype, seed=lens[0], **how)
    cache = ref.Cache(30, 1, dim, seed=5)  # the tiles' weights far apart, in either order
    cache.scale[1] = np.exp2(np.random.default_rng(2).integers(-60, 1, cache.scale[1].shape)).astype(np.float32)
    cache.scale[0] *= np.float32(8)
    table, q = ref.blocks_of(lens, 30, seed=1), rows((sum(news), 2, dim), BF16, 8)
    want, _, bound = ref.attention(cache, q, table, lens, news, **how)
    holds(call(cache.tensors(), q, table, lens, news, **how), want, bound)


@pytest.mark.parametrize("batch", [2, 17, 64, 65])
@pytest.mark.parametrize("how", [{}, {"window": 90}, {"causal": False}])
def test_prompts_of_different_lengths(hip_lib, batch, how):
    """Many rows of many sequences: none, a few and all of their tokens new, prefixes of no and of many tokens, rows before the first position."""
    rng = np.random.default_rng(batch)
    news = [int(n) for n in np.exp2(rng.uniform(0, 6, batch))]
    lens = [n + int(p) for n, p in zip(news, rng.integers(0, 200, batch) * rng.integers(0, 2, batch))]
    news[0], lens[0] = 70, 70
    if batch > 2:
        news[1], lens[2], lens[3] = 0, 0, max(news[3] - 1, 0)
    run(lens, news, 16, 1, 64, BF16, seed=batch, **how)
    run(lens[:9], news[:9], 18, 2, 128, F16, seed=batch, **how)


@pytest.mark.parametrize("how", [{}, {"causal": False}, {"window": 500}])
@pytest.mark.parametrize("dim, heads, kv_heads", [(128, 32, 8), (64, 32, 32), (256, 16, 4), (96, 12, 12), (96, 32, 8)])
def test_long_prompts(hip_lib, dim, heads, kv_heads, how):
    """Some thousands of tokens of all heads, against 64 bits on the card; the bound is tests/kv8_ref.py's."""
    n, new = 4221, 4090
    cache = ref.Cache(68, kv_heads, dim, seed=dim)
    table, q = ref.blocks_of([n], 68), rows((new, heads, dim), BF16, 9)
    out, lse = call(cache.tensors(), q, table, [n], [new], return_lse=True, **how)
    pos = torch.arange(n - new, n).cuda()[:, None]
    key = torch.arange(n).cuda()[None]
    seen = (key <= pos if how.get("causal", True) else key >= 0) & (key > pos - how.get("window", n))
    for h in range(heads):
        kv, blocks = h // (heads // kv_heads), table[0].astype(np.int64)
        k, v = (torch.from_numpy(cache.values(w)[blocks, kv]).reshape(-1, dim)[:n].cuda() for w in (0, 1))
        x = q[:, h].cuda().double()
        s = ((x @ k.T.contiguous()) * dim ** -0.5).masked_fill(~seen, -torch.inf)
        want_lse = torch.logsumexp(s, 1)
        w = torch.exp(s - want_lse[:, None])
        want, size = w @ v, w @ v.abs()
        near = (x.abs() @ k.abs().T.contiguous()).masked_fill(~seen, 0).amax(1)
        score = (dim + 8) * 2.0 ** -24 * near * dim ** -0.5 + 2.0 ** -22 * s.masked_fill(~seen, 0).abs().amax(1)
        scale = torch.from_numpy(cache.scale[1][blocks, kv].astype(np.float64)).repeat_interleave(64)[:n].cuda()
        under = seen.sum(1) * 2.0 ** -25 * 127 * (seen * scale).amax(1)
        bound = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * score + 2.0 ** -18)[:, None] * size + under[:, None]
        assert ((out[:, h].double() - want).abs() <= bound).all()
        assert ((lse[:, h].double() - want_lse).abs() <= score + 2.0 ** -20 * (1 + want_lse.abs())).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("tokens", [1, 4, 90])
def test_windows(hip_lib, tokens, window, dim):
    lens = [tokens, 100 + tokens, 330]
    run(lens, [tokens] * 3, 4, 2, dim, BF16, seed=window, window=window)


@pytest.mark.parametrize("tokens", [1, 4, 90])
@pytest.mark.parametrize("window", [0, 70])
def test_without_the_causal_mask(hip_lib, tokens, window):
    run([100, 200, 300], [tokens] * 3, 4, 2, 64, BF16, causal=False, window=window)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [1, 90])
def test_scales_of_the_scores_and_peaked_rows(hip_lib, tokens, dtype):
    """Scores in the hundreds, where one key takes all the weight, and nearly none."""
    run([400], [tokens], 2, 2, 128, dtype, scale=3.0)
    run([400], [tokens], 2, 2, 128, dtype, scale=1e-6)
    run([400], [tokens], 2, 2, 128, dtype, std=1e-3)


@pytest.mark.parametrize("tokens", [1, 5, 90])
def test_rows_that_see_nothing(hip_lib, tokens):
    """Sequences shorter than their new tokens, and empty ones: zeros, and -inf for the denominator's logarithm."""
    lens, news = [0, max(tokens - 2, 0), 70, 300], [tokens] * 4
    run(lens, news, 4, 2, 64, BF16)
    run(lens, news, 4, 2, 128, F16, window=3)


@pytest.mark.parametrize("tokens", [1, 20, 90])
@pytest.mark.parametrize("dim", [64, 128])
def test_parts_of_the_keys(hip_lib, tokens, dim):
    """Long keys for few rows: several workgroups to a row and a second launch; the same rows without a workspace agree."""
    from latentq_llm_amd import _C, ops
    lens, news, heads = [5000, 3000], [tokens, tokens], 2
    kernel, parts, _ = ops.kv8_attention_plan(2, 2 * tokens, tokens, 5000, heads, heads, dim)
    assert parts > 1
    run(lens, news, heads, heads, dim, F16, seed=3)
    run(lens, news, heads, heads, dim, F16, seed=3, window=900)
    cache = ref.Cache(130, heads, dim, seed=4)
    table, tensors, q = ref.blocks_of(lens, 130), cache.tensors(), rows((2 * tokens, heads, dim), F16, 5).cuda()
    one = torch.empty_like(q)
    t, n = i32(table), i32(lens)
    _C.call("lq_kv8_attention", q.data_ptr(), q.stride(0), q.stride(1), *(x.data_ptr() for x in tensors), 130, t.data_ptr(), t.shape[1], n.data_ptr(), None, 2,
            2 * tokens, tokens, 5000, heads, heads, dim, 1, dim ** -0.5, 1, 0, one.data_ptr(), one.stride(0), one.stride(1), None, None, 0,
            torch.cuda.current_stream().cuda_stream)
    want, _, bound = ref.attention(cache, q.cpu(), table, lens, news)
    holds(one, want, bound)
    holds(ops.kv8_attention(q, *tensors, t, n), want, bound)


@pytest.mark.parametrize("batch", [3, 70, 200])
def test_shares_over_a_batch(hip_lib, batch):
    """Equal shares of all tiles: units of one tile to many, sequences without new tokens and without keys between them, more than
    one pass of 64 sequences; and repeated calls give the same bits."""
    from latentq_llm_amd import ops
    rng = np.random.default_rng(batch)
    lens = [int(n) for n in np.exp2(rng.uniform(0, 8.5, batch))]
    lens[1], lens[0] = 3300, 0
    if batch > 3:
        lens[-1], lens[64], lens[65] = 1700, 0, 2
    for most in (1, 3):
        news = [most if i % 4 else min(most, i % 3) for i in range(batch)]
        assert ops.kv8_attention_plan(batch, sum(news), most, 20000, 4, 2, 64)[1] > 1
        run(lens, news, 4, 2, 64, BF16, seed=batch, max_len=20000, max_tokens=most, width=313)
        run(lens, news, 4, 2, 64, BF16, seed=batch, max_len=20000, max_tokens=most, width=313, window=200)
    cache = ref.Cache(sum(-(-n // 64) for n in lens) + 1, 2, 64)
    table, t = ref.blocks_of(lens, len(cache.scale[0])), cache.tensors()
    q = rows((batch, 4, 64), BF16, 1)
    first = call(t, q, table, lens, [1] * batch)
    assert all(torch.equal(call(t, q, table, lens, [1] * batch), first) for _ in range(3))


def test_a_max_len_that_is_too_small_costs_nothing_but_time(hip_lib):
    for tokens in (1, 90):
        run([700, 100], [tokens] * 2, 2, 2, 64, BF16, max_len=65)


@pytest.mark.parametrize("tokens", [1, 6, 90])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_scales_of_blocks_far_apart(hip_lib, tokens, dim):
    """Value scales over sixty binary orders and key scales over eight: neither overflows nor hides what carries the weight."""
    lens, news = [400], [tokens]
    cache = ref.Cache(9, 2, dim, seed=5)
    rng = np.random.default_rng(1)
    cache.scale[1] = np.exp2(rng.integers(-60, 1, cache.scale[1].shape)).astype(np.float32)
    cache.scale[0] = np.exp2(rng.integers(-12, -3, cache.scale[0].shape)).astype(np.float32)
    table = ref.blocks_of(lens, 9)
    q = rows((tokens, 4, dim), F16, 6)
    # an f16 output has no such range: the largest scale is 1 and tiny outputs are compared with f16's smallest step
    want, _, bound = ref.attention(cache, q, table, lens, news)
    holds(call(cache.tensors(), q, table, lens, news), want, bound + 2.0 ** -25)
    q = q.to(BF16)
    want, _, bound = ref.attention(cache, q, table, lens, news)
    holds(call(cache.tensors(), q, table, lens, news), want, bound)


@pytest.mark.parametrize("tokens", [1, 6, 90])
def test_what_lies_beyond_a_sequence_does_not_matter(hip_lib, tokens):
    """Codes behind the last token, scales of other blocks (NaN, infinite) and table entries behind the last block (out of range)."""
    lens, news, dim = [150, 64], [tokens, min(tokens, 64)], 128
    cache = ref.Cache(8, 2, dim, seed=2)
    table = ref.blocks_of(lens, 8, spare=2 ** 31 - 1, width=6)
    q = rows((sum(news), 4, dim), BF16, 3)
    want = call(cache.tensors(), q, table, lens, news)
    used = set(table[0, :3].tolist() + table[1, :1].tolist())
    for w in (0, 1):
        cache.codes[w][table[0, 2], :, 150 % 64:] = 255
        for b in range(8):
            if b not in used:
                cache.scale[w][b] = np.float32([np.nan, np.inf])[w]
    table[1, 1:] = -5
    got = call(cache.tensors(), q, table, lens, news)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tokens", [1, 6, 90])
def test_a_query_that_is_not_finite_spoils_its_own_row(hip_lib, tokens, dtype):
    lens, news = [200], [tokens]
    cache = ref.Cache(5, 2, 64, seed=2)
    table = ref.blocks_of(lens, 5)
    q = rows((tokens, 4, 64), dtype, 3)
    want = call(cache.tensors(), q, table, lens, news)
    q[0, 1, 7], q[tokens - 1, 2, 0] = float("nan"), float("inf")
    got = call(cache.tensors(), q, table, lens, news)
    assert got[0, 1].isnan().all() and got[tokens - 1, 2].isnan().all()
    same = torch.ones((tokens, 4), dtype=torch.bool)
    same[0, 1] = same[tokens - 1, 2] = False
    assert torch.equal(got[same.cuda()], want[same.cuda()])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_queries_of_any_size(hip_lib, dtype):
    """Rows of very large, very small and zero queries: scores keep their precision, and a row of zeros is the plain mean."""
    lens, news, dim = [130], [4], 64
    cache = ref.Cache(4, 1, dim, seed=2)
    q = rows((4, 1, dim), dtype, 3)
    q[0] *= 1e-4
    q[1] *= 1e3
    q[2] = 0
    if dtype == BF16:
        q[3] *= 1e-30
        cache.scale[0][:] = 2.0 ** -4
    table = ref.blocks_of(lens, 4)
    want, _, bound = ref.attention(cache, q, table, lens, news)
    holds(call(cache.tensors(), q, table, lens, news), want, bound)


def test_strides_and_a_given_output(hip_lib):
    from latentq_llm_amd import ops
    lens, dim, heads = [200], 128, 4
    cache = ref.Cache(5, 2, dim)
    t, table, n = cache.tensors(), i32(ref.blocks_of(lens, 5)), i32(lens)
    for tokens in (1, 90):
        packed = rows((tokens, 3 * heads * dim), BF16, 1).cuda()
        q = packed[:, :heads * dim].view(tokens, heads, dim)
        want = ops.kv8_attention(q.contiguous(), *t, table, n)
        assert torch.equal(ops.kv8_attention(q, *t, table, n), want)
        out = torch.zeros((tokens, 2 * heads, dim), dtype=BF16, device="cuda")
        got = ops.kv8_attention(q, *t, table, n, out=out[:, ::2])
        assert got.data_ptr() == out.data_ptr() and torch.equal(out[:, ::2], want) and not out[:, 1::2].any()
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(ops.kv8_attention(turned, *t, table, n), want)
        odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape).copy_(q)
        assert torch.equal(ops.kv8_attention(odd, *t, table, n), want)


def test_two_sequences_share_the_blocks_of_a_prefix(hip_lib):
    lens, news, dim = [150, 170], [1, 1], 64
    cache = ref.Cache(6, 2, dim)
    table = np.array([[3, 1, 0], [3, 1, 5]], np.int32)
    q = rows((2, 2, dim), F16, 1)
    want, _, bound = ref.attention(cache, q, table, lens, news)
    holds(call(cache.tensors(), q, table, lens, news), want, bound)


@pytest.mark.parametrize("tokens", [1, 90])
def test_another_stream_and_replays_of_a_graph(hip_lib, tokens):
    """On a stream of its own, and captured: every replay on changed inputs equals the eager call."""
    from latentq_llm_amd import ops
    lens, dim, heads = [2000, 900], 128, 4
    cache = ref.Cache(50, heads, dim)
    t, table, n = cache.tensors(), i32(ref.blocks_of(lens, 50)), i32(lens)
    qs = [rows((2 * tokens, heads, dim), BF16, s).cuda() for s in range(4)]
    want = [ops.kv8_attention(q, *t, table, n) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.kv8_attention(q, *t, table, n) for q in qs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    q = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.kv8_attention(q, *t, table, n)
    for i in (1, 2, 3, 0):
        q.copy_(qs[i])
        graph.replay()
        eager = ops.kv8_attention(qs[i], *t, table, n)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(eager, want[i])


def test_nothing_to_do(hip_lib):
    from latentq_llm_amd import ops
    t = ref.Cache(2, 2, 64).tensors()
    q = torch.empty((0, 4, 64), dtype=BF16, device="cuda")
    out, lse = ops.kv8_attention(q, *t, i32(np.zeros((0, 1))), i32([]), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert ops.kv8_attention(q, *t, i32(np.zeros((3, 1))), i32([1, 2, 3])).shape == (0, 4, 64)


def test_refusals(hip_lib):
    from latentq_llm_amd import _C, ops
    t = ref.Cache(4, 2, 64).tensors()
    q = torch.zeros((2, 4, 64), dtype=BF16, device="cuda")
    good = dict(q=q, k_codes=t[0], v_codes=t[1], k_scale=t[2], v_scale=t[3], block_table=i32([[0], [1]]), seq_lens=i32([3, 3]))

    def refuses(kind, match, **change):
        with pytest.raises(kind, match=match):
            ops.kv8_attention(**dict(good, **change))

    refuses(TypeError, "q: expected", q=q.float())
    refuses(_C.LatentQError, "GPU tensor", q=q.cpu())
    refuses(ValueError, "q must be", q=q[..., :32])
    refuses(ValueError, "multiple of 2", q=q[:, :3])
    refuses(ValueError, "scale must be positive", scale=0.0)
    refuses(ValueError, "scale must be positive", scale=float("nan"))
    refuses(ValueError, "window", window=-1)
    refuses(ValueError, "max_len", max_len=-1)
    refuses(ValueError, "block_table must be", block_table=i32([0, 1]))
    refuses(ValueError, "no columns", block_table=i32(np.zeros((2, 0))))
    refuses(TypeError, "out: expected", out=q.half())
    refuses(ValueError, "heads of their own", out=q[:1].expand(2, 4, 64))
    refuses(RuntimeError, "no backward", q=q.clone().requires_grad_())
