"""lq_kv8_append and lq_kv8_read against their definition, bit for bit: every operation of the definition is one float32 rounding,
which numpy makes the same way."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def starts(news, device="cuda"):
    return torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=device)


def check(cache, tensors, untouched=None):
    k, v = ref.from_layout(tensors[0], tensors[1])
    for got, want, name in ((k, cache.codes[0], "key codes"), (v, cache.codes[1], "value codes")):
        assert np.array_equal(got, want), (name, np.argwhere(got != want)[:4].tolist())
    for got, want, name in ((tensors[2], cache.scale[0], "key scales"), (tensors[3], cache.scale[1], "value scales")):
        assert np.array_equal(got.cpu().numpy().view(np.int32), want.view(np.int32)), name


def step(cache, tensors, k, v, table, lens, news, q=None, rot=0, positions=None, uniform=False, **more):
    from latentq_llm_amd import ops
    cos = sin = None
    if rot:
        cos, sin = ref.tables(positions or max(max(lens), 1), rot)
    got = ops.kv8_append(k.cuda(), v.cuda(), *tensors, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                         q=None if q is None else q.cuda(), cos=None if not rot else torch.from_numpy(cos).cuda(),
                         sin=None if not rot else torch.from_numpy(sin).cuda(), cu_tokens=None if uniform else starts(news), **more)
    pos = ref.append(cache, k.float().numpy(), v.float().numpy(), table, lens, news, cos, sin)
    if q is not None:
        at = np.clip(pos, 0, cos.shape[0] - 1)
        want = torch.from_numpy(ref.rotated(q.float().numpy(), cos[at], sin[at])).to(q.dtype)
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim, rot", [(64, 0), (64, 64), (96, 96), (96, 32), (128, 128), (128, 48), (256, 256), (256, 16)])
def test_ragged_tokens(hip_lib, dim, rot, dtype):
    """Whole blocks, parts at either end, one token, none, beside a sequence that does not change."""
    lens, news = [200, 64, 1, 65, 130, 63], [137, 64, 1, 0, 3, 63]
    cache = ref.Cache(16, 3, dim, seed=dim + rot)
    tensors = cache.tensors()
    table = ref.blocks_of(lens, 16, seed=3)
    k, v, q = rows((sum(news), 3, dim), dtype, 1), rows((sum(news), 3, dim), dtype, 2), rows((sum(news), 6, dim), dtype, 3)
    step(cache, tensors, k, v, table, lens, news, q=q if rot else None, rot=rot)
    check(cache, tensors)


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("at", [1, 4, 8, 9])
def test_few_tokens_at_every_place_of_a_block(hip_lib, dim, at):
    """`at` new tokens behind 0 .. 70 tokens: every alignment to the groups of four and to the block's end."""
    lens = [n + at for n in (0, 1, 2, 3, 5, 59, 60, 61, 62, 63, 64, 70)]
    news = [at] * len(lens)
    cache = ref.Cache(40, 2, dim, seed=at)
    tensors = cache.tensors()
    table = ref.blocks_of(lens, 40, seed=at)
    k, v = rows((sum(news), 2, dim), BF16, 5), rows((sum(news), 2, dim), BF16, 6)
    step(cache, tensors, k, v, table, lens, news, rot=dim, uniform=True)
    check(cache, tensors)


def test_a_sequence_grown_token_by_token(hip_lib):
    """Scales that grow in the middle of a block: what is there is rounded again, by keys and values on their own."""
    dim, heads = 128, 2
    cache = ref.Cache(4, heads, dim, seed=1)
    tensors = cache.tensors()
    table = ref.blocks_of([140], 4)
    for n in range(1, 141):
        grow = 1.0 + 0.05 * n if n % 3 else 0.2
        step(cache, tensors, rows((1, heads, dim), BF16, n, grow), rows((1, heads, dim), BF16, 1000 + n, 3 - grow / 4), table, [n], [1], rot=128, positions=140)
        if n in (1, 2, 5, 63, 64, 65, 100, 140):
            check(cache, tensors)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_special_values(hip_lib, dtype):
    """Infinities saturate, NaN becomes zero, and neither moves a scale; zeros and tiny values have a scale that is a normal number."""
    dim, lens = 64, [70, 64, 10, 64]
    big = 3e38 if dtype == BF16 else 6e4
    k = rows((sum(lens), 2, dim), dtype, 1)
    v = rows((sum(lens), 2, dim), dtype, 2)
    k[3, 0, 5], k[4, 1, 0], k[5, 0, 63] = float("inf"), float("nan"), -float("inf")
    v[66, 1, 2], v[67, 0, 3], v[68, 0, 4] = float("nan"), float("inf"), big
    k[70:134] = 0
    v[70:134, 0] = float("nan")
    v[70:134, 1] = 1e-30 if dtype == BF16 else 6e-8
    k[134:144, 0] = float("inf")
    cache = ref.Cache(8, 2, dim, seed=4)
    tensors = cache.tensors()
    step(cache, tensors, k, v, ref.blocks_of(lens, 8), lens, lens)
    check(cache, tensors)
    assert all(torch.isfinite(t).all() and (t > 0).all() for t in tensors[2:])


def test_a_block_that_opens_forgets_the_scale_of_what_it_held(hip_lib):
    cache = ref.Cache(2, 1, 64, seed=1)
    cache.scale[0][:], cache.scale[1][:] = np.float32(np.nan), np.float32(1e30)
    tensors = cache.tensors()
    step(cache, tensors, rows((1, 1, 64), BF16, 1), rows((1, 1, 64), BF16, 2), np.array([[1]], np.int32), [1], [1])
    check_one = [t[1].cpu() for t in tensors[2:]]
    assert all(torch.isfinite(t).all() and t.item() < 1 for t in check_one)
    assert np.array_equal(ref.from_layout(tensors[0], tensors[1])[0][1], cache.codes[0][1])


def test_values_come_back_within_half_a_step(hip_lib):
    """Against the inputs themselves, in 64 bits: half a step of the block's scale (and fp32's rounding of the quotient)."""
    from latentq_llm_amd import ops
    dim, n = 128, 150
    k, v = rows((n, 4, dim), BF16, 1), rows((n, 4, dim), BF16, 2)
    cache = ref.Cache(4, 4, dim)
    tensors = cache.tensors()
    table = ref.blocks_of([n], 4, seed=2)
    step(cache, tensors, k, v, table, [n], [n])
    got = ops.kv8_read(*tensors, torch.from_numpy(table[0]).cuda(), dtype=torch.float32)
    for x, y, s in zip((k, v), got, tensors[2:]):
        y = y.cpu().double().reshape(-1, 4, dim)[:n]
        steps = s.cpu().double()[torch.from_numpy(table[0]).long()].repeat_interleave(64, 0)[:n, :, None]
        assert ((y - x.double()).abs() <= steps * (0.5 + 1e-4)).all()


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_read(hip_lib, dim, dtype):
    from latentq_llm_amd import ops
    cache = ref.Cache(6, 5, dim, seed=dim)
    tensors = cache.tensors()
    blocks = [5, 0, 3, 3, -1, 6]
    k, v = ops.kv8_read(*tensors, torch.tensor(blocks, dtype=torch.int32, device="cuda"), dtype=dtype)
    for which, got in ((0, k), (1, v)):
        c = (cache.codes[which] - 128).astype(np.float32) * cache.scale[which][:, :, None, None]
        want = torch.from_numpy(c).to(dtype).transpose(1, 2)
        for i, b in enumerate(blocks):
            assert torch.equal(got[i].cpu(), want[b] if 0 <= b < 6 else torch.zeros_like(want[0])), (which, i)
    k, v = ops.kv8_read(*tensors, torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert k.shape == v.shape == (0, 64, 5, dim)


def test_views_of_a_packed_projection_and_rotation_in_place(hip_lib):
    from latentq_llm_amd import ops
    dim, heads, n = 128, 4, 70
    packed = rows((n, 3 * heads * dim), BF16, 1).cuda()
    q, k, v = (t.view(n, heads, dim) for t in packed.split(heads * dim, 1))
    assert not k.is_contiguous()
    cos, sin = (torch.from_numpy(t).cuda() for t in ref.tables(n, dim))
    table, lens = torch.from_numpy(ref.blocks_of([n], 3)).cuda(), torch.tensor([n], dtype=torch.int32, device="cuda")
    a, b = ref.Cache(3, heads, dim).tensors(), ref.Cache(3, heads, dim).tensors()
    want = ops.kv8_append(k.contiguous(), v.contiguous(), *a, table, lens, q=q.contiguous(), cos=cos, sin=sin)
    got = ops.kv8_append(k, v, *b, table, lens, q=q, cos=cos, sin=sin, q_out=q)
    assert got is q and torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(a, b))
    # strides that the kernels do not take (a transposed view, an odd offset) are copied
    odd = torch.empty(n * heads * dim + 1, dtype=BF16, device="cuda")[1:].view(n, heads, dim).copy_(k)
    turned = v.transpose(0, 1).contiguous().transpose(0, 1)
    c = ref.Cache(3, heads, dim).tensors()
    ops.kv8_append(odd, turned.transpose(1, 2).contiguous().transpose(1, 2), *c, table, lens, cos=cos, sin=sin)
    assert all(torch.equal(x, y) for x, y in zip(a, c))


def test_what_the_device_holds_is_kept_inside_the_operands(hip_lib):
    """Blocks outside the pool, tokens beyond the table or before position 0: not stored, and nothing else is touched."""
    dim = 64
    lens, news = [100, 3, 130], [100, 5, 10]
    table = np.array([[2, 9], [0, -1], [1, 3]], np.int32)  # 9: outside; sequence 1 has more new tokens than tokens; 2: beyond two columns
    cache = ref.Cache(5, 2, dim, seed=9)
    tensors = cache.tensors()
    k, v, q = rows((115, 2, dim), BF16, 1), rows((115, 2, dim), BF16, 2), rows((115, 4, dim), BF16, 3)
    step(cache, tensors, k, v, table, lens, news, q=q, rot=64, positions=90)
    check(cache, tensors)


def test_nothing_to_do(hip_lib):
    from latentq_llm_amd import ops
    cache = ref.Cache(2, 2, 64)
    tensors = cache.tensors()
    empty = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    cos = torch.ones((4, 32), device="cuda")
    q = ops.kv8_append(empty, empty, *tensors, torch.zeros((0, 1), **i32), torch.zeros(0, **i32), q=empty, cos=cos, sin=cos)
    assert q.shape == (0, 2, 64)
    ops.kv8_append(empty, empty, *tensors, torch.zeros((2, 1), **i32), torch.tensor([5, 0], **i32))
    check(cache, tensors)


def test_a_pool_beyond_32_bit_offsets(hip_lib):
    from latentq_llm_amd import ops
    heads, dim, pool = 32, 256, 8500  # 4.4 GiB of codes each
    k_codes = torch.empty((pool, heads, 64, dim), dtype=torch.uint8, device="cuda")
    v_codes = torch.empty((pool, heads, 16, dim, 4), dtype=torch.uint8, device="cuda")
    k_scale, v_scale = (torch.ones((pool, heads), device="cuda") for _ in range(2))
    assert k_codes.numel() > 2 ** 32
    lens, news = [70], [70]
    table = np.array([[pool - 1, pool - 2]], np.int32)
    k, v = rows((70, heads, dim), BF16, 1), rows((70, heads, dim), BF16, 2)
    ops.kv8_append(k.cuda(), v.cuda(), k_codes, v_codes, k_scale, v_scale, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    cache = ref.Cache(2, heads, dim)
    ref.append(cache, k.float().numpy(), v.float().numpy(), np.array([[1, 0]], np.int32), lens, news)
    got = ref.from_layout(k_codes[-2:], v_codes[-2:])
    assert np.array_equal(got[0][1], cache.codes[0][1]) and np.array_equal(got[1][1], cache.codes[1][1])
    assert np.array_equal(got[0][0, :, :6], cache.codes[0][0, :, :6]) and np.array_equal(got[1][0, :, :6], cache.codes[1][0, :, :6])
    x, y = ops.kv8_read(k_codes, v_codes, k_scale, v_scale, torch.tensor([pool - 1], dtype=torch.int32, device="cuda"), dtype=torch.float32)
    want = cache.values(0)[1].transpose(1, 0, 2)
    assert np.abs(x[0].cpu().numpy() - want).max() <= 1e-6 * np.abs(want).max()
    # and attention over them
    q = rows((1, heads, dim), BF16, 3)
    out = ops.kv8_attention(q.cuda(), k_codes, v_codes, k_scale, v_scale, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))
    want, _, bound = ref.attention(cache, q, np.array([[1, 0]], np.int32), lens, [1])
    assert (np.abs(out.cpu().double().numpy() - want) <= bound).all()


def test_refusals(hip_lib):
    from latentq_llm_amd import _C, ops
    t = ref.Cache(4, 2, 64).tensors()
    i32 = dict(dtype=torch.int32, device="cuda")
    k = torch.zeros((6, 2, 64), dtype=BF16, device="cuda")
    table, lens, cu = torch.zeros((2, 2), **i32), torch.tensor([3, 3], **i32), torch.tensor([0, 3, 6], **i32)
    cos = torch.ones((8, 32), device="cuda")
    good = dict(k=k, v=k, k_codes=t[0], v_codes=t[1], k_scale=t[2], v_scale=t[3], block_table=table, seq_lens=lens)

    def refuses(kind, match, **change):
        with pytest.raises(kind, match=match):
            ops.kv8_append(**dict(good, **change))

    refuses(TypeError, "k: expected", k=k.float())
    refuses(TypeError, "v: expected", v=k.half())
    refuses(_C.LatentQError, "GPU tensor", v=k.cpu())
    refuses(ValueError, r"k must be \[tokens, 2, 64\]", k=k[:, :1])
    refuses(ValueError, "k has 6 rows and v 5", v=k[:5])
    refuses(TypeError, "k_codes: expected", k_codes=t[0].to(torch.int8))
    refuses(ValueError, "dim one of", k_codes=t[0][..., :32].contiguous())
    refuses(ValueError, "v_codes must be", v_codes=t[1][..., :2].contiguous())
    refuses(ValueError, "k_scale must be", k_scale=t[2][:2])
    refuses(ValueError, "contiguous", v_scale=t[3].t().contiguous().t())
    refuses(TypeError, "seq_lens: expected", seq_lens=lens.long())
    refuses(ValueError, "block_table must be", block_table=table[:1])
    refuses(ValueError, "cu_tokens must be", cu_tokens=cu[:2])
    refuses(ValueError, "same number of tokens", k=k[:5], v=k[:5])
    refuses(ValueError, "max_tokens", max_tokens=1)
    refuses(ValueError, "max_tokens", max_tokens=0, cu_tokens=cu)
    refuses(ValueError, "go together", cos=cos)
    refuses(ValueError, "cos and sin must be", cos=cos[:, :28].contiguous(), sin=cos[:, :28].contiguous())
    refuses(ValueError, "cos and sin must be", cos=torch.ones((8, 40), device="cuda"), sin=torch.ones((8, 40), device="cuda"))
    refuses(TypeError, "cos: expected", cos=cos.half(), sin=cos)
    refuses(ValueError, "needs cos and sin", q=k)
    refuses(ValueError, "q_out without q", q_out=k, cos=cos, sin=cos)
    refuses(ValueError, "q_out must be", q=k, q_out=k[:5], cos=cos, sin=cos)
    refuses(ValueError, "heads of their own", q=k, q_out=k[:1].expand(6, 2, 64), cos=cos, sin=cos)
    refuses(RuntimeError, "no backward", k=k.clone().requires_grad_())
    with pytest.raises(TypeError, match="dtype"):
        ops.kv8_read(*t, torch.zeros(1, **i32), dtype=torch.float64)
    with pytest.raises(ValueError, match="one-dimensional"):
        ops.kv8_read(*t, torch.zeros((1, 1), **i32))
    with torch.no_grad():
        ops.kv8_append(**dict(good, k=k.clone().requires_grad_()))
