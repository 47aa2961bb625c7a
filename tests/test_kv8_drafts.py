"""What drafts that were appended and taken back leave in the cache, on the definition itself (tests/kv8_ref.py, which the kernels equal bit for bit): lengths are given back, a block's
scale is not, so the tokens that stay are rounded to the step that the largest refused one asked for."""
import numpy as np
import pytest

from tests import kv8_ref as ref

BLOCKS, HEADS, DIM, DRAFTS = 3, 4, 64, 3


def drafted(x, draft_size, seed=5):
    """(cache, growths of each block's scale) after a pass for each token of x with DRAFTS drafts behind it, all of them refused."""
    rng = np.random.default_rng(seed)
    n = x.shape[0]
    cache, grown = ref.Cache(BLOCKS + 1, HEADS, DIM), np.zeros((BLOCKS + 1, HEADS))
    table = np.arange(BLOCKS + 1, dtype=np.int32)[None]
    for at in range(n):
        rows = np.concatenate([x[at:at + 1], (rng.standard_normal((DRAFTS, HEADS, DIM)) * draft_size).astype(np.float32)]) if draft_size else x[at:at + 1]
        before = cache.scale[0].copy()
        ref.append(cache, rows, rows, table, [at + len(rows)], [len(rows)])
        for place in {at // 64, (at + len(rows) - 1) // 64}:
            if at > 64 * place:
                grown[place] += cache.scale[0][place] > before[place]
    return cache, grown


def error(cache, x):
    """Of the values that the cache gives back, in steps of their block's scale."""
    n = x.shape[0]
    back = cache.values(0).transpose(0, 2, 1, 3).reshape(-1, HEADS, DIM)[:n]
    return np.abs(back - x) / np.repeat(cache.scale[0], 64, axis=0)[:n, :, None]


@pytest.mark.parametrize("size", [0.25, 1.0, 10.0])
def test_refused_drafts(size):
    x = np.random.default_rng(4).standard_normal((64 * BLOCKS - 5, HEADS, DIM)).astype(np.float32)
    alone, grown_alone = drafted(x, 0)
    with_drafts, grown = drafted(x, size)
    # half a step when a token comes, and half a step at each growth of the scale, of steps that are no larger than the last one
    for cache, g in ((alone, grown_alone), (with_drafts, grown)):
        assert error(cache, x).max() <= 0.5 * (1 + g.max()) + 1e-3
    here = slice(0, BLOCKS)
    assert (with_drafts.scale[0][here] >= alone.scale[0][here]).all()
    ratio = float((with_drafts.scale[0][here] / alone.scale[0][here]).mean())
    print("drafts of size %g: steps %.2f times as large, growths a block %.1f for %.1f" % (size, ratio, grown[here].mean(), grown_alone[here].mean()))
    if size < 1:  # drafts that are smaller than what a block holds leave nothing there
        assert ratio < 1.02
    if size > 1:  # the largest of 64 x DIM normal numbers is about 4, that of as many refused ones 40
        assert ratio > 5 and not np.array_equal(with_drafts.codes[0][here], alone.codes[0][here])


def test_a_block_that_only_refused_drafts_had():
    """A token that begins a block finds its scale by itself, whatever refused drafts were there."""
    x = np.random.default_rng(4).standard_normal((65, HEADS, DIM)).astype(np.float32)
    table = np.arange(BLOCKS + 1, dtype=np.int32)[None]
    results = []
    for size in (0.0, 100.0):
        cache = ref.Cache(BLOCKS + 1, HEADS, DIM)
        ref.append(cache, x[:64], x[:64], table, [64], [64])
        if size:
            rows = np.full((DRAFTS, HEADS, DIM), size, dtype=np.float32)
            ref.append(cache, rows, rows, table, [64 + DRAFTS], [DRAFTS])
        ref.append(cache, x[64:], x[64:], table, [65], [1])
        results.append((cache.scale[0][1].copy(), cache.codes[0][1][:, 0].copy(), cache.codes[0][0].copy()))
    assert all(np.array_equal(a, b) for a, b in zip(*results))
