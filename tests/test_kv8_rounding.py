"""What rounding a block again costs, on the definition itself (tests/kv8_ref.py, which the kernels equal bit for bit): tokens appended one by
one against the same tokens at once, both against the unrounded values."""
import numpy as np
import pytest

from tests import kv8_ref as ref

BLOCKS, DIM = 4, 128


def errors(x, pieces):
    """Errors of the values that the cache gives back, in steps of their block's scale, and how often each block's scale grew."""
    n, heads, _ = x.shape
    cache = ref.Cache(BLOCKS, heads, DIM)
    table, at, grown = np.arange(BLOCKS, dtype=np.int32)[None], 0, np.zeros((BLOCKS, heads))
    while at < n:
        new = min(pieces, n - at)
        before = cache.scale[0].copy()
        ref.append(cache, x[at:at + new], x[at:at + new], table, [at + new], [new])
        grown[at // 64] += (cache.scale[0][at // 64] > before[at // 64]) & (at % 64 > 0)
        at += new
    back = cache.values(0).transpose(0, 2, 1, 3).reshape(-1, heads, DIM)[:n]
    step = np.repeat(cache.scale[0], 64, axis=0)[:n, :, None]
    return (back - x) / step, grown


@pytest.mark.parametrize("kind", ["normal", "outliers", "rising"])
def test_one_by_one(kind):
    x = np.random.default_rng(1).standard_normal((64 * BLOCKS, 8, DIM))
    if kind == "outliers":
        x[:, :, ::32] *= 4
    if kind == "rising":  # the scale grows with every token
        x *= np.exp2(np.arange(64 * BLOCKS) % 64 / 8)[:, None, None]
    x = x.astype(np.float32)
    whole, _ = errors(x, 64)
    single, grown = errors(x, 1)
    # half a step at once; and at each growth half a step of the scale that it grows to, which is no more than the last one
    assert np.abs(whole).max() <= 0.5 + 1e-4
    assert np.abs(single).max() <= 0.5 * (1 + grown.max()) + 1e-3
    rms = [float(np.sqrt((e ** 2).mean())) for e in (whole, single)]
    print(kind, "rms steps at once %.3f, one by one %.3f; growths a block %.1f, most %d, largest error %.2f" % (*rms, grown.mean(), grown.max(), np.abs(single).max()))
    # rounding errors add like independent ones: a twelfth of a squared step each
    assert rms[0] <= 12 ** -0.5 * 1.02 and rms[1] <= (1 + grown.mean()) ** 0.5 * 12 ** -0.5 * 1.02
