"""The plan of attention over the 8-bit cache, on the host."""
import random

from latentq_llm_amd import ops

CAP = ops.WORKSPACE_MAX_BYTES


def shapes(seed, n):
    rng = random.Random(seed)
    log = lambda lo, hi: min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))  # noqa: E731
    for _ in range(n):
        heads, kv = rng.choice(((32, 32), (32, 8), (32, 4), (12, 12), (16, 2), (24, 8), (8, 1), (1, 1)))
        most = log(1, 8192)
        batch = log(1, max(1, 8192 // most)) if rng.random() < 0.5 else 1
        length = max(most, log(1, 131072))
        yield dict(batch=batch, tokens=batch * most, max_tokens=most, max_len=length, heads=heads, kv_heads=kv, dim=rng.choice((64, 96, 128, 256)),
                   window=log(1, 8192) if rng.random() < 0.3 else 0, compute_units=rng.choice((256, 256, 64)))


def test_the_workspace_that_a_plan_names_gives_the_same_plan(hip_lib):
    """A call that gets no more than what its plan takes, as one that is captured does, is cut like one that gets the whole buffer."""
    cut = 0
    for case in shapes(1, 60000):
        first = ops.kv8_attention_plan(**case, workspace_bytes=CAP)
        again = ops.kv8_attention_plan(**case, workspace_bytes=-(-first[2] // 32) * 32)
        assert again == first, case
        cut += first[0] == "prompt" and first[1] > 1
    assert cut > 1000
