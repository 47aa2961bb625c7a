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


def test_no_slice_beyond_what_a_window_shows(hip_lib):
    """Slices of the keys are of what the rows of a workgroup see: of 128 or 256 rows, their tokens' windows."""
    def plan(tokens, length, heads, kv_heads, dim, window, **more):
        return ops.kv8_attention_plan(1, tokens, tokens, length, heads, kv_heads, dim, window, compute_units=256, **more)

    for case in ((2048, 2048, 12, 12, 96, 128), (2048, 2048, 8, 1, 128, 64), (4096, 4096, 8, 1, 128, 16), (4096, 4096, 8, 1, 128, 128), (1024, 8192, 12, 12, 96, 256)):
        assert plan(*case) == ("prompt", 1, 0), case
    assert plan(512, 16384, 32, 8, 128, 0)[1] > 1 and plan(512, 16384, 32, 8, 128, 8192)[1] > 1
    seen = 0
    for case in shapes(2, 40000):
        kernel, parts, _ = ops.kv8_attention_plan(**case)
        if kernel != "prompt" or not case["window"]:
            continue
        group = case["heads"] // case["kv_heads"]
        tiles = (case["window"] + min(case["max_tokens"], 256 // group + 1) - 1 + 62) // 64 + 1
        assert parts <= tiles, case
        seen += parts > 1
        wide = dict(case, window=case["max_len"] + 1)  # a window that hides nothing
        assert ops.kv8_attention_plan(**wide) == ops.kv8_attention_plan(**dict(case, window=0)), case
    assert seen > 300
