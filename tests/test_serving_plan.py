"""What attention over shared blocks plans for a pass whose bound of a sequence's new tokens is far above what the sequences have: all rows of the pass, say, as is the default."""
import pytest

CUS = 256


def plan(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, shared, **how):
    from latentq_llm_amd import ops
    return ops.kv8_attention_shared_plan(batch, tokens, max_tokens, max_len, heads, kv_heads, dim, shared, compute_units=CUS, **how)


@pytest.mark.parametrize("batch, tokens, shared, own, heads, kv_heads, dim", [(64, 1, 128, 512, 32, 8, 128), (17, 1, 2048, 257, 32, 8, 128), (12, 1, 32, 1019, 32, 32, 128), (8, 5, 64, 640, 32, 32, 64),
                                                                             (64, 2, 128, 300, 24, 8, 96), (30, 4, 64, 100, 8, 1, 256), (300, 1, 64, 100, 32, 8, 128), (4096, 1, 32, 64, 8, 2, 64)])
def test_all_rows_for_a_bound(hip_lib, batch, tokens, shared, own, heads, kv_heads, dim):
    """The same cut as with the bound that a caller who counted would give."""
    exact = plan(batch, batch * tokens, tokens, 64 * shared + own, heads, kv_heads, dim, shared)
    assert exact[0] > 0
    for bound in (batch * tokens, batch * tokens + 5, 10 ** 9):
        assert plan(batch, batch * tokens, bound, 64 * shared + own, heads, kv_heads, dim, shared) == exact


def test_one_prompt_among_single_tokens(hip_lib):
    assert plan(64, 63 + 512, 512, 9000, 32, 8, 128, 128)[0] > 0
    assert plan(64, 63 + 512, 512, 9000, 32, 8, 128, 0)[:2] == (0, 0)


@pytest.mark.parametrize("tokens, group, shares", [(16, 4, True), (17, 4, False), (64, 1, True), (65, 1, False), (8, 8, True), (9, 8, False)])
def test_sequences_that_have_many_rows_themselves(hip_lib, tokens, group, shares):
    """Rows enough to fill matrix tiles by themselves are left to ordinary attention, by their number on average, whatever the bound is."""
    for bound in (tokens, 8 * tokens):
        assert (plan(8, 8 * tokens, bound, 9000, 8 * group, 8, 128, 128)[0] > 0) == shares


def test_a_bound_close_to_what_the_sequences_have(hip_lib):
    """More than 64 rows at the most, and not half of that on average: as many rows as the bound says."""
    for total, shares in ((64 * 10, True), (64 * 13, False), (64 * 15, False)):  # of up to 20 tokens each, four heads to a kv head
        assert (plan(64, total, 20, 9000, 32, 8, 128, 128)[0] > 0) == shares


def test_a_plan_made_again_with_the_bytes_that_it_took(hip_lib):
    for batch, total, bound in ((64, 64, 64), (17, 60, 40), (40, 300, 200), (5, 5, 5)):
        first = plan(batch, total, bound, 9000, 32, 8, 128, 128)
        assert first[0] > 0 and plan(batch, total, bound, 9000, 32, 8, 128, 128, workspace_bytes=first[2]) == first


@pytest.mark.parametrize("batch, tokens, shared, own, heads, kv_heads, dim", [(64, 1, 128, 512, 32, 8, 128), (16, 1, 2048, 257, 32, 8, 128), (8, 5, 64, 640, 32, 32, 64), (4, 1, 128, 100, 32, 8, 128),
                                                                             (8, 4, 16, 300, 32, 32, 128)])
def test_lengths_that_are_not_known(hip_lib, batch, tokens, shared, own, heads, kv_heads, dim):
    """Without a bound of the lengths the shared keys are cut as for sequences that have few of their own, not by all that the table has room for."""
    args = (heads, kv_heads, dim, shared)
    exact = plan(batch, batch * tokens, tokens, 64 * shared + own, *args)
    unknown = plan(batch, batch * tokens, tokens, 1 << 31, *args)
    assert unknown[0] >= exact[0] > 0 and unknown[0] <= 2 * exact[0]
    assert plan(batch, batch * tokens, tokens, (1 << 63) - 1, *args) == unknown
    assert plan(batch, batch * tokens, tokens, 1 << 31, *args, workspace_bytes=unknown[2]) == unknown
