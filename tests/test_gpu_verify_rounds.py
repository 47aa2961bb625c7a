"""verify_drafts of sequences with more rows than a workgroup tests at a time (32: a wave has a row, eight waves four times): the first refused draft on either side of each change of rounds, in
the last row, and nowhere; greedy, by the target's logits alone and with the drafter's, against the definition (tests/test_gpu_verify_drafts.py)."""
import pytest
import torch

from tests.test_gpu_verify_drafts import check, inputs

pytestmark = pytest.mark.gpu
VOCAB = 90
ROWS = [1, 2, 31, 32, 33, 34, 63, 64, 65, 66, 97, 129]


@pytest.fixture(scope="module")
def verify(hip_lib):
    from latentq_llm_amd import ops
    return ops.verify_drafts


@pytest.mark.parametrize("mode", ["greedy", "alone", "both"])
@pytest.mark.parametrize("refused", [0, 1, 7, 8, 30, 31, 32, 33, 62, 63, 64, 65, 95, 96, 127, None])
@pytest.mark.parametrize("outside", [True, False])
def test_refused_at(verify, mode, refused, outside):
    """Every draft but one of each sequence is taken: the largest logit, by the number 0. The refused one (draft behind row `refused`) lies outside the vocabulary, or is the least likely
    token by a number close to 1."""
    (logits, _, draft, accept), gen = inputs(sum(ROWS), VOCAB, "f32", 21, mode == "both")
    cu = [0]
    for n in ROWS:
        cu.append(cu[-1] + n)
    tokens = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), logits.argmax(-1)[:-1]))
    accept.zero_()
    want = []
    for a, b in zip(cu, cu[1:]):
        hit = refused is not None and a + refused + 1 < b
        if hit:
            at = a + refused
            tokens[at + 1] = VOCAB if outside else (draft - logits if mode == "both" else -logits)[at].argmax()
            accept[at] = 1 - 2.0 ** -24
        want.append(refused if hit else b - a - 1)
    sample = torch.rand(len(ROWS), generator=gen).cuda()
    counts = check(verify, logits, tokens, cu, draft, accept, sample, 0.0 if mode == "greedy" else 1.0)
    assert counts == want
    # and with rows that are not looked at
    for most in (32, 33, 64):
        check(verify, logits, tokens, cu, draft, accept, sample, 0.0 if mode == "greedy" else 1.0, most=most)


@pytest.mark.parametrize("mode", ["greedy", "alone", "both"])
def test_refused_twice(verify, mode):
    """Two refused drafts of one round, and of two: the first counts."""
    (logits, _, draft, accept), gen = inputs(200, VOCAB, "f32", 22, mode == "both")
    sample = torch.rand(2, generator=gen).cuda()
    for first, second in ((3, 4), (3, 30), (31, 32), (30, 64), (32, 63), (64, 98)):
        tokens = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), logits.argmax(-1)[:-1]))
        for row in (first, second, 100 + second, 100 + first):
            tokens[row + 1] = -1
        assert check(verify, logits, tokens, [0, 100, 200], draft, accept * 0, sample, 0.0 if mode == "greedy" else 1.0) == [first, first]
