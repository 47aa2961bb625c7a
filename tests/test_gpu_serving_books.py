"""What DeviceSequences says of each change of its books, those that cannot be done among them: books that were changed from outside, as nothing else makes giving back fail."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def world():
    from latentq_llm_amd.kv_cache import DeviceSequences
    seqs = DeviceSequences(12, 3, 200, 1)
    step = seqs.extend(i32([70, 3, 64]), 137)
    assert step.status.item() == 0 and seqs.status is step.status
    return seqs, step


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def books(seqs):
    return [t.clone() for t in seqs._books()]


def drafts(seqs, rows):
    """A verification that refuses every draft: room for two more, of which the second never is the largest logit."""
    step = seqs.extend(i32([2, 2, 2]), rows, max_tokens=2)
    logits = torch.zeros((rows, 100), device="cuda")
    logits[:, 5] = 1.0
    return step, lambda: seqs.verify(logits, torch.full((rows,), 7, dtype=torch.int64, device="cuda"), step, temperature=0.0)


def test_changes_that_are_done(hip_lib):
    seqs, step = world()
    status = seqs.give_back(i32([6, 0, 64]))
    assert status.item() == 0 and seqs.status is status and seqs.seq_lens.tolist() == [128, 67, 64]
    step, verify = drafts(seqs, 6)
    out, accepted = verify()
    assert accepted.tolist() == [0, 0, 0] and out.tolist() == [[5, -1]] * 3
    assert seqs.status.item() == 0 and seqs.status is not step.status and seqs.seq_lens.tolist() == [129, 68, 65]


def test_a_pass_that_cannot_be(hip_lib):
    from latentq_llm_amd import ops
    seqs, _ = world()
    before = books(seqs)
    step = seqs.extend(i32([100, 0, 0]), 100)  # (of 134 tokens, where a table holds 256)
    assert step.status.item() == 0
    seqs.give_back(i32([100, 0, 0]))
    step = seqs.extend(i32([200, 0, 0]), 200)
    assert step.status.item() == seqs.status.item() == ops.KV_NARROW
    assert all(torch.equal(a, b) for a, b in zip(before[1:2], seqs._books()[1:2]))


@pytest.mark.parametrize("broken, want", [("count", "KV_LIST"), ("length", "KV_NARROW")])
def test_books_that_are_none(hip_lib, broken, want):
    from latentq_llm_amd import ops
    seqs, _ = world()
    step, verify = drafts(seqs, 6)
    if broken == "count":
        seqs.free_count.fill_(-1)
    else:
        seqs.seq_lens[2] = 4000
    before = books(seqs)
    _, accepted = verify()
    assert accepted.tolist() == [0, 0, 0] and step.status.item() == 0
    assert seqs.status.item() == getattr(ops, want)  # the refused drafts are still there
    assert all(torch.equal(a, b) for a, b in zip(before, seqs._books()))
    assert seqs.give_back(i32([1, 1, 1])).item() == getattr(ops, want)
    assert all(torch.equal(a, b) for a, b in zip(before, seqs._books()))


def test_the_status_of_a_captured_pass(hip_lib):
    """The tensors that a graph writes: each replay says anew whether its changes were done."""
    from latentq_llm_amd import ops
    seqs, _ = world()
    drafts(seqs, 6)[1]()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    logits, tokens, new = torch.zeros((6, 100), device="cuda"), torch.full((6,), 7, dtype=torch.int64, device="cuda"), i32([2, 2, 2])
    logits[:, 5] = 1.0
    with torch.cuda.graph(graph):
        step = seqs.extend(new, 6, max_tokens=2)
        seqs.verify(logits, tokens, step, temperature=0.0)
        status = seqs.status
    for n in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert (step.status.item(), status.item()) == (0, 0)
    held = seqs.seq_lens.clone()
    seqs.free_count.sub_(100)
    graph.replay()
    torch.cuda.synchronize()
    assert (step.status.item(), status.item()) == (ops.KV_LIST, ops.KV_LIST) and torch.equal(seqs.seq_lens, held)
    seqs.free_count.add_(100)
    graph.replay()
    torch.cuda.synchronize()
    assert (step.status.item(), status.item()) == (0, 0) and torch.equal(seqs.seq_lens, held + 1)
