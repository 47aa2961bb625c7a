"""A generation step whose books are kept on the device, as it is used: room for drafted tokens, appending, attention over a shared prompt, verification, and what
was refused given back. Each pass is checked against the host's books, the plain forms of the operators, and ordinary attention on the same state."""
import numpy as np
import pytest
import torch

from tests import kv8_ref as ref
from tests.test_gpu_kv8_shared import holds
from tests.test_gpu_verify_drafts import reference

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HEADS, KV, DIM, VOCAB = 8, 2, 64, 500


class Model:
    """One layer without weights to speak of: what a token gives for queries, keys and values, and logits from attention's output."""

    def __init__(self, capacity):
        from latentq_llm_amd.kv_cache import KVCache8, rotation_tables
        gen = torch.Generator().manual_seed(1)
        self.q, self.k, self.v = (torch.randn((VOCAB, n * DIM), generator=gen).to(BF16).cuda() for n in (HEADS, KV, KV))
        self.head = (torch.randn((HEADS * DIM, VOCAB), generator=gen) * 0.3).to(BF16).cuda()
        self.cos, self.sin = rotation_tables(capacity, DIM)
        self.cache = KVCache8(200, KV, DIM)

    def __call__(self, tokens, step):
        n = tokens.numel()
        q = self.q[tokens].view(n, HEADS, DIM)
        turned = self.cache.append(self.k[tokens].view(n, KV, DIM), self.v[tokens].view(n, KV, DIM), step, q=q, cos=self.cos, sin=self.sin)
        out = self.cache.attend(turned, step)
        return turned, out, out.view(n, -1) @ self.head


@pytest.mark.parametrize("shared, heat", [(0, 1.0), (16, 1.0), (16, 0.0)])
def test_passes(hip_lib, shared, heat):
    from latentq_llm_amd import ops
    from latentq_llm_amd.kv_cache import DeviceSequences
    batch, drafts, capacity = 5, 3, 64 * shared + 300
    model, seqs, gen = Model(capacity + 64), DeviceSequences(200, batch, capacity, shared), torch.Generator().manual_seed(2)
    if shared:
        model(torch.randint(0, VOCAB, (64 * shared,), generator=gen).cuda(), seqs.prompt())
    lens = [64 * shared] * batch
    known = torch.randint(0, VOCAB, (batch,), generator=gen).tolist()
    for n in range(12):
        counts = [int(c) for c in torch.randint(0, drafts + 2, (batch,), generator=gen)]
        if n == 0:
            counts = [70, 1, 33, 2, 5]  # prompts of their own
        rows = sum(counts) + n % 2
        cu = np.concatenate([[0], np.cumsum(counts)])
        tokens = torch.randint(0, VOCAB, (rows,), generator=gen)
        for i, c in enumerate(counts):
            if c:
                tokens[cu[i]] = known[i]
        step = seqs.extend(torch.tensor(counts, dtype=torch.int32, device="cuda"), rows, max_tokens=max(counts))
        assert step.status.item() == 0 and step.cu_tokens.tolist() == cu.tolist() and step.shared == shared
        lens = [a + b for a, b in zip(lens, counts)]
        assert seqs.seq_lens.tolist() == lens
        assert step.positions[:cu[-1]].tolist() == [p for length, c in zip(lens, counts) for p in range(length - c, length)]
        table = seqs.block_table.cpu().numpy()
        have = [b for i, length in enumerate(lens) for b in table[i, shared:max(shared, -(-length // 64))]] + table[0, :shared].tolist()
        assert len(set(have)) == len(have) == 200 - seqs.free_count.item()
        tokens = tokens.cuda()
        turned, out, logits = model(tokens, step)
        # attention, against 64 bits on what the cache holds
        cache = ref.Cache(1, KV, DIM)
        cache.codes = list(ref.from_layout(*model.cache.tensors()[:2]))
        cache.scale = [t.cpu().numpy() for t in model.cache.tensors()[2:]]
        want, _, bound = ref.attention(cache, turned[:cu[-1]].cpu(), table, lens, counts)
        holds(out[:cu[-1]], want, bound)
        # verification, against the definition on the same logits
        accept, sample = torch.rand(rows, generator=gen).cuda(), torch.rand(batch, generator=gen).cuda()
        if n == 5:
            accept.zero_()  # (every draft that has any probability)
        got, accepted = seqs.verify(logits, tokens, step, accept_draws=accept, sample_draws=sample, temperature=heat)
        want, taken = reference(logits[:cu[-1]], tokens, cu.tolist(), None, accept, sample, heat, max(counts))
        assert accepted.tolist() == taken and got.tolist() == want.tolist()
        lens = [length - (c - 1 - a if c else 0) for length, c, a in zip(lens, counts, taken)]
        assert seqs.seq_lens.tolist() == lens
        for i, (c, a) in enumerate(zip(counts, taken)):
            if c:
                known[i] = int(want[i, a])
    # a sequence that is done begins again on the shared blocks
    seqs.give_back(torch.full((batch,), 10 ** 6, dtype=torch.int32, device="cuda"))
    assert seqs.seq_lens.tolist() == [64 * shared] * batch and seqs.free_count.item() == 200 - shared
    assert sorted(seqs.free_blocks[:200 - shared].tolist()) == list(range(shared, 200))
    assert ops.KV_BLOCK == 64


def test_a_captured_pass(hip_lib):
    """The whole of a greedy pass in a graph: room, appending, attention, logits, verification, giving back, and the next tokens; replayed, with the eager pass on the
    same books between, which has to do the same."""
    from latentq_llm_amd.kv_cache import DeviceSequences
    batch, drafts, shared = 4, 3, 15
    rows, capacity = batch * (drafts + 1), 64 * shared + 400
    gen = torch.Generator().manual_seed(3)
    prompt = torch.randint(0, VOCAB, (64 * shared,), generator=gen).cuda()
    worlds = []
    for _ in range(2):
        model, seqs = Model(capacity + 64), DeviceSequences(100, batch, capacity, shared)
        model(prompt, seqs.prompt())
        tokens = torch.arange(rows, device="cuda") * 7 % VOCAB
        worlds.append((model, seqs, tokens, torch.full((batch,), drafts + 1, dtype=torch.int32, device="cuda")))

    def one(world):
        model, seqs, tokens, new = world
        step = seqs.extend(new, rows, max_tokens=drafts + 1)
        logits = model(tokens, step)[2]
        out, accepted = seqs.verify(logits, tokens, step, temperature=0.0)
        behind = out.gather(1, accepted.long()[:, None])  # drafted as if the last token came again
        tokens.copy_(behind.expand(-1, drafts + 1).reshape(-1))
        return out, accepted, step.status

    for _ in range(2):  # first calls load code
        for world in worlds:
            one(world)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = one(worlds[0])
    for n in range(6):
        graph.replay()
        eager = one(worlds[1])
        torch.cuda.synchronize()
        assert captured[2].item() == eager[2].item() == 0
        assert torch.equal(captured[0], eager[0]) and torch.equal(captured[1], eager[1]), n
        for a, b in zip(worlds[0][1]._books(), worlds[1][1]._books()):
            assert torch.equal(a, b), n
        assert torch.equal(worlds[0][2], worlds[1][2])
        for a, b in zip(worlds[0][0].cache.tensors(), worlds[1][0].cache.tensors()):
            assert torch.equal(a, b), n


def test_a_pool_that_is_used_up(hip_lib):
    """The pass is refused as a whole, on the device: it has no tokens, so nothing is appended and no row is written."""
    from latentq_llm_amd.kv_cache import DeviceSequences
    model, seqs = Model(500), DeviceSequences(4, 3, 300)
    step = seqs.extend(torch.tensor([100, 64, 10], dtype=torch.int32, device="cuda"), 174, max_tokens=100)
    assert step.status.item() == 0 and seqs.free_count.item() == 0
    model(torch.zeros(174, dtype=torch.int64, device="cuda"), step)
    before = [t.clone() for t in (*seqs._books(), *model.cache.tensors())]
    step = seqs.extend(torch.tensor([100, 0, 10], dtype=torch.int32, device="cuda"), 110, max_tokens=100)
    assert step.status.item() == 2 and step.cu_tokens.tolist() == [0] * 4
    out, accepted = seqs.verify(model(torch.zeros(110, dtype=torch.int64, device="cuda"), step)[2], torch.zeros(110, dtype=torch.int64, device="cuda"), step, temperature=0.0)
    assert accepted.tolist() == [0] * 3 and (out == -1).all()
    assert all(torch.equal(a, b) for a, b in zip(before, (*seqs._books(), *model.cache.tensors())))


def test_refusals(hip_lib):
    from latentq_llm_amd.kv_cache import DeviceSequences, KVCache8
    for args in ((10, 0, 100), (10, 2, 0), (10, 2, 100, 3), (1, 2, 1000, 2), (10, 2, 100, -1)):
        with pytest.raises(ValueError):
            DeviceSequences(*args)
    with pytest.raises(ValueError):
        DeviceSequences(10, 2, 100).prompt()
    step = DeviceSequences(10, 2, 100, 1).extend(torch.ones(2, dtype=torch.int32, device="cuda"), 2)
    x = torch.zeros((2, 1, 64), dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="cache of 9"):
        KVCache8(9, 1, 64).append(x, x, step)
    table = torch.zeros((100, 32), device="cuda")
    with pytest.raises(ValueError, match="100 positions"):
        KVCache8(10, 1, 64).append(x, x, step, q=x, cos=table, sin=table)


def test_example(hip_lib):
    """The example's drafted generation runs and gives as many tokens as asked, all of the vocabulary, and the same ones again."""
    import importlib.util
    import os

    from latentq_llm_amd.kv_cache import DeviceSequences, KVCache8
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "generate_kv8.py")
    spec = importlib.util.spec_from_file_location("generate_kv8", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    shared, new, drafts = 15, 9, 3
    model = m.Decoder(2, 512, 1024, 8, 2, 1000, 64 * shared + 320).eval()
    caches = [KVCache8(60, 2, 64) for _ in range(2)]
    gen = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, 1000, (64 * shared,), generator=gen).tolist()
    questions = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (200, 33, 1)]
    questions[1] = questions[1][:3] * 11  # (something to look up)
    runs = []
    for _ in range(2):
        sequences = DeviceSequences(60, 3, 64 * shared + 260, shared)
        out, _, _, passes = m.generate_drafted(model, caches, sequences, prompt, questions, new, drafts)
        assert [len(o) for o in out] == [new] * 3 and all(0 <= t < 1000 for o in out for t in o)
        assert passes % 8 == 0 and passes >= (new - 1) / (drafts + 1)
        assert all(64 * shared + len(q) + new - 1 <= n <= 64 * shared + len(q) + new + drafts for q, n in zip(questions, sequences.seq_lens.tolist()))
        runs.append(out)
    assert runs[0] == runs[1]
