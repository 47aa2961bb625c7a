"""Checking drafted tokens and drawing the one that follows, against the definition in 64 bits, row by row.

Tokens are whole numbers: they have to be the same. (Both sides sum up to 100003 numbers in 64 bits, so a border of the cumulative sum differs by some
1e-15 of it, and a given number lies that near to one of 100003 borders once in 10^10 rows.)"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def softmax(row, heat):
    x = row.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, float(np.finfo(np.float32).max))
    if heat == 0:
        p = np.zeros_like(x)
        if x.max() > -np.inf:
            p[x.argmax()] = 1.0
        return p
    if x.max() == -np.inf:
        return np.zeros_like(x)
    e = np.exp((x - x.max()) / heat)
    return e / e.sum()


def drawn(rest, u):
    upto = np.cumsum(rest)
    if upto[-1] == 0:
        return -1
    at = np.flatnonzero((upto > u * upto[-1]) & (rest > 0))
    return int(at[0]) if at.size else int(np.flatnonzero(rest > 0)[-1])


def reference(logits, tokens, cu, draft, accept, sample, heat, most):
    logits, draft = (None if t is None else t.float().cpu().numpy() for t in (logits, draft))
    accept, sample = (None if t is None else t.cpu().numpy().astype(np.float64) for t in (accept, sample))
    tokens = tokens.tolist()
    out, counts = np.full((len(cu) - 1, most), -1, dtype=np.int64), []
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        b, taken = min(b, a + most), 0
        for r in range(a, b):
            p = softmax(logits[r], heat)
            x = tokens[r + 1] if r + 1 < b else None
            if x is not None:
                inside = 0 <= x < p.size
                if heat == 0:
                    good = inside and p[x] == 1.0
                    q = np.zeros_like(p)
                else:
                    q = softmax(draft[r], heat) if draft is not None else np.zeros_like(p)
                    if draft is None and inside:
                        q[x] = 1.0
                    good = inside and accept[r] * q[x] < p[x]
                if good:
                    out[i, taken] = x
                    taken += 1
                    continue
                rest = np.maximum(p - q, 0.0)
                p = rest if rest.sum() > 0 else p
            out[i, taken] = drawn(p, 0.0 if heat == 0 else sample[i])
            break
        counts.append(taken)
    return out, counts


def inputs(rows, vocab, dtype, seed, with_draft, heat=1.0, noise=0.5):
    gen = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn((rows, vocab), generator=gen) + torch.empty((rows, vocab)).exponential_(generator=gen)
    draft = (logits + noise * torch.randn((rows, vocab), generator=gen)).to(TYPES[dtype]) if with_draft else None
    logits = logits.to(TYPES[dtype])
    source = (draft if with_draft else logits).float() / (heat or 1.0)
    following = (source + torch.empty_like(source).exponential_(generator=gen).log().neg() * (heat > 0)).argmax(-1)
    tokens = torch.cat((torch.zeros(1, dtype=torch.int64), following[:-1]))
    accept = torch.rand(rows, generator=gen)
    return [None if t is None else t.cuda() for t in (logits, tokens, draft, accept)], gen


@pytest.fixture(scope="module")
def verify(hip_lib):
    from latentq_llm_amd import ops
    return ops.verify_drafts


def check(verify, logits, tokens, cu, draft, accept, sample, heat, most=None, given=None, uniform=False):
    """The call against the definition; given: logits and draft as the call has them (other strides)."""
    longest = max((b - a for a, b in zip(cu, cu[1:])), default=0)
    most = longest if most is None else most
    where = dict(batch=len(cu) - 1) if uniform else dict(max_tokens=most)
    args, change = given or (logits, draft), torch.full((len(cu) - 1,), 99, dtype=torch.int32, device="cuda")
    out, accepted = verify(args[0], tokens, None if uniform else torch.tensor(cu, dtype=torch.int32, device="cuda"), draft_logits=args[1], accept_draws=accept, sample_draws=sample,
                           temperature=heat, change=change, **where)
    want, counts = reference(logits, tokens, cu, draft, accept, sample, heat, most)
    assert out.dtype == torch.int64 and accepted.dtype == torch.int32
    assert accepted.tolist() == counts
    assert out.tolist() == want.tolist()
    assert change.tolist() == [c + 1 - (b - a) if b > a else 0 for c, a, b in zip(counts, cu, cu[1:])]
    return counts


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 255, 2047, 2048, 2049, 5000, 32000, 100003])
@pytest.mark.parametrize("with_draft", [False, True])
def test_sizes(verify, dtype, vocab, with_draft):
    cu = [0, 1, 6, 6, 9, 13]
    (logits, tokens, draft, accept), gen = inputs(13, vocab, dtype, vocab, with_draft)
    check(verify, logits, tokens, cu, draft, accept, torch.rand(5, generator=gen).cuda(), 1.0)


@pytest.mark.parametrize("heat", [0.0, 0.05, 0.7, 1.0, 3.0, 1e4, 1e-6])
@pytest.mark.parametrize("with_draft", [False, True])
def test_temperatures(verify, heat, with_draft):
    (logits, tokens, draft, accept), gen = inputs(40, 3001, "bf16", 3, with_draft, heat)
    sample = torch.rand(8, generator=gen).cuda()
    counts = check(verify, logits, tokens, list(range(0, 41, 5)), draft, accept, sample, heat, uniform=True)
    if with_draft or heat <= 1:  # (a token looked up has its own probability alone)
        assert sum(counts) > 0
    if heat == 0.0:  # without the numbers, too
        out, accepted = verify(logits, tokens, batch=8, temperature=0)
        assert accepted.tolist() == counts


def test_greedy_takes_the_first_of_equals(verify):
    logits = torch.zeros((6, 5000), dtype=torch.bfloat16)
    for row, places in enumerate(([4999, 17], [0, 1], [2048, 2047], [3000, 4000], [255, 256], [1])):
        logits[row, places] = 3.0
    best = [17, 0, 2047, 3000, 255, 1]
    tokens = torch.tensor([9] + best[:-1]).cuda()
    out, accepted = verify(logits.cuda(), tokens, batch=1, temperature=0.0)
    assert out.tolist() == [best] and accepted.tolist() == [5]
    tokens[3] = 2048  # as large, but not the first
    out, accepted = verify(logits.cuda(), tokens, batch=1, temperature=0.0)
    assert out.tolist() == [best[:3] + [-1] * 3] and accepted.tolist() == [2]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("with_draft", [False, True])
def test_rows_anywhere(verify, dtype, with_draft):
    """Rows that begin at any element, at any distance, the two logits' differing; and every row the same one."""
    (logits, tokens, draft, accept), gen = inputs(12, 1234, dtype, 5, with_draft)
    sample = torch.rand(3, generator=gen).cuda()

    def placed(t, distance, offset):
        if t is None:
            return None
        wide = torch.full((12 * distance + offset + 8,), float("nan"), dtype=t.dtype, device="cuda")
        view = wide[offset:offset + 12 * distance].view(12, distance)[:, :t.shape[1]]
        view.copy_(t)
        return view

    for distance, offset in ((1234, 1), (1235, 3), (1300, 7), (1237, 0)):
        check(verify, logits, tokens, [0, 4, 8, 12], draft, accept, sample, 1.0, given=(placed(logits, distance, offset), placed(draft, distance + 1, offset + 1)))
    turned = torch.empty((1234, 12), dtype=logits.dtype, device="cuda").t()
    turned.copy_(logits)
    check(verify, logits, tokens, [0, 4, 8, 12], draft, accept, sample, 1.0, given=(turned, draft))
    same = logits[:1].expand(12, -1)
    check(verify, same, tokens, [0, 4, 8, 12], draft, accept, sample, 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("heat", [0.0, 1.0])
def test_masked_entries(verify, dtype, with_draft, heat):
    (logits, tokens, draft, accept), gen = inputs(24, 4100, dtype, 6, with_draft)
    inf, lowest = float("inf"), torch.finfo(TYPES[dtype]).min
    kept = tokens[1:].clamp(max=4099)
    logits[2, :] = -inf                      # nothing is left
    logits[3, :] = float("nan")
    logits[5, 100:] = -inf
    logits[6, :4000] = lowest                # as masks are written in the type
    logits[7, :] = lowest                    # and where they hide all: equal entries
    logits[8, 7] = inf
    logits[9, [7, 9, 4099]] = inf
    logits[10, 7] = float("nan")
    logits[11, int(kept[11])] = -inf         # the draft itself
    logits[12, [0, 4099]] = 1000.0
    logits[13, :] = torch.finfo(TYPES[dtype]).max
    if with_draft:
        draft[14, :] = -inf
        draft[15, int(kept[15])] = -inf
        draft[16, 7] = inf
        draft[17, :] = float("nan")
        draft[18, :2048] = -inf
    sample = torch.rand(24, generator=gen).cuda()
    check(verify, logits, tokens, list(range(25)), draft, accept, sample, heat)  # each row is drawn from
    check(verify, logits, tokens, list(range(0, 25, 2)), draft, accept, sample[:12].clone(), heat)
    check(verify, logits, tokens, [0, 2, 5, 9, 10, 14, 24], draft, accept, sample[:6].clone(), heat)


def test_numbers_at_the_ends(verify):
    below = np.nextafter(np.float32(1), np.float32(0)).item()
    (logits, tokens, draft, accept), _ = inputs(12, 3000, "f32", 7, True)
    logits[:, 2990:] = -float("inf")
    for u in (0.0, below, 1e-30):
        for a in (0.0, below):
            sample = torch.full((6,), u, device="cuda")
            check(verify, logits, tokens, list(range(0, 13, 2)), draft, torch.full((12,), a, device="cuda"), sample, 1.0)


@pytest.mark.parametrize("cut", [1.0, 2.0 ** -30])
def test_an_acceptance_at_its_border(verify, cut):
    """u q = p exactly is a refusal; the next smaller number is taken."""
    logits = torch.zeros((2, 2), device="cuda")  # p = 1/2, 1/2
    draft = torch.tensor([[0.0, 80.0]] * 2, device="cuda")  # q = 1 at 1 (and 2^-115 at 0)
    tokens = torch.tensor([0, 1], device="cuda")
    for u, counts in ((0.5, [0]), (float(np.nextafter(np.float32(0.5), np.float32(0))), [1])):
        out, accepted = verify(logits, tokens, batch=1, draft_logits=draft, accept_draws=torch.full((2,), u, device="cuda"), sample_draws=torch.tensor([0.25 * cut], device="cuda"))
        assert accepted.tolist() == counts and out.tolist() == [[0, -1] if counts == [0] else [1, 0]]


def test_the_same_logits_are_always_taken(verify):
    (logits, tokens, _, accept), gen = inputs(40, 9000, "bf16", 8, True)
    sample = torch.rand(5, generator=gen).cuda()
    counts = check(verify, logits, tokens, list(range(0, 41, 8)), logits, accept.clamp(max=0.999), sample, 1.0)
    assert counts == [7] * 5


def test_drafts_outside_the_vocabulary(verify):
    (logits, tokens, draft, accept), gen = inputs(12, 500, "f32", 9, True)
    tokens[1], tokens[3], tokens[5], tokens[7] = -1, 500, 1 << 40, -(1 << 40)
    sample = torch.rand(6, generator=gen).cuda()
    for heat in (0.0, 1.0):
        for d in (draft, None):
            counts = check(verify, logits, tokens, list(range(0, 13, 2)), d, accept * 0, sample, heat)
            assert counts[:4] == [0] * 4


@pytest.mark.parametrize("with_draft", [False, True])
def test_many_sequences(verify, with_draft):
    """Rows enough for the longest slices and blocks, of 8192 and 4096 entries, and a vocabulary that ends inside one."""
    (logits, tokens, draft, accept), gen = inputs(900, 20001, "bf16", 15, with_draft)
    check(verify, logits, tokens, list(range(0, 901, 3)), draft, accept, torch.rand(300, generator=gen).cuda(), 1.0)


@pytest.mark.parametrize("heat", [0.0, 1.0])
def test_long_sequences(verify, heat):
    """Sequences of more rows than are looked at together (128), refused early, late and never."""
    (logits, _, _, accept), gen = inputs(700, 90, "f32", 10, False)
    cu = [0, 129, 129, 430, 443, 700]
    tokens = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), logits.argmax(-1)[:-1]))
    accept.zero_()
    sample = torch.rand(5, generator=gen).cuda()
    assert check(verify, logits, tokens, cu, None, accept, sample, heat) == [128, 0, 300, 12, 256]
    tokens[128], tokens[129 + 256], tokens[443 + 1] = 90, 90, 90
    assert check(verify, logits, tokens, cu, None, accept, sample, heat) == [127, 0, 255, 12, 0]
    check(verify, logits, tokens, cu, None, accept, sample, heat, most=130)  # rows beyond are not looked at
    check(verify, logits, tokens, cu, None, accept, sample, heat, most=1)


def test_sampling_alone(verify):
    """One row each: no drafts, no numbers for them."""
    (logits, tokens, _, _), gen = inputs(33, 777, "f16", 11, False)
    sample = torch.rand(33, generator=gen).cuda()
    out, accepted = verify(logits, tokens, sample_draws=sample)
    want, counts = reference(logits, tokens, list(range(34)), None, None, sample, 1.0, 1)
    assert out.tolist() == want.tolist() and accepted.tolist() == [0] * 33


def test_tokens_are_distributed_as_the_targets(verify):
    """20000 sequences of three rows over 5 tokens: the first token of each follows the target's p, whatever the drafter thinks. Counts of a
    multinomial: five deviations of each, sqrt(n p (1 - p))."""
    n, gen = 20000, torch.Generator().manual_seed(12)
    p, q = torch.tensor([0.5, 0.2, 0.15, 0.1, 0.05]), torch.tensor([0.1, 0.2, 0.3, 0.0, 0.4])
    logits, draft = p.log().repeat(3 * n, 1).cuda(), q.log().repeat(3 * n, 1).cuda()
    tokens = torch.multinomial(q, 3 * n, replacement=True, generator=gen).cuda()
    for d in (draft, None):
        out, accepted = verify(logits, tokens, batch=n, draft_logits=d, accept_draws=torch.rand(3 * n, generator=gen).cuda(), sample_draws=torch.rand(n, generator=gen).cuda())
        counts = torch.bincount(out[:, 0].cpu(), minlength=5).double()
        assert (counts - n * p).abs().le(5 * (n * p * (1 - p)).sqrt()).all(), counts
        assert 0.3 < accepted.double().mean().item() / 2 < 0.6 or d is None


def test_nothing_to_do(verify):
    empty = torch.empty((0, 10), device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    change = torch.full((3,), 99, dtype=torch.int32, device="cuda")
    out, accepted = verify(empty, none, torch.zeros(4, dtype=torch.int32, device="cuda"), sample_draws=torch.rand(3, device="cuda"), change=change)
    assert out.shape == (3, 0) and accepted.tolist() == change.tolist() == [0, 0, 0]
    out, accepted = verify(empty, none)
    assert out.shape == (0, 0) and accepted.shape == (0,)


def test_broken_starts_stay_inside(verify):
    (logits, tokens, draft, accept), gen = inputs(10, 300, "bf16", 13, True)
    sample = torch.rand(4, generator=gen).cuda()
    for cu in ([-5, 3, 2, 1 << 30, 4], [10, 0, 10, 3, 99], [0, 0, 0, 0, 0]):
        out, accepted = verify(logits, tokens, torch.tensor(cu, dtype=torch.int32, device="cuda"), draft_logits=draft, accept_draws=accept, sample_draws=sample)
        assert out.shape == (4, 10) and ((accepted >= 0) & (accepted < 10)).all()


@pytest.mark.parametrize("heat", [0.0, 1.0])
def test_another_stream_and_a_graph(verify, heat):
    cu = [0, 5, 6, 11]
    sets = [inputs(11, 6000, "bf16", 20 + i, True) for i in range(4)]
    samples = [torch.rand(3, generator=gen).cuda() for _, gen in sets]
    starts = torch.tensor(cu, dtype=torch.int32, device="cuda")

    def call(t, sample):
        logits, tokens, draft, accept = t
        return verify(logits, tokens, starts, draft_logits=draft, accept_draws=accept, sample_draws=sample, temperature=heat, max_tokens=5)

    want = [[x.clone() for x in call(t, s)] for (t, _), s in zip(sets, samples)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(sets[1][0], samples[1])
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    held, held_sample = [t.clone() for t in sets[0][0]], samples[0].clone()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = call(held, held_sample)
        graphs.append((graph, result))
    for n in range(6):
        for into, x in zip(held + [held_sample], sets[n % 4][0] + [samples[n % 4]]):
            into.copy_(x)
        for graph, _ in graphs:
            graph.replay()
        call(sets[3][0], samples[3])  # eager work between the replays
        torch.cuda.synchronize()
        for _, result in graphs:
            assert all(torch.equal(a, b) for a, b in zip(result, want[n % 4])), n


def test_refusals(verify):
    (logits, tokens, draft, accept), gen = inputs(6, 100, "bf16", 14, True)
    sample = torch.rand(2, generator=gen).cuda()
    good = dict(batch=2, draft_logits=draft, accept_draws=accept, sample_draws=sample)
    verify(logits, tokens, **good)
    for kind, change in ((ValueError, dict(batch=4)), (ValueError, dict(batch=0)), (ValueError, dict(temperature=-1.0)), (ValueError, dict(temperature=float("nan"))),
                         (ValueError, dict(temperature=float("inf"))), (ValueError, dict(sample_draws=None)), (ValueError, dict(accept_draws=None)), (ValueError, dict(max_tokens=2)),
                         (ValueError, dict(draft_logits=draft[:, :99])), (ValueError, dict(draft_logits=draft.float())), (TypeError, dict(sample_draws=sample.double())),
                         (ValueError, dict(sample_draws=sample[:1])), (ValueError, dict(accept_draws=accept[:5])), (ValueError, dict(draft_logits=draft.cpu())),
                         (ValueError, dict(change=torch.zeros(3, dtype=torch.int32, device="cuda"))), (TypeError, dict(change=tokens[:2]))):
        with pytest.raises(kind):
            verify(logits, tokens, **{**good, **change})
    with pytest.raises(TypeError):
        verify(logits, tokens.int(), **good)
    with pytest.raises(TypeError):
        verify(logits.double(), tokens, **{**good, "draft_logits": None})
    with pytest.raises(ValueError):
        verify(logits[0], tokens, **good)
    with pytest.raises(ValueError):
        verify(logits, tokens[:5], **good)
    with pytest.raises(ValueError):
        verify(logits, tokens, torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda"), **good)
    with pytest.raises(RuntimeError):
        verify(logits.cpu(), tokens, **good)
    with pytest.raises(RuntimeError, match="cannot be recorded in a trace"):
        torch.jit.trace(lambda x: verify(x, tokens, **good)[0], logits, check_trace=False)


def test_numbers_that_are_none(verify):
    """NaN and 1 in the place of uniform numbers: tokens of the vocabulary all the same, the last one left for them."""
    (logits, tokens, draft, accept), gen = inputs(12, 300, "f32", 15, True)
    logits[:, 250:] = -float("inf")
    for u in (float("nan"), 1.0, 2.0, float("inf")):
        for d in (draft, None):
            out, accepted = verify(logits, tokens, batch=6, draft_logits=d, accept_draws=torch.full((12,), u, device="cuda"), sample_draws=torch.full((6,), u, device="cuda"))
            given = out[out >= 0]
            assert given.numel() >= 6 and (given < 250).all()


def test_a_row_that_is_one_token(verify):
    """p is 1 at the draft and 0 elsewhere: whatever the number, nothing else can come."""
    logits = torch.full((4, 5000), -float("inf"), device="cuda")
    logits[:, 4321] = 2.0
    tokens = torch.full((4,), 4321, device="cuda")
    for u in (0.0, 0.999999, 1.0):
        out, accepted = verify(logits, tokens, batch=2, accept_draws=torch.full((4,), u, device="cuda"), sample_draws=torch.full((2,), min(u, 0.5), device="cuda"))
        assert (out[out >= 0] == 4321).all() and (out[:, 0] == 4321).all()
