"""The operators of a generation step in which sequences share a prompt and drafted tokens are checked, as cases to be timed: what a
server does around the paged 8-bit cache without asking the host.

kind     one pass
resize   ``ops.kv8_resize``, twice: room is made for the new tokens of a pass (block tables, lengths, free list, and for each new
         token its position and its slot in the pool), and, as none of them was taken, given back
shared   ``ops.kv8_attention_shared``: attention of the last tokens of each sequence over the cache, the first ``prefix`` tokens
         of all sequences being in the same blocks
verify   ``ops.verify_drafts``: drafted tokens against the target's logits, by given uniform numbers; the token that follows the
         accepted ones is drawn on the way (without drafts: sampling)

Layout of the cache and of its block tables: perf/operators.py. A pass's rows are the new tokens of its sequences one after the other. In
``verify`` the rows of a sequence are the tokens that went through the model, the first one known and the others drafted, and
the logits what the model gave for each; ``drafts``: "logits" (the drafter's, of which the tokens were drawn) or "none" (tokens looked up somewhere).
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a chat with one user: room for five tokens, four of them drafted
        {"name": "room_1", "kind": "resize", "batch": 1, "tokens": 5, "context": 1019, "shared": 0, "ragged": False},
        # a server's batch behind a prompt of 256 tokens in common, one to eight tokens each
        {"name": "room_64", "kind": "resize", "batch": 64, "tokens": 8, "context": 8192, "shared": 4, "ragged": True},
        # prompts of up to 512 tokens for 128 sequences
        {"name": "room_128x512", "kind": "resize", "batch": 128, "tokens": 512, "context": 45, "shared": 0, "ragged": True},
        # four answers to one question, one token each: the smallest
        {"name": "answers_4", "kind": "shared", "batch": 4, "tokens": 1, "prefix": 512, "own": 45, "heads": 32, "kv_heads": 32, "dim": 128,
         "ragged": True, "dtype": "bf16"},
        # a dozen users behind two pages of instructions
        {"name": "users_12", "kind": "shared", "batch": 12, "tokens": 1, "prefix": 2048, "own": 1019, "heads": 32, "kv_heads": 32, "dim": 128,
         "ragged": True, "dtype": "bf16"},
        # a server's batch behind long instructions, four query heads to a key head
        {"name": "users_64", "kind": "shared", "batch": 64, "tokens": 1, "prefix": 8192, "own": 512, "heads": 32, "kv_heads": 8, "dim": 128,
         "ragged": True, "dtype": "bf16"},
        # five tokens of eight sequences are checked at once, smaller heads
        {"name": "drafts_8x5", "kind": "shared", "batch": 8, "tokens": 5, "prefix": 4096, "own": 640, "heads": 32, "kv_heads": 32, "dim": 64,
         "ragged": False, "dtype": "f16"},
        # sixteen questions about one long document: the largest
        {"name": "document_16", "kind": "shared", "batch": 16, "tokens": 1, "prefix": 131072, "own": 257, "heads": 32, "kv_heads": 8, "dim": 128,
         "ragged": False, "dtype": "f16"},
        # a chat with one user: one token is drawn
        {"name": "sample_1", "kind": "verify", "batch": 1, "tokens": 1, "vocab": 32000, "drafts": "none", "temperature": 1.0, "ragged": False,
         "dtype": "bf16"},
        # four drafted tokens of eight sequences
        {"name": "verify_8x5", "kind": "verify", "batch": 8, "tokens": 5, "vocab": 32000, "drafts": "logits", "temperature": 0.75, "ragged": False,
         "dtype": "bf16"},
        # tokens looked up in the prompt, a large vocabulary of a size nobody chose
        {"name": "lookup_16x4", "kind": "verify", "batch": 16, "tokens": 4, "vocab": 100003, "drafts": "none", "temperature": 1.0, "ragged": True,
         "dtype": "f16"},
        # a server's batch, logits in 32 bits
        {"name": "verify_64x6", "kind": "verify", "batch": 64, "tokens": 6, "vocab": 32000, "drafts": "logits", "temperature": 1.0, "ragged": True,
         "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(("resize", "shared", "shared", "verify"))
    case = {"kind": kind, "ragged": rng.random() < 0.6}
    if kind == "resize":
        batch = _log(rng, 1, 512)
        tokens = rng.randint(1, 8) if rng.random() < 0.6 else _log(rng, 9, max(9, 65536 // batch))
        return dict(case, batch=batch, tokens=tokens, context=_log(rng, 1, 8192), shared=rng.choice((0, 0, _log(rng, 1, 64))))
    if kind == "verify":
        batch, tokens = _log(rng, 1, 64), rng.choice((1, rng.randint(2, 8)))
        return dict(case, batch=batch, tokens=tokens, vocab=_log(rng, 2048, max(2048, min(150000, 64 * 6 * 32000 // (batch * tokens)))),
                    drafts=rng.choice(("none", "logits")), temperature=rng.choice((0.0, 0.6, 1.0, 1.3)), dtype=rng.choice(("bf16", "f16", "f32")))
    heads, kv_heads = rng.choice(((32, 32), (32, 32), (32, 8), (32, 4), (12, 12), (16, 2), (24, 8), (8, 1)))
    dim = rng.choice((64, 64, 96, 128, 128, 128, 256))
    batch, tokens = _log(rng, 2, 64), rng.choice((1, 1, rng.randint(2, 8)))
    most = 16 * 32 * 128 * 131072  # of the largest listed case: rows times keys, and keys, of the prefix
    prefix = _log(rng, 128, max(128, min(131072, most // (batch * tokens * heads * dim), 131072 * 8 * 128 // (kv_heads * dim))))
    room = max(tokens + 16, 12 * 1019 * 32 * 128 // (batch * kv_heads * dim))
    return dict(case, batch=batch, tokens=tokens, prefix=prefix // BLOCK * BLOCK, own=_log(rng, tokens, min(4096, room)), heads=heads,
                kv_heads=kv_heads, dim=dim, dtype=rng.choice(("bf16", "f16")))


# ---------------------------------------------------------------------------------------------------- sizes --
def _spread(i):
    return (0.6180339887 * i) % 1.0


def lengths(case):
    """(tokens of its own that each sequence has after the pass, new ones among them): by the case alone. ``resize``: before the pass."""
    have, news = [], []
    for i in range(case["batch"]):
        n, new = case["context"] if case["kind"] == "resize" else case.get("own", case["tokens"]), case["tokens"]
        if case["ragged"] and i:
            n = max(1, n - int(0.75 * n * _spread(i)))
            new = 0 if new > 1 and i % 7 == 5 else 1 if i % 5 == 3 else max(1, new - int(0.75 * new * _spread(i)))
        have.append(n)
        news.append(new if case["kind"] == "resize" else min(n, new))
    return have, news


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    have, news = lengths(case)
    rows = sum(news)
    if case["kind"] == "resize":
        moved = sum(_blocks(n + new) - _blocks(n) for n, new in zip(have, news))
        # room is made: changes, lengths in and out, the list's blocks into the tables, a position and a slot for each row, first rows;
        # and given back: changes, lengths in and out, the tables' blocks into the list
        return {"bytes": case["batch"] * 4 * 7 + moved * 16 + rows * 16, "flops": 0}
    if case["kind"] == "verify":
        size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
        read = rows * case["vocab"] * size
        drafted = sum(max(0, new - 1) for new in news) * case["vocab"] * size if case["drafts"] == "logits" and case["temperature"] > 0 else 0
        return {"bytes": read + drafted + 8 * rows + case["batch"] * (8 * case["tokens"] + 4),
                "flops": (3 if case["temperature"] > 0 else 1) * (read + drafted) // size}
    d, hq, hk = case["dim"], case["heads"], case["kv_heads"]
    keys = case["prefix"] + sum(n for n, new in zip(have, news) if new)
    pairs = sum(case["prefix"] + n - new + 1 + t for n, new in zip(have, news) for t in range(new))
    return {"bytes": 2 * keys * hk * d + 8 * hk * (keys // BLOCK) + 2 * 2 * rows * hq * d, "flops": 4 * d * hq * pairs}


# --------------------------------------------------------------------------------------------------- inputs --
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    have, news = lengths(case)
    starts = [0]
    for new in news:
        starts.append(starts[-1] + new)
    state = {"case": case, "rows": starts[-1], "most": max(news)}
    make = {"resize": _prepare_resize, "shared": _prepare_shared, "verify": _prepare_verify}[case["kind"]]
    return make(state, case, gen, have, news, starts)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pool(gen, per, shared, spare):
    """(table [batch, blocks of the longest], blocks that nobody has): the first `shared` blocks of all sequences are the same."""
    own_blocks = [max(0, n - shared) for n in per]
    count = shared + sum(own_blocks) + spare
    order = torch.randperm(count, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((len(per), max(max(per), shared)), int(order[-1]), dtype=torch.int32), shared
    table[:, :shared] = order[:shared]
    for i, n in enumerate(own_blocks):
        table[i, shared:shared + n] = order[at:at + n]
        at += n
    return table, order[at:], count


def _prepare_resize(state, case, gen, have, news, starts):
    shared = case["shared"]
    lens = [shared * BLOCK + n for n in have]
    wanted = sum(_blocks(n + new) - _blocks(n) for n, new in zip(lens, news))
    table, free, pool = _pool(gen, [_blocks(n) for n in lens], shared, wanted + 5)
    wide = torch.full((len(lens), max(_blocks(n + new) for n, new in zip(lens, news)) + 3), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    stack = torch.full((pool,), -1, dtype=torch.int32)
    stack[:len(free)] = free
    change = _i32(news)
    return dict(state, block_table=wide.cuda(), seq_lens=_i32(lens), free_blocks=stack.cuda(), free_count=_i32([len(free)]), change=change,
                back=-change)


def _prepare_shared(state, case, gen, have, news, starts):
    shared, b, hk, d = case["prefix"] // BLOCK, case["batch"], case["kv_heads"], case["dim"]
    lens = [case["prefix"] + n for n in have]
    table, _, pool = _pool(gen, [_blocks(n) for n in lens], shared, 3)

    def normal(*shape):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, 1, generator=gen)

    def codes(*shape):
        c = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0, 34, generator=gen)  # the largest of 64 x dim values near 127
        return c.clamp_(-127, 127).round_().add_(128).to(torch.uint8)

    def scales():
        return torch.exp(0.2 * normal(pool, hk)) / 34

    return dict(state, block_table=table.cuda(), seq_lens=_i32(lens), cu_tokens=_i32(starts) if len(set(news)) > 1 else None, max_len=max(lens),
                shared=shared, k_codes=codes(pool, hk, BLOCK, d), v_codes=codes(pool, hk, BLOCK // 4, d, 4), k_scale=scales(), v_scale=scales(),
                q=normal(state["rows"], case["heads"], d).to(TYPES[case["dtype"]]))


def _prepare_verify(state, case, gen, have, news, starts):
    rows, vocab, dtype, heat = state["rows"], case["vocab"], TYPES[case["dtype"]], case["temperature"]

    def noise(kind, *shape):
        return getattr(torch.empty(shape, dtype=torch.float32, device="cuda"), kind)(generator=gen)

    # a few likely tokens before a long tail; the drafter's opinion is the target's with an error
    logits = noise("normal_", rows, vocab) * 2.0
    logits += noise("exponential_", rows, vocab)
    draft = (logits + 0.5 * noise("normal_", rows, vocab)).to(dtype) if case["drafts"] == "logits" else None
    logits = logits.to(dtype)
    if draft is not None:
        likely = draft.float() / heat - noise("exponential_", rows, vocab).log() if heat > 0 else draft.float()
        following = likely.argmax(-1)
    else:
        following = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.7, logits.float().argmax(-1),
                                torch.randint(0, vocab, (rows,), generator=gen, device="cuda"))
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")  # the first of each sequence
    first = set(starts)
    at = torch.tensor([r for r in range(rows) if r not in first], dtype=torch.int64, device="cuda")
    tokens[at] = following[at - 1]
    return dict(state, logits=logits, draft_logits=draft, tokens=tokens, cu_tokens=_i32(starts),
                accept_draws=torch.rand(rows, generator=gen, device="cuda") if heat > 0 else None,
                sample_draws=torch.rand(case["batch"], generator=gen, device="cuda") if heat > 0 else None)


# ------------------------------------------------------------------------------------------------- one pass --
def run(state):
    kind = state["case"]["kind"]
    if kind == "resize":
        return _resize_own(state) if own else _resize_plain(state)
    if kind == "shared":
        return _shared_own(state) if own else _shared_plain(state)
    return _verify_own(state) if own else _verify_plain(state)


def _resize_own(s):
    from latentq_llm_amd import ops
    books, shared = (s["block_table"], s["seq_lens"], s["free_blocks"], s["free_count"]), s["case"]["shared"]
    cu, positions, slots, status = ops.kv8_resize(*books, s["change"], rows=s["rows"], shared=shared)
    back = ops.kv8_resize(*books, s["back"], shared=shared)
    return {"cu_tokens": cu, "positions": positions, "slots": slots, "status": status, "status_back": back[3], "block_table": books[0],
            "seq_lens": books[1], "free_blocks": books[2], "free_count": books[3]}


def _shared_own(s):
    from latentq_llm_amd import ops
    return ops.kv8_attention_shared(s["q"], s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"], s["shared"],
                                    cu_tokens=s["cu_tokens"], max_tokens=s["most"], max_len=s["max_len"])


def _verify_own(s):
    from latentq_llm_amd import ops
    tokens, accepted = ops.verify_drafts(s["logits"], s["tokens"], s["cu_tokens"], draft_logits=s["draft_logits"], accept_draws=s["accept_draws"],
                                         sample_draws=s["sample_draws"], temperature=s["case"]["temperature"], max_tokens=s["most"])
    return {"tokens": tokens, "accepted": accepted}


def _resize_once(s, change, rows):
    """One change of all sequences' lengths. The blocks given back go onto the list before any are taken from it; a block's place in the order
    is its sequence's, then its own in the sequence; the first one taken, and the first one given back, is at the top of the list."""
    table, lens, free, count = s["block_table"], s["seq_lens"].long(), s["free_blocks"], s["free_count"].long()
    shared, (batch, width), pool = s["case"]["shared"], table.shape, free.shape[0]
    after = (lens + change.long()).clamp_min(0)
    have, need = ((n + BLOCK - 1).div(BLOCK, rounding_mode="floor").clamp_min(shared) for n in (lens, after))
    more, less, new = (need - have).clamp_min(0), (have - need).clamp_min(0), (after - lens).clamp_min(0)
    more_sum, less_sum, total = more.sum(), less.sum(), new.sum()
    # 0: done; else nothing changes: the number of blocks that are missing, -1: a table is too narrow, -2: more new tokens than rows
    missing = (more_sum - less_sum - count).clamp_min(0)[0]
    status = torch.where((need > width).any(), -1, torch.where(total > rows, -2, missing))
    good = status == 0
    index = torch.arange(width, device="cuda")
    at = index - need[:, None]
    leaving = good & (at >= 0) & (index < have[:, None])
    place = count + less_sum - 1 - ((less.cumsum(0) - less)[:, None] + at)
    ext = torch.cat((free, free.new_zeros(1)))
    ext.scatter_(0, torch.where(leaving, place, pool).flatten(), torch.where(leaving, table, 0).flatten())
    at = index - have[:, None]
    coming = good & (at >= 0) & (index < need[:, None])
    place = count + less_sum - 1 - ((more.cumsum(0) - more)[:, None] + at)
    table.copy_(torch.where(coming, ext[torch.where(coming, place, pool)], table))
    free.copy_(ext[:-1])
    s["free_count"].copy_(torch.where(good, count + less_sum - more_sum, count))
    s["seq_lens"].copy_(torch.where(good, after, lens))
    cu = torch.cat((new.new_zeros(1), torch.where(good, new.cumsum(0), 0)))
    row = torch.arange(rows, device="cuda")
    seq = torch.bucketize(row, cu[1:], right=True).clamp(max=batch - 1)
    there = row < cu[-1]
    positions = torch.where(there, lens[seq] + row - cu[seq], 0)
    block = table[seq, (positions // BLOCK).clamp(max=width - 1)].long()
    slots = torch.where(there, block * BLOCK + positions % BLOCK, -1)
    return cu.int(), positions, slots, status.int().view(1)


def _resize_plain(s):
    cu, positions, slots, status = _resize_once(s, s["change"], s["rows"])
    back = _resize_once(s, s["back"], 0)
    return {"cu_tokens": cu, "positions": positions, "slots": slots, "status": status, "status_back": back[3], "block_table": s["block_table"],
            "seq_lens": s["seq_lens"], "free_blocks": s["free_blocks"], "free_count": s["free_count"]}


def _places(cu, rows, batch):
    """(sequence, place among the sequence's rows) of each row, and rows of each sequence."""
    at = torch.arange(rows, device="cuda")
    if cu is None:
        seq = at // (rows // batch)
        return seq, at % (rows // batch), torch.full((batch,), rows // batch, dtype=torch.int64, device="cuda")
    cu = cu.long()
    seq = torch.bucketize(at, cu[1:], right=True)
    return seq, at - cu[seq], cu[1:] - cu[:-1]


def _values(s, blocks):
    """Keys and values of the blocks, [..., 64, kv_heads, dim]."""
    n = blocks.dim()
    k = (s["k_codes"][blocks].float() - 128) * s["k_scale"][blocks][..., None, None]
    v = (s["v_codes"][blocks].float() - 128) * s["v_scale"][blocks][..., None, None, None]
    v = v.transpose(-1, -2).reshape(k.shape)
    return k.transpose(n, n + 1), v.transpose(n, n + 1)


def _shared_plain(s):
    q, lens, table, shared, most = s["q"], s["seq_lens"].long(), s["block_table"].long(), s["shared"], s["most"]
    b, hk, d = lens.numel(), s["k_codes"].shape[1], q.shape[-1]
    group = q.shape[1] // hk
    seq, place, new = _places(s["cu_tokens"], q.shape[0], b)
    rows = torch.zeros((b, most, hk, group, d), dtype=torch.float32, device="cuda")
    rows[seq, place] = q.float().view(-1, hk, group, d) / math.sqrt(d)
    kp, vp = (x.reshape(-1, hk, d).transpose(0, 1).contiguous() for x in _values(s, table[0, :shared]))  # [kv head, key, dim]
    ko, vo = (x.reshape(b, -1, hk, d).transpose(1, 2).contiguous() for x in _values(s, table[:, shared:]))  # [b, kv head, key, dim]
    of_prefix = rows.permute(2, 0, 1, 3, 4).reshape(hk, -1, d) @ kp.transpose(1, 2).contiguous()
    of_own = rows.permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d) @ ko.transpose(2, 3).contiguous()
    of_prefix, of_own = of_prefix.view(hk, b, most, group, -1), of_own.view(b, hk, most, group, -1).transpose(0, 1)
    at = (lens - new)[:, None] + torch.arange(most, device="cuda")  # [b, row]
    of_prefix.masked_fill_((torch.arange(shared * BLOCK, device="cuda") > at[..., None])[:, :, None], -math.inf)
    of_own = of_own.masked_fill((torch.arange(of_own.shape[-1], device="cuda") + shared * BLOCK > at[..., None])[:, :, None], -math.inf)
    top = torch.maximum(of_prefix.amax(-1, keepdim=True), of_own.amax(-1, keepdim=True)).clamp_min(-3e38)
    of_prefix.sub_(top).exp_()
    of_own.sub_(top).exp_()
    total = of_prefix.sum(-1, keepdim=True) + of_own.sum(-1, keepdim=True)
    out = (of_prefix.view(hk, b * most * group, -1) @ vp).view(hk, b, most, group, d)
    out = out + (of_own.reshape(hk, b, most * group, -1) @ vo.transpose(0, 1).contiguous()).view(hk, b, most, group, d)
    out = out / total.clamp_min(1e-38)
    return out.permute(1, 2, 0, 3, 4)[seq, place].reshape(q.shape).to(q.dtype)


def _probabilities(logits, heat):
    x = logits.double()
    x = x.masked_fill(x.isnan(), -math.inf).clamp(max=float(np.finfo(np.float32).max))
    x = ((x - x.amax(-1, keepdim=True).clamp_min(-1e300)) * (1.0 / heat)).exp_()
    return x / x.sum(-1, keepdim=True).clamp_min(1e-300)


def _verify_plain(s):
    logits, tokens, cu, heat, most = s["logits"], s["tokens"], s["cu_tokens"].long(), s["case"]["temperature"], s["most"]
    (rows, vocab), batch = logits.shape, cu.numel() - 1
    seq, place, n = _places(cu, rows, batch)
    drafted = place + 1 < n[seq]
    following = torch.where(drafted, tokens.roll(-1), 0)
    if heat > 0:
        p = _probabilities(logits, heat)
        q = _probabilities(s["draft_logits"], heat) if s["draft_logits"] is not None else None
        of_draft = q.gather(1, following[:, None])[:, 0] if q is not None else 1.0
        taken = s["accept_draws"].double() * of_draft < p.gather(1, following[:, None])[:, 0]
    else:
        best = logits.argmax(-1)
        taken = following == best
    refused = torch.where(drafted & ~taken, place, most)
    accepted = torch.full((batch,), most, device="cuda").scatter_reduce(0, seq, refused, "amin").minimum((n - 1).clamp_min(0))
    row = (cu[:-1] + accepted).clamp(max=rows - 1)
    if heat > 0:
        p, at = p[row], following[row]
        if q is not None:
            rest = (p - q[row]).clamp_min(0)
        else:
            rest = p.scatter(1, at[:, None], 0.0)
        rest = torch.where(drafted[row, None], rest, p)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
        upto = rest.cumsum(-1)
        beyond = upto > s["sample_draws"].double()[:, None] * upto[:, -1:]
        last = vocab - 1 - (rest > 0).flip(-1).byte().argmax(-1)
        last = torch.where(beyond.any(-1), beyond.byte().argmax(-1), last)
    else:
        last = best[row]
    index = torch.arange(most, device="cuda")
    given = tokens[(cu[:-1, None] + 1 + index).clamp(max=rows - 1)]
    out = torch.where(index < accepted[:, None], given, torch.where(index == accepted[:, None], last[:, None], -1))
    return {"tokens": torch.where((n > 0)[:, None], out, -1), "accepted": accepted.int()}


# --------------------------------------------------------------------------------------------- in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    return {"resize": _resize_exact, "shared": _shared_exact, "verify": _verify_exact}[case["kind"]](s)


def _resize_exact(s):
    table, lens, stack = s["block_table"].tolist(), s["seq_lens"].tolist(), s["free_blocks"].tolist()
    count, shared = s["free_count"].item(), s["case"]["shared"]

    def once(change, count):
        cu, positions, slots = [0], [], []
        left = [(i, j) for i, c in enumerate(change) if c < 0 for j in range(max(shared, _blocks(lens[i] + c)), max(shared, _blocks(lens[i])))]
        for i, j in reversed(left):
            stack[count] = table[i][j]
            count += 1
        for i, c in enumerate(change):
            for j in range(max(shared, _blocks(lens[i])), max(shared, _blocks(lens[i] + c))):
                count -= 1
                table[i][j] = stack[count]
            for p in range(lens[i], lens[i] + c):
                positions.append(p)
                slots.append(table[i][p // BLOCK] * BLOCK + p % BLOCK)
            lens[i] += c
            cu.append(cu[-1] + max(0, c))
        return cu, positions, slots, count

    cu, positions, slots, count = once(s["change"].tolist(), count)
    count = once(s["back"].tolist(), count)[3]
    i64 = dict(dtype=torch.int64, device="cuda")
    return {"cu_tokens": _i32(cu), "positions": torch.tensor(positions, **i64), "slots": torch.tensor(slots, **i64), "status": _i32([0]),
            "status_back": _i32([0]), "block_table": _i32(table), "seq_lens": _i32(lens), "free_blocks": _i32(stack), "free_count": _i32([count])}


def _shared_exact(s):
    q, table, group = s["q"].double(), s["block_table"].long(), s["q"].shape[1] // s["k_codes"].shape[1]
    have, news = lengths(s["case"])
    hk, d, out, start = s["k_codes"].shape[1], q.shape[-1], torch.empty_like(q), 0

    def dense(blocks, h):
        k = ((s["k_codes"][blocks, h].double() - 128) * s["k_scale"][blocks, h].double()[:, None, None]).reshape(-1, d)
        v = (s["v_codes"][blocks, h].double() - 128) * s["v_scale"][blocks, h].double()[:, None, None, None]
        return k, v.permute(0, 1, 3, 2).reshape(-1, d)

    common = [dense(table[0, :s["shared"]], h) for h in range(hk)]
    for i, (n, new) in enumerate(zip(have, news)):
        n += s["case"]["prefix"]
        if not new:
            continue
        at = torch.arange(n - new, n, device="cuda").repeat_interleave(group)[:, None]
        for h in range(hk):
            mine = dense(table[i, s["shared"]:_blocks(n)], h)
            k, v = (torch.cat((a, b))[:n] for a, b in zip(common[h], mine))
            rows = q[start:start + new, h * group:(h + 1) * group].reshape(-1, d)
            score = (rows @ k.t().contiguous() / math.sqrt(d)).masked_fill_(torch.arange(n, device="cuda") > at, -math.inf)
            out[start:start + new, h * group:(h + 1) * group] = (torch.softmax(score, -1) @ v).view(new, group, d)
        start += new
    return out


def _verify_exact(s):
    heat, cu, tokens = s["case"]["temperature"], s["cu_tokens"].tolist(), s["tokens"].tolist()
    logits = s["logits"].float().cpu().numpy()
    draft = s["draft_logits"].float().cpu().numpy() if s["draft_logits"] is not None else None
    accept, sample = ((s[x].cpu().numpy().astype(np.float64) if s[x] is not None else None) for x in ("accept_draws", "sample_draws"))

    def softmax(x):
        x = x.astype(np.float64) / heat
        e = np.exp(x - x.max())
        return e / e.sum()

    out, counts = np.full((len(cu) - 1, s["most"]), -1, dtype=np.int64), []
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        taken = 0
        for r in range(a, b):
            x = tokens[r + 1] if r + 1 < b else None
            if heat > 0:
                rest = softmax(logits[r])
                if x is not None:
                    q = softmax(draft[r]) if draft is not None else np.eye(1, rest.size, x)[0]
                    if accept[r] * q[x] < rest[x]:
                        out[i, taken] = x
                        taken += 1
                        continue
                    rest = np.maximum(rest - q, 0.0)
                upto = np.cumsum(rest)
                out[i, taken] = np.searchsorted(upto, sample[i] * upto[-1], side="right")
            else:
                best = int(logits[r].argmax())
                out[i, taken] = best
                if x == best:
                    taken += 1
                    continue
            break
        counts.append(taken)
    return {"tokens": torch.from_numpy(out).cuda(), "accepted": _i32(counts)}
