"""The operators around a paged 8-bit cache of keys and values, as cases to be timed: what a generation loop does in
attention between the quantised projections of a decoder layer.

kind     one pass
append   ``ops.kv8_append``: keys (rotated by their position) and values of the new tokens are rounded to 8 bits into the
         blocks of their sequences, the queries are rotated on the way; then ``ops.kv8_read``, which gives the blocks that
         changed as the values they stand for
attend   ``ops.kv8_attention``: attention of the last tokens of each sequence over all that the cache holds of it

The cache is a pool of blocks of 64 tokens, shared by the sequences of a batch; ``block_table`` lists each sequence's blocks.
  k_codes  uint8 [blocks, kv_heads, 64, dim]       v_codes  uint8 [blocks, kv_heads, 16, dim, 4]
  k_scale  float32 [blocks, kv_heads]              v_scale  float32 [blocks, kv_heads]
A code u stands for (u - 128) * scale. v_codes keeps four consecutive tokens of one dimension together: token t of a block is
at [t // 4, :, t % 4].

Keys and values are N(0, 1) with a few channels of keys four times that, as rotated keys have them; queries N(0, 1). Blocks
are drawn from the pool in random order. ``ragged``: sequences of the batch differ in length (down to a quarter) and in
the number of new tokens (some have one, or none).
"""
import math

import torch

own = False

BLOCK = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
LEAST = 2.0 ** -90  # the least magnitude that a block's scale is made for


def listed():
    return [
        # a chat with one user: the cache takes one token
        {"name": "append_1", "kind": "append", "batch": 1, "tokens": 1, "context": 1019, "heads": 32, "kv_heads": 32, "dim": 128,
         "rotate": True, "ragged": False, "dtype": "bf16"},
        # four prompts of up to 512 tokens in a model with learned positions (nothing to rotate), lengths nobody chose
        {"name": "append_4x512", "kind": "append", "batch": 4, "tokens": 512, "context": 512, "heads": 32, "kv_heads": 32, "dim": 64,
         "rotate": False, "ragged": True, "dtype": "bf16"},
        # two long prompts behind a short prefix, four query heads to a key head
        {"name": "append_2x4096", "kind": "append", "batch": 2, "tokens": 4096, "context": 4133, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotate": True, "ragged": False, "dtype": "f16"},
        # a chat with one user: one token attends to a page of text
        {"name": "decode_1", "kind": "attend", "batch": 1, "tokens": 1, "context": 1019, "heads": 32, "kv_heads": 32, "dim": 128,
         "window": 0, "ragged": False, "dtype": "bf16"},
        # a dozen sequences generated together, of different lengths
        {"name": "decode_12", "kind": "attend", "batch": 12, "tokens": 1, "context": 4096, "heads": 32, "kv_heads": 32, "dim": 128,
         "window": 0, "ragged": True, "dtype": "bf16"},
        # a server's batch, four query heads to a key head
        {"name": "decode_64", "kind": "attend", "batch": 64, "tokens": 1, "context": 8192, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "ragged": True, "dtype": "bf16"},
        # one sequence of 128 K tokens
        {"name": "decode_128k", "kind": "attend", "batch": 1, "tokens": 1, "context": 131072, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "ragged": False, "dtype": "f16"},
        # five drafted tokens of eight sequences are checked at once, smaller heads
        {"name": "verify_8x5", "kind": "attend", "batch": 8, "tokens": 5, "context": 2048, "heads": 32, "kv_heads": 32, "dim": 64,
         "window": 0, "ragged": False, "dtype": "f16"},
        # a short question
        {"name": "prompt_45", "kind": "attend", "batch": 1, "tokens": 45, "context": 45, "heads": 32, "kv_heads": 32, "dim": 128,
         "window": 0, "ragged": False, "dtype": "bf16"},
        # four prompts of up to a page, smaller heads
        {"name": "prompt_4x1019", "kind": "attend", "batch": 4, "tokens": 1019, "context": 1019, "heads": 32, "kv_heads": 32, "dim": 64,
         "window": 0, "ragged": True, "dtype": "bf16"},
        # a long prompt: the largest
        {"name": "prompt_8192", "kind": "attend", "batch": 1, "tokens": 8192, "context": 8192, "heads": 32, "kv_heads": 32, "dim": 128,
         "window": 0, "ragged": False, "dtype": "bf16"},
        # one more piece of a long prompt that is taken in pieces, four query heads to a key head
        {"name": "piece_512", "kind": "attend", "batch": 1, "tokens": 512, "context": 16384, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "ragged": False, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    """An integer of lo..hi, spread over its logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    heads, kv_heads = rng.choice(((32, 32), (32, 32), (32, 8), (32, 4), (12, 12), (16, 2), (24, 8), (8, 1)))
    case = {"kind": rng.choice(("append", "attend", "attend", "attend")), "heads": heads, "kv_heads": kv_heads,
            "dim": rng.choice((64, 64, 96, 128, 128, 128, 256)), "dtype": rng.choice(("bf16", "f16")), "ragged": rng.random() < 0.5}
    if case["kind"] == "append":
        one = rng.random() < 0.4
        tokens = 1 if one else _log(rng, 2, 8192)
        batch = _log(rng, 1, max(1, min(64, 8192 // tokens)))
        before = _log(rng, 1, 4096) if one else rng.choice((0, _log(rng, 1, 2048)))
        return dict(case, batch=batch, tokens=tokens, context=tokens + before, rotate=rng.random() < 0.75)
    how = rng.choice(("decode", "decode", "few", "prompt", "prompt", "piece"))
    tokens = 1 if how == "decode" else rng.randint(2, 8) if how == "few" else _log(rng, 9, 4096) if how == "prompt" else _log(rng, 64, 1024)
    batch = _log(rng, 1, 64) if how in ("decode", "few") else _log(rng, 1, max(1, 4096 // tokens))
    if how == "prompt":
        context = tokens
    else:  # no more bytes in the cache than the largest listed batch has
        context = _log(rng, max(16, tokens), max(tokens + 16, min(131072, 64 * 8192 * 8 * 128 // (batch * kv_heads * case["dim"]))))
        if how == "piece":
            context = max(tokens, min(context, 4096 * 4096 // (batch * tokens)))
    window = _log(rng, 16, 4096) if rng.random() < 0.25 else 0
    return dict(case, batch=batch, tokens=tokens, context=context, window=window)


# ---------------------------------------------------------------------------------------------------- sizes --
def lengths(case):
    """(tokens in the cache after the call, new tokens) of each sequence: by the case alone."""
    lens, news = [], []
    for i in range(case["batch"]):
        n, new = case["context"], case["tokens"]
        if case["ragged"] and i:
            n = max(1, n - int(0.75 * n * ((0.6180339887 * i) % 1.0)))
            new = 0 if new > 1 and i % 7 == 5 else 1 if i % 5 == 3 else max(1, new - int(0.75 * new * ((0.6180339887 * i) % 1.0)))
        lens.append(n)
        news.append(min(n, new))
    return lens, news


def _visible(n, new, window):
    """Keys that the new tokens of one sequence attend to, in all, and how many of them are different ones."""
    at = range(n - new, n)
    pairs = sum(min(p + 1, window) if window else p + 1 for p in at)
    return pairs, (min(n, window + new - 1) if window else n) if new else 0


def work(case):
    lens, news = lengths(case)
    total, d, hq, hk = sum(news), case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        blocks = sum(_touched(n, new) for n, new in zip(lens, news))
        new_in = 2 * 2 * total * hk * d + (2 * 2 * total * hq * d if case["rotate"] else 0)  # k, v; q in and out
        tables = 4 * total * d if case["rotate"] else 0
        codes = 2 * total * hk * d
        read = 2 * blocks * BLOCK * hk * d * 3  # codes in, 16-bit values out
        return {"bytes": new_in + tables + codes + read, "flops": total * d * (6 * hk + (3 * hq if case["rotate"] else 0))}
    seen = [_visible(n, new, case["window"]) for n, new in zip(lens, news)]
    keys = sum(s[1] for s in seen)
    return {"bytes": 2 * keys * hk * d + 8 * hk * (keys // BLOCK) + 2 * 2 * total * hq * d, "flops": 4 * d * hq * sum(s[0] for s in seen)}


def _touched(n, new):
    return (n - 1) // BLOCK - (n - new) // BLOCK + 1 if new else 0


# --------------------------------------------------------------------------------------------------- inputs --
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, news = lengths(case)
    b, hk, d, dtype = case["batch"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
    per = [-(-n // BLOCK) for n in lens]
    width, pool = max(per), sum(per) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32).cpu()
    table, at = torch.full((b, width), int(order[-1]), dtype=torch.int32), 0  # a block that no sequence has where a row is longer than its sequence
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for new in news:
        starts.append(starts[-1] + new)
    total = starts[-1]

    def normal(*shape):
        return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0, 1, generator=gen)

    def codes(*shape):
        c = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0, 34, generator=gen)  # the largest of 64 x dim values near 127
        return c.clamp_(-127, 127).round_().add_(128).to(torch.uint8)

    def scales():
        return torch.exp(0.2 * normal(pool, hk)) / 34

    ragged = len(set(news)) > 1
    state = {"case": case, "block_table": table.cuda(), "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "cu_tokens": torch.tensor(starts, dtype=torch.int32, device="cuda") if ragged else None,
             "max_tokens": max(news), "max_len": max(lens),
             "k_codes": codes(pool, hk, BLOCK, d), "v_codes": codes(pool, hk, BLOCK // 4, d, 4), "k_scale": scales(), "v_scale": scales(),
             "q": normal(total, case["heads"], d).to(dtype)}
    if case["kind"] == "append":
        k = normal(total, hk, d)
        k[:, :, :: d // 4] *= 4
        state["k"], state["v"] = k.to(dtype), normal(total, hk, d).to(dtype)
        touched = [table[i, (n - new) // BLOCK:(n - 1) // BLOCK + 1] for i, (n, new) in enumerate(zip(lens, news)) if new]
        state["blocks"] = torch.cat(touched).cuda()
        state["cos"] = state["sin"] = None
        if case["rotate"]:
            rate = 10000.0 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d // 2))
            angle = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * rate
            state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


# ------------------------------------------------------------------------------------------------- one pass --
def run(state):
    if state["case"]["kind"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def _cache(s):
    return s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"]


def _append_own(s):
    from latentq_llm_amd import ops
    q = ops.kv8_append(s["k"], s["v"], *_cache(s), s["block_table"], s["seq_lens"], q=s["q"] if s["cos"] is not None else None,
                       cos=s["cos"], sin=s["sin"], cu_tokens=s["cu_tokens"], max_tokens=s["max_tokens"])
    k, v = ops.kv8_read(*_cache(s), s["blocks"], dtype=s["k"].dtype)
    return {"q": q, "k": k, "v": v}


def _attend_own(s):
    from latentq_llm_amd import ops
    return ops.kv8_attention(s["q"], *_cache(s), s["block_table"], s["seq_lens"], cu_tokens=s["cu_tokens"], max_tokens=s["max_tokens"],
                             max_len=s["max_len"], window=s["case"]["window"])


def _tokens(s):
    """(sequence, position in the sequence, place among the sequence's new tokens) of each new token, and new tokens of each sequence."""
    total, lens = s["q"].shape[0], s["seq_lens"].long()
    at = torch.arange(total, device="cuda")
    if s["cu_tokens"] is None:
        new = torch.full_like(lens, total // lens.numel())
        seq = at // max(1, total // lens.numel())
        place = at - seq * (total // lens.numel())
    else:
        cu = s["cu_tokens"].long()
        new = cu[1:] - cu[:-1]
        seq = torch.bucketize(at, cu[1:], right=True)
        place = at - cu[seq]
    return seq, (lens - new)[seq] + place, place, new


def _rotated(x, cos, sin):
    x, half = x.float(), x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = cos[:, None], sin[:, None]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _append_plain(s):
    seq, pos, _, new = _tokens(s)
    lens, table = s["seq_lens"].long(), s["block_table"].long()
    before = lens - new
    q, k, v = None, s["k"].float(), s["v"].float()
    if s["cos"] is not None:
        cos, sin = s["cos"][pos], s["sin"][pos]
        q, k = _rotated(s["q"], cos, sin).to(s["q"].dtype), _rotated(s["k"], cos, sin)
    block, slot = table[seq, pos // BLOCK], pos % BLOCK
    # the blocks that the new tokens begin in: what they hold so far is rounded again where their scale grows
    part = (before % BLOCK) * (new > 0)
    first = table.gather(1, (before // BLOCK).clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    for_old = (torch.arange(BLOCK, device="cuda") < part[:, None])[:, None, :, None]
    touched = torch.zeros(s["k_scale"].shape[0], dtype=torch.bool, device="cuda")
    touched[block] = True
    for x, codes, scale in ((k, s["k_codes"], s["k_scale"]), (v, s["v_codes"], s["v_scale"])):
        in_v = codes.dim() == 5
        most = x.abs().masked_fill(~x.isfinite(), 0).amax(-1)
        amax = torch.zeros_like(scale).scatter_reduce(0, block[:, None].expand(-1, x.shape[1]), most, "amax")
        held = torch.zeros_like(scale)
        held[first] = torch.where((part > 0)[:, None], scale[first], held[first])
        grown = torch.where(touched[:, None], torch.maximum(held, amax.clamp_min(LEAST) * (1.0 / 127)), scale)
        old = codes[first]
        if in_v:
            old = old.transpose(-1, -2).reshape(old.shape[0], old.shape[1], BLOCK, -1)
        ratio = (held[first] / grown[first])[:, :, None, None]
        again = torch.where(for_old & (ratio < 1), ((old.float() - 128) * ratio).round() + 128, old.float()).to(torch.uint8)
        if in_v:
            again = again.view(again.shape[0], again.shape[1], BLOCK // 4, 4, -1).transpose(-1, -2)
        codes[first] = again
        scale.copy_(grown)
        u = ((x * grown[block].reciprocal()[:, :, None]).round().clamp(-127, 127) + 128).nan_to_num(128.0).to(torch.uint8)
        if in_v:
            codes[block, :, slot // 4, :, slot % 4] = u
        else:
            codes[block, :, slot] = u
    kk, vv = _values(s, s["blocks"].long())
    return {"q": q, "k": kk.to(s["k"].dtype), "v": vv.to(s["k"].dtype)}


def _values(s, blocks):
    """Keys and values of the blocks, [..., 64, kv_heads, dim]."""
    n = blocks.dim()
    k = (s["k_codes"][blocks].float() - 128) * s["k_scale"][blocks][..., None, None]
    v = (s["v_codes"][blocks].float() - 128) * s["v_scale"][blocks][..., None, None, None]
    v = v.transpose(-1, -2).reshape(k.shape)
    return k.transpose(n, n + 1), v.transpose(n, n + 1)


def _attend_plain(s):
    seq, pos, place, new = _tokens(s)
    q, (b, hk, d) = s["q"], (s["seq_lens"].numel(), s["k_codes"].shape[1], s["q"].shape[-1])
    group, most, window = q.shape[1] // hk, s["max_tokens"], s["case"]["window"]
    k, v = _values(s, s["block_table"].long()[:, :-(-s["max_len"] // BLOCK)])
    k = k.reshape(b, -1, hk, d).permute(0, 2, 3, 1).contiguous()  # [b, kv head, dim, key]
    v = v.reshape(b, -1, hk, d).permute(0, 2, 1, 3).contiguous()  # [b, kv head, key, dim]
    rows = torch.zeros((b, most, hk, group, d), dtype=torch.float32, device="cuda")
    rows[seq, place] = q.float().view(-1, hk, group, d) / math.sqrt(d)
    score = (rows.permute(0, 2, 3, 1, 4).reshape(b, hk, group * most, d) @ k).view(b, hk, group, most, -1)
    at = (s["seq_lens"].long() - new)[:, None] + torch.arange(most, device="cuda")  # [b, row]
    key = torch.arange(score.shape[-1], device="cuda")
    hidden = key > at[..., None]
    if window:
        hidden |= key <= at[..., None] - window
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.view(b, hk, group * most, -1) @ v
    out = out.view(b, hk, group, most, d) / total.clamp_min(1e-38)
    return out.permute(0, 3, 1, 2, 4)[seq, place].reshape(q.shape).to(q.dtype)


# --------------------------------------------------------------------------------------------- in 64 bits --
def exact(case, seed):
    s = prepare(case, seed)
    lens, news = lengths(case)
    return _append_exact(s, lens, news) if case["kind"] == "append" else _attend_exact(s, lens, news)


def _turned(x, cos, sin):
    half = x.shape[-1] // 2
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    return torch.cat((x[..., :half] * cos - x[..., half:] * sin, x[..., half:] * cos + x[..., :half] * sin), -1)


def _dense(codes, block):
    """Codes of one block as [64, kv_heads, dim]."""
    c = codes[block].double() - 128
    if c.dim() == 4:
        c = c.permute(1, 3, 0, 2).reshape(BLOCK, c.shape[0], -1)
    else:
        c = c.permute(1, 0, 2)
    return c


def _append_exact(s, lens, news):
    table, q, given = s["block_table"].tolist(), [], {"k": [], "v": []}
    start = 0
    for i, (n, new) in enumerate(zip(lens, news)):
        if not new:
            continue
        first, rows = n - new, slice(start, start + new)
        start += new
        x = {"k": s["k"][rows].double(), "v": s["v"][rows].double()}
        if s["cos"] is not None:
            cos, sin = s["cos"][first:n], s["sin"][first:n]
            x["k"] = _turned(x["k"], cos, sin)
            q.append(_turned(s["q"][rows].double(), cos, sin))
        for place in range(first // BLOCK, (n - 1) // BLOCK + 1):
            block, lo, hi = table[i][place], max(first, place * BLOCK), min(n, place * BLOCK + BLOCK)
            for name in ("k", "v"):
                codes, mine = _dense(s[name + "_codes"], block), x[name][lo - first:hi - first]
                held = s[name + "_scale"][block].double()
                scale = mine.abs().amax((0, 2)).clamp_min(LEAST) / 127
                kept = lo - place * BLOCK  # tokens that the block holds already
                if kept:
                    scale = torch.maximum(scale, held)
                    codes[:kept] = torch.round(codes[:kept] * (held / scale)[:, None])
                codes[kept:hi - place * BLOCK] = torch.round(mine / scale[:, None]).clamp(-127, 127)
                given[name].append(codes * scale[:, None])
    return {"q": torch.cat(q) if q else None, "k": torch.stack(given["k"]), "v": torch.stack(given["v"])}


def _attend_exact(s, lens, news):
    q, table, window = s["q"].double(), s["block_table"].long(), s["case"]["window"]
    hk, d = s["k_codes"].shape[1], q.shape[-1]
    group, out, start = q.shape[1] // hk, torch.empty_like(q), 0
    for i, (n, new) in enumerate(zip(lens, news)):
        if not new:
            continue
        mine = q[start:start + new]
        blocks = table[i, :-(-n // BLOCK)]
        at = torch.arange(n - new, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = key <= at
        if window:
            seen &= key > at - window
        for h in range(hk):
            k = ((s["k_codes"][blocks, h].double() - 128) * s["k_scale"][blocks, h].double()[:, None, None]).reshape(-1, d)[:n]
            v = (s["v_codes"][blocks, h].double() - 128) * s["v_scale"][blocks, h].double()[:, None, None, None]
            v = v.permute(0, 1, 3, 2).reshape(-1, d)[:n].contiguous()
            for g in range(h * group, (h + 1) * group):
                score = (mine[:, g].contiguous() @ k.t().contiguous() / math.sqrt(d)).masked_fill_(~seen, -math.inf)
                out[start:start + new, g] = torch.softmax(score, -1) @ v
        start += new
    return out
