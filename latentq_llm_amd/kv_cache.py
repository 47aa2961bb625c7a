"""A paged 8-bit cache of keys and values, and the attention of a decoder layer over it, for generation.

``KVCache8`` holds the blocks of one layer (layout and rounding: include/latentq.h, lq_kv8_*), ``Sequences`` which blocks each
sequence has (one for all layers), ``CachedAttention`` the four projections of a layer with the operators between them:
rotation and appending in one launch, attention over the cache in one or two. ``DeviceSequences`` keeps the same books on the
device, for a batch that may begin with blocks in common and whose lengths follow from what the device computed (drafted tokens that
were accepted): a pass can be captured into a graph. The reference's counterparts are the rotation of
PTQ/quant/fused_attn.py:8-93 and the tensor library's cache and attention, in 16 bits. Inference only.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn as nn

from . import ops

BLOCK = ops.KV_BLOCK


class KVCache8:
    """Blocks of 64 tokens for the kv heads of one layer: 2 * head_dim bytes a token and head, and 8 a block and head."""

    def __init__(self, num_blocks: int, kv_heads: int, head_dim: int, device="cuda"):
        if head_dim not in ops.KV_DIMS:
            raise ValueError(f"head_dim must be one of {ops.KV_DIMS}, got {head_dim}")
        if num_blocks < 1 or kv_heads < 1:
            raise ValueError("the cache needs at least one block and one kv head")
        self.num_blocks, self.kv_heads, self.head_dim = num_blocks, kv_heads, head_dim
        u8, f32 = dict(dtype=torch.uint8, device=device), dict(dtype=torch.float32, device=device)
        self.k_codes = torch.full((num_blocks, kv_heads, BLOCK, head_dim), 128, **u8)
        self.v_codes = torch.full((num_blocks, kv_heads, BLOCK // 4, head_dim, 4), 128, **u8)
        self.k_scale, self.v_scale = torch.ones((num_blocks, kv_heads), **f32), torch.ones((num_blocks, kv_heads), **f32)

    def tensors(self):
        return self.k_codes, self.v_codes, self.k_scale, self.v_scale

    def _holds(self, step: "Step") -> None:
        if step.pool > self.num_blocks:  # (the kernels would drop its tokens and read another block)
            raise ValueError(f"the pass uses block {step.pool - 1} of a cache of {self.num_blocks} blocks")

    def append(self, k, v, step: "Step", q=None, cos=None, sin=None):
        """ops.kv8_append of a step's new tokens; returns the rotated q, or None. Raises, and appends nothing, where a sequence has outgrown the
        rotation tables or its blocks are not of this cache (Sequences has counted the tokens by then: such a sequence is to be dropped)."""
        self._holds(step)
        if cos is not None and step.longest > cos.shape[0]:  # (the kernel would turn what lies beyond by the last row)
            raise ValueError(f"the rotation tables have {cos.shape[0]} positions, a sequence {step.longest} tokens")
        return ops.kv8_append(k, v, *self.tensors(), step.block_table, step.seq_lens, q=q, cos=cos, sin=sin, cu_tokens=step.cu_tokens,
                              max_tokens=step.max_tokens)

    def attend(self, q, step: "Step", scale=None, window=0):
        """ops.kv8_attention of a step's new tokens over what the cache holds of their sequences (kv8_attention_shared of sequences that
        begin with blocks in common). Rows that have no token are zeros."""
        self._holds(step)
        # (what follows may look at all rows, as a projection does that finds one scale for all of them)
        out = torch.zeros_like(q, memory_format=torch.contiguous_format) if step.padded and step.cu_tokens is not None else None
        if step.shared and not window:
            return ops.kv8_attention_shared(q, *self.tensors(), step.block_table, step.seq_lens, step.shared, cu_tokens=step.cu_tokens, max_tokens=step.max_tokens,
                                            max_len=step.max_len, scale=scale, out=out)
        return ops.kv8_attention(q, *self.tensors(), step.block_table, step.seq_lens, cu_tokens=step.cu_tokens, max_tokens=step.max_tokens,
                                 max_len=step.max_len, scale=scale, window=window, out=out)

    def read(self, blocks, dtype=torch.bfloat16):
        """ops.kv8_read: (keys, values) [n, 64, kv_heads, head_dim] of blocks."""
        return ops.kv8_read(*self.tensors(), blocks, dtype=dtype)


@dataclass
class Step:
    """The new tokens of a pass: tensors on the device and the host's bounds that size the launches. Rows of the operands are the
    sequences' new tokens one after the other. longest and pool are what the host knows exactly, for checks."""
    block_table: torch.Tensor  # int32 [sequences, blocks of the longest]
    seq_lens: torch.Tensor     # int32 [sequences], new tokens included
    cu_tokens: torch.Tensor | None
    max_tokens: int
    max_len: int | None        # None: not known
    last: torch.Tensor         # int64 [sequences]: the row of each one's last new token
    positions: torch.Tensor    # int64 [rows]
    longest: int = 0           # tokens of the longest sequence (0: not known, not checked)
    pool: int = 0              # blocks that a cache must have: the highest one named, and 1 (0: as above)
    shared: int = 0            # blocks that all the sequences begin with
    slots: torch.Tensor | None = None   # int64 [rows]: block * 64 + place of each new token (of DeviceSequences; -1 behind the last)
    padded: bool = True        # with cu_tokens: there may be rows that no sequence has, behind the last one's
    status: torch.Tensor | None = None  # int32 [1]: of ops.kv8_resize (of DeviceSequences)


class Sequences:
    """Which blocks of a pool each sequence has: host bookkeeping, shared by the caches of all layers."""

    def __init__(self, num_blocks: int, device="cuda"):
        self.device = torch.device(device)
        self._free = list(range(num_blocks - 1, -1, -1))
        self._blocks: dict[object, list[int]] = {}
        self._lens: dict[object, int] = {}

    @property
    def free_blocks(self) -> int:
        return len(self._free)

    def length(self, name) -> int:
        return self._lens[name]

    def blocks(self, name) -> list[int]:
        return list(self._blocks[name])

    def drop(self, name) -> None:
        """Give a sequence's blocks back."""
        self._free.extend(reversed(self._blocks.pop(name)))
        del self._lens[name]

    def extend(self, new: dict) -> Step:
        """Make room for new[name] (at least one) more tokens of each sequence (unknown names begin one) and describe the pass that
        appends them. Raises MemoryError, and changes nothing, where the pool has too few blocks left."""
        if not new or any(n < 1 for n in new.values()):
            raise ValueError("each sequence of a pass needs at least one new token")
        lens = {s: self._lens.get(s, 0) + n for s, n in new.items()}
        wanted = {s: -(-lens[s] // BLOCK) - len(self._blocks.get(s, ())) for s in new}
        if sum(wanted.values()) > len(self._free):
            raise MemoryError(f"{sum(wanted.values())} more blocks are needed, {len(self._free)} are free")
        for s, n in wanted.items():
            self._blocks.setdefault(s, []).extend(self._free.pop() for _ in range(n))
            self._lens[s] = lens[s]
        width = max(len(self._blocks[s]) for s in new)
        counts = list(new.values())
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        i32 = dict(dtype=torch.int32, device=self.device)
        return Step(block_table=torch.tensor([self._blocks[s] + [0] * (width - len(self._blocks[s])) for s in new], **i32),
                    seq_lens=torch.tensor([lens[s] for s in new], **i32),
                    cu_tokens=None if len(set(counts)) == 1 else torch.tensor(starts, **i32), max_tokens=max(counts), max_len=max(lens.values()),
                    last=torch.tensor(starts[1:], device=self.device) - 1,
                    positions=torch.cat([torch.arange(lens[s] - n, lens[s]) for s, n in new.items()]).to(self.device),
                    longest=max(lens.values()), pool=1 + max(max(self._blocks[s]) for s in new), padded=False)


class DeviceSequences:
    """Which blocks of a pool a fixed batch of sequences has, kept on the device (ops.kv8_resize): no pass asks the host. `capacity` is the most tokens of
    a sequence, rounded up to whole blocks: sequences may have as many as the attribute then says, and rotation tables reach as far. The first `shared` blocks of the pool are every sequence's first ones: their tokens are appended once, by the pass
    that prompt() describes, and a sequence without tokens of its own has those. Every change of the books names its success in a tensor on the device, `status` of the latest one
    (int32 [1], ops.kv8_resize's: 0, or the books are as they were)."""

    def __init__(self, num_blocks: int, batch: int, capacity: int, shared: int = 0, device="cuda"):
        width = -(-capacity // BLOCK)
        if batch < 1 or capacity < 1 or not 0 <= shared <= min(num_blocks, width):
            raise ValueError(f"needs a sequence, a token for it, and no more shared blocks than the pool and a sequence have, got {batch}, {capacity} and {shared}")
        self.num_blocks, self.batch, self.shared, self.capacity = num_blocks, batch, shared, width * BLOCK
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.zeros((batch, width), **i32)
        self.block_table[:, :shared] = torch.arange(shared, **i32)
        self.seq_lens = torch.full((batch,), shared * BLOCK, **i32)
        self.free_blocks = torch.zeros(num_blocks, **i32)  # the last free one is the next to be taken
        self.free_blocks[:num_blocks - shared] = torch.arange(num_blocks - 1, shared - 1, -1, **i32)
        self.free_count = torch.full((1,), num_blocks - shared, **i32)
        self.status = torch.zeros(1, **i32)

    def _books(self):
        return self.block_table, self.seq_lens, self.free_blocks, self.free_count

    def prompt(self) -> Step:
        """The pass that appends the shared blocks' tokens, as those of one sequence."""
        if not self.shared:
            raise ValueError("the sequences share no blocks")
        n, dev = self.shared * BLOCK, self.block_table.device
        return Step(block_table=self.block_table[:1], seq_lens=torch.full((1,), n, dtype=torch.int32, device=dev), cu_tokens=None, max_tokens=n, max_len=n,
                    last=torch.full((1,), n - 1, device=dev), positions=torch.arange(n, device=dev), longest=n, pool=self.num_blocks)

    def extend(self, new, rows: int, max_tokens: int | None = None, max_len: int | None = None) -> Step:
        """Make room for new[i] more tokens of sequence i (int32 [batch] on the device, none negative) and describe the pass that appends them. `rows`
        is the number of rows that the pass has, as many as there are new tokens or more: those behind them belong to no sequence, but a layer that finds one scale for all rows
        of its input (QLinearA8W8 as constructed) sees what the caller puts there. max_tokens and max_len bound a sequence's
        new tokens and its length (defaults: rows, the capacity); attention over shared blocks is about as fast with the defaults, without them a max_tokens close to what the
        sequences have is faster, and verify() gives as many columns. Where step.status is not 0 nothing has changed and the pass has no tokens. The
        step names the tables themselves: it describes the pass until they are changed again."""
        cu, positions, slots, self.status = ops.kv8_resize(*self._books(), new, rows=rows, shared=self.shared)
        return Step(block_table=self.block_table, seq_lens=self.seq_lens, cu_tokens=cu, max_tokens=rows if max_tokens is None else max_tokens,
                    max_len=max_len, last=(cu[1:].long() - 1).clamp_min(0), positions=positions, longest=self.capacity,
                    pool=self.num_blocks, shared=self.shared, slots=slots, status=self.status)

    def give_back(self, tokens):
        """Take the last tokens[i] tokens of sequence i away (int32 [batch] on the device, none negative; more than there are: all of its own). Blocks that
        they alone had are free again. Returns the status."""
        self.status = ops.kv8_resize(*self._books(), -torch.minimum(tokens, self.seq_lens - self.shared * BLOCK), shared=self.shared)[3]
        return self.status

    def verify(self, logits, tokens, step: Step, draft_logits=None, accept_draws=None, sample_draws=None, temperature=1.0):
        """ops.verify_drafts of a step's rows, each sequence's first one a known token and the others drafts; refused drafts leave their sequences. Returns
        (accepted drafts, the token behind them and -1, int64 [batch, max_tokens]; how many were accepted, int32 [batch]); where self.status is not 0 then, the books were none (changed by
        others, say) and the refused drafts are still in them. What they leave in the cache is the scale of the block that they ended in, and codes rounded to it, where they
        were larger than what the block held: accepted tokens are rounded as if they had come behind the refused ones, so a generation with drafts is not, bit for bit, that without."""
        change = torch.empty_like(self.seq_lens)
        out, accepted = ops.verify_drafts(logits, tokens, step.cu_tokens, draft_logits=draft_logits, accept_draws=accept_draws, sample_draws=sample_draws,
                                          temperature=temperature, max_tokens=step.max_tokens, change=change)
        self.status = ops.kv8_resize(*self._books(), change, shared=self.shared)[3]
        return out, accepted


def rotation_tables(positions: int, head_dim: int, base: float = 10000.0, device="cuda"):
    """(cos, sin), float32 [positions, head_dim / 2], of the rotation by halves: angle p * base^(-2 i / head_dim)."""
    rate = base ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return angle.cos().float().to(device), angle.sin().float().to(device)


class CachedAttention(nn.Module):
    """o_proj(attention(rotate(q_proj(x)), cache)) of a decoder layer: keys and values of x's rows are appended to the cache on the way.
    The projections are this package's quantised layers (or any with their shapes); cos and sin None: nothing is rotated.
    For inference: nothing is recorded for a backward."""

    def __init__(self, q_proj, k_proj, v_proj, o_proj, heads: int, kv_heads: int, head_dim: int, cos=None, sin=None, window: int = 0):
        super().__init__()
        if heads % kv_heads:
            raise ValueError(f"heads must be a multiple of kv_heads, got {heads} and {kv_heads}")
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = q_proj, k_proj, v_proj, o_proj
        self.heads, self.kv_heads, self.head_dim, self.window = heads, kv_heads, head_dim, window
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)

    def _apply(self, fn, recurse=True):
        """The rotation tables go where the module goes and stay float32, which the kernels take, when it is cast."""
        tables = {"cos": self.cos, "sin": self.sin}
        super()._apply(fn, recurse)
        for name, t in tables.items():
            if t is not None and not t.is_meta:
                self._buffers[name] = t.to(self._buffers[name].device)
        return self

    @torch.no_grad()
    def forward(self, x, cache: KVCache8, step: Step):
        rows = x.shape[0]
        q = self.q_proj(x).view(rows, self.heads, self.head_dim)
        k = self.k_proj(x).view(rows, self.kv_heads, self.head_dim)
        v = self.v_proj(x).view(rows, self.kv_heads, self.head_dim)
        turned = cache.append(k, v, step, q=q if self.cos is not None else None, cos=self.cos, sin=self.sin)
        out = cache.attend(q if turned is None else turned, step, window=self.window)
        return self.o_proj(out.view(rows, self.heads * self.head_dim))
