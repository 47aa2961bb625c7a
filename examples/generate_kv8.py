"""Generation with int4 layers and a paged 8-bit cache of keys and values: prompts of different lengths go in together, then every
sequence gives one token a pass; one that is done gives its blocks back.

    python examples/generate_kv8.py [--layers 4] [--hidden 4096] [--inter 11008] [--heads 32] [--kv-heads 32] [--new 32]

Weights are random (the sizes of a 7B decoder by default), so the tokens mean nothing; it shows the calls and prints their speed.
"""
import argparse
import os
import sys
import time

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from latentq_llm_amd.fused_mlp import QuantLlamaMLP  # noqa: E402
from latentq_llm_amd.kv_cache import CachedAttention, KVCache8, Sequences, rotation_tables  # noqa: E402
from latentq_llm_amd.quant import QLinearA16W4  # noqa: E402

BF16 = torch.bfloat16


def linear4(out_features, in_features, gen):
    """An int4 layer whose weights have a standard deviation of about 1 / sqrt(in_features)."""
    layer = QLinearA16W4(in_features, out_features, bias=False)
    groups = out_features * in_features // 128
    layer.scales.data = torch.full((groups, 1), in_features ** -0.5 / 4.6, dtype=BF16, device="cuda")
    layer.zeros.data = torch.full((groups, 1), 7.5, dtype=BF16, device="cuda")
    codes = torch.randint(-128, 128, (out_features * in_features // 2,), generator=gen, device="cuda", dtype=torch.int8)
    layer.weight.set_value(codes, [layer.scales, layer.zeros, layer.wshape])
    return layer.eval()


class Norm(nn.Module):
    def __init__(self, hidden):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden, dtype=BF16, device="cuda"), requires_grad=False)

    def forward(self, x):
        return torch.nn.functional.rms_norm(x, (x.shape[-1],), self.weight, 1e-5)


class Decoder(nn.Module):
    def __init__(self, layers, hidden, inter, heads, kv_heads, vocab, positions, seed=0):
        super().__init__()
        gen = torch.Generator(device="cuda").manual_seed(seed)
        dim = hidden // heads
        cos, sin = rotation_tables(positions, dim)
        self.embed = (torch.randn((vocab, hidden), generator=gen, device="cuda")).to(BF16)
        self.head = (torch.randn((vocab, hidden), generator=gen, device="cuda") * hidden ** -0.5).to(BF16)
        self.norm = Norm(hidden)
        self.layers = nn.ModuleList()
        for _ in range(layers):
            attention = CachedAttention(linear4(hidden, hidden, gen), linear4(kv_heads * dim, hidden, gen), linear4(kv_heads * dim, hidden, gen),
                                        linear4(hidden, hidden, gen), heads, kv_heads, dim, cos, sin)
            mlp = QuantLlamaMLP(linear4(inter, hidden, gen), linear4(hidden, inter, gen), linear4(inter, hidden, gen))
            self.layers.append(nn.ModuleList([Norm(hidden), attention, Norm(hidden), mlp]))

    @torch.no_grad()
    def forward(self, tokens, caches, step):
        """Logits of each sequence's last new token."""
        x = self.embed[tokens]
        for (norm1, attention, norm2, mlp), cache in zip(self.layers, caches):
            x = x + attention(norm1(x), cache, step)
            x = x + mlp(norm2(x))
        return self.norm(x[step.last]) @ self.head.t()


def generate(model, caches, sequences, prompts, new):
    """Greedy continuation of each prompt (lists of tokens) by new[i] tokens; returns (tokens, seconds of the prompts, of the rest)."""
    out = [[] for _ in prompts]
    torch.cuda.synchronize()
    begin = time.perf_counter()
    step = sequences.extend({i: len(p) for i, p in enumerate(prompts)})
    token = model(torch.cat([torch.tensor(p) for p in prompts]).cuda(), caches, step).argmax(-1)
    torch.cuda.synchronize()
    middle = time.perf_counter()
    alive = list(range(len(prompts)))
    while alive:
        for i, t in zip(alive, token.tolist()):
            out[i].append(t)
        keep = [n for n, i in enumerate(alive) if len(out[i]) < new[i]]
        for i in alive:
            if len(out[i]) >= new[i]:
                sequences.drop(i)
        token, alive = token[keep], [alive[n] for n in keep]
        if alive:
            token = model(token, caches, sequences.extend({i: 1 for i in alive})).argmax(-1)
    torch.cuda.synchronize()
    return out, middle - begin, time.perf_counter() - middle


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 4), ("hidden", 4096), ("inter", 11008), ("heads", 32), ("kv-heads", 32), ("vocab", 32000), ("new", 32)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--prompts", type=int, nargs="+", default=[45, 512, 1019, 7], help="their lengths")
    a = ap.parse_args()
    positions = max(a.prompts) + a.new
    blocks = sum(-(-(n + a.new) // 64) for n in a.prompts)
    model = Decoder(a.layers, a.hidden, a.inter, a.heads, a.kv_heads, a.vocab, positions).eval()
    caches = [KVCache8(blocks, a.kv_heads, a.hidden // a.heads) for _ in range(a.layers)]
    sequences = Sequences(blocks)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, a.vocab, (n,), generator=gen).tolist() for n in a.prompts]
    new = [a.new] * len(prompts)
    generate(model, caches, sequences, prompts, new)  # first calls load code
    out, first, rest = generate(model, caches, sequences, prompts, new)
    print(f"{sum(a.prompts)} prompt tokens in {first * 1e3:.2f} ms, then {a.new - 1} passes of {len(prompts)} tokens, {rest / max(1, a.new - 1) * 1e3:.3f} ms each "
          f"({a.layers} layers); cache {sum(t.numel() * t.element_size() for c in caches for t in c.tensors()) >> 20} MiB")
    for p, o in zip(a.prompts, out):
        print(f"prompt of {p}: {o[:8]} ...")


if __name__ == "__main__":
    main()
