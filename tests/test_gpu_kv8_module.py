"""The cache's bookkeeping and a decoder layer's attention over it: prompts and single tokens of several sequences against plain
attention in 64 bits over the values that the cache gives back, and the example's decoder against itself in other batches."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Linear(torch.nn.Module):
    def __init__(self, n, k, seed):
        super().__init__()
        self.w = (torch.randn((n, k), generator=torch.Generator().manual_seed(seed)) * k ** -0.5).to(BF16).cuda()

    def forward(self, x):
        return x @ self.w.t()


def test_layer_over_prompts_and_single_tokens(hip_lib):
    from latentq_llm_amd.kv_cache import CachedAttention, KVCache8, Sequences, rotation_tables
    heads, kv, dim, hidden, seed = 8, 2, 64, 256, 1
    cos, sin = rotation_tables(300, dim)
    layer = CachedAttention(Linear(heads * dim, hidden, 1), Linear(kv * dim, hidden, 2), Linear(kv * dim, hidden, 3), Linear(hidden, heads * dim, 4), heads, kv,
                            dim, cos, sin)
    cache, seqs = KVCache8(12, kv, dim), Sequences(12)
    for new in ({"a": 100, "b": 3}, {"a": 1, "b": 1}, {"b": 70, "c": 5}, {"c": 1, "a": 1, "b": 1}):
        step = seqs.extend(new)
        x = torch.randn((sum(new.values()), hidden), generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()
        seed += 1
        got = layer(x, cache, step)
        # what the layer computes, from the cache's own values
        host = ref.Cache(12, kv, dim)
        host.codes = list(ref.from_layout(cache.k_codes, cache.v_codes))
        host.scale = [cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()]
        q = layer.q_proj(x).view(-1, heads, dim)
        turned = torch.from_numpy(ref.rotated(q.float().cpu().numpy(), cos.cpu().numpy()[step.positions.cpu()], sin.cpu().numpy()[step.positions.cpu()])).to(BF16)
        out, _, bound = ref.attention(host, turned, step.block_table.cpu().numpy(), step.seq_lens.tolist(), list(new.values()))
        want = layer.o_proj(torch.from_numpy(out).to(BF16).cuda().view(-1, heads * dim))
        # an output of o_proj: the bounds of its inputs (and half an ulp of each) through |w|, and its own rounding
        slack = torch.from_numpy(bound + np.abs(out) * 2.0 ** -8).float().cuda().view(-1, heads * dim) @ layer.o_proj.w.float().abs().t()
        assert ((got.float() - want.float()).abs() <= slack + 2.0 ** -7 * want.float().abs()).all()
        # values are the projections, rounded to 8 bits: the last new token of each sequence
        v = layer.v_proj(x).view(-1, kv, dim)
        for i, name in enumerate(new):
            at = seqs.length(name) - 1
            block = seqs.blocks(name)[at // 64]
            value = cache.read(torch.tensor([block], dtype=torch.int32, device="cuda"), torch.float32)[1][0, at % 64]
            assert ((value - v[step.last[i]].float()).abs() <= 0.5001 * cache.v_scale[block][:, None]).all()


def test_example(hip_lib):
    """A prompt alone, with others, and in two pieces: the same tokens (single sequences and batches go through the same kernels here)."""
    from latentq_llm_amd.kv_cache import KVCache8, Sequences
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "generate_kv8.py")
    spec = importlib.util.spec_from_file_location("generate_kv8", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    model = m.Decoder(2, 512, 1024, 8, 2, 1000, 400).eval()
    caches, seqs = [KVCache8(30, 2, 64) for _ in range(2)], Sequences(30)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=gen).tolist() for n in (200, 33, 129)]
    out, _, _ = m.generate(model, caches, seqs, prompts, [6, 3, 5])
    assert [len(o) for o in out] == [6, 3, 5] and seqs.free_blocks == 30
    again, _, _ = m.generate(model, caches, seqs, prompts, [6, 3, 5])
    assert again == out
    # logits of a prompt in one piece and in two: the second piece reads the first from the cache
    whole = model(torch.tensor(prompts[0]).cuda(), caches, seqs.extend({"w": 200}))
    model(torch.tensor(prompts[0][:128]).cuda(), caches, seqs.extend({"p": 128}))
    parts = model(torch.tensor(prompts[0][128:]).cuda(), caches, seqs.extend({"p": 72}))
    # blocks are whole in both, so the caches hold the same codes but for what other kernels of the products round otherwise
    assert float((whole - parts).float().norm() / whole.float().norm()) < 0.05
