"""The capacity of DeviceSequences is whole blocks: what its sequences may grow to, so what rotation tables have to reach."""
import pytest
import torch

from latentq_llm_amd.kv_cache import CachedAttention, DeviceSequences, KVCache8, Step, rotation_tables


@pytest.mark.parametrize("asked, has", [(1, 64), (64, 64), (65, 128), (1000, 1024), (1024, 1024)])
def test_capacity(asked, has):
    seqs = DeviceSequences(40, 2, asked, device="cpu")
    assert seqs.capacity == has == 64 * seqs.block_table.shape[1]


def test_rotation_tables_for_it():
    """A step names the capacity as the longest that a sequence may be: tables of as many positions are taken, shorter ones refused before anything is launched."""
    seqs, cache, x = DeviceSequences(40, 2, 1000, device="cpu"), KVCache8(40, 1, 64, device="cpu"), torch.zeros((2, 64), dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    step = Step(seqs.block_table, seqs.seq_lens, torch.zeros(3, **i32), 2, seqs.capacity, torch.zeros(2, dtype=torch.long), torch.zeros(2, dtype=torch.long), longest=seqs.capacity, pool=40)

    def attention(positions):
        cos, sin = rotation_tables(positions, 64, device="cpu")
        return CachedAttention(*(torch.nn.Linear(64, 64, bias=False, dtype=torch.bfloat16) for _ in range(4)), 1, 1, 64, cos, sin)

    with pytest.raises(ValueError, match="rotation tables have 1000 positions, a sequence 1024 tokens"):
        attention(1000)(x, cache, step)
    with pytest.raises(RuntimeError, match="GPU tensor"):  # as far as the kernels
        attention(seqs.capacity)(x, cache, step)
