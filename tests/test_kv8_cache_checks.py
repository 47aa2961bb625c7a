"""What the cache of a layer refuses on the host, before anything is launched: passes beyond the rotation tables, and blocks that it has not."""
import pytest
import torch

from latentq_llm_amd.kv_cache import CachedAttention, KVCache8, Sequences, Step, rotation_tables


def layer(positions, window=0):
    torch.manual_seed(0)
    cos, sin = rotation_tables(positions, 64, device="cpu")
    return CachedAttention(*(torch.nn.Linear(64, 64, bias=False, dtype=torch.bfloat16) for _ in range(4)), 1, 1, 64, cos, sin, window)


def test_a_sequence_longer_than_the_rotation_tables():
    attention, cache, seqs = layer(100), KVCache8(8, 1, 64, device="cpu"), Sequences(8, device="cpu")
    x = torch.zeros((101, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="rotation tables have 100 positions, a sequence 101 tokens"):
        attention(x, cache, seqs.extend({"a": 101}))
    step = seqs.extend({"b": 100})
    assert step.longest == 100
    with pytest.raises(RuntimeError, match="GPU tensor"):  # within them: as far as the kernels
        attention(x[:100], cache, step)
    with pytest.raises(ValueError, match="a sequence 101 tokens"):
        attention(x[:1], cache, seqs.extend({"b": 1}))
    assert (cache.k_codes == 128).all() and (cache.v_codes == 128).all()


def test_a_pool_larger_than_the_cache():
    """Sequences may be of more blocks than a cache has, as long as none of those is used."""
    attention, cache, seqs = layer(1000), KVCache8(3, 1, 64, device="cpu"), Sequences(5, device="cpu")
    x = torch.zeros((192, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        attention(x, cache, seqs.extend({"a": 192}))
    step = seqs.extend({"b": 1})
    assert step.pool == 4
    for call in (lambda: attention(x[:1], cache, step), lambda: cache.attend(x[:1].view(1, 1, 64), step), lambda: cache.append(x[:1].view(1, 1, 64), x[:1].view(1, 1, 64), step)):
        with pytest.raises(ValueError, match="block 3 of a cache of 3 blocks"):
            call()


def test_a_step_made_by_hand_is_taken_as_it_is():
    i32 = dict(dtype=torch.int32)
    step = Step(torch.zeros((1, 9), **i32), torch.ones(1, **i32), None, 1, 9 * 64, torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU tensor"):
        layer(10)(torch.zeros((1, 64), dtype=torch.bfloat16), KVCache8(3, 1, 64, device="cpu"), step)
