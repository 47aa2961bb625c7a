"""Which blocks of the pool the sequences of the 8-bit cache have (host bookkeeping)."""
import pytest


def test_bookkeeping():
    from latentq_llm_amd.kv_cache import Sequences
    s = Sequences(4, device="cpu")
    step = s.extend({"x": 65, "y": 1})
    assert s.free_blocks == 1 and step.block_table.shape == (2, 2) and step.seq_lens.tolist() == [65, 1] and step.cu_tokens.tolist() == [0, 65, 66]
    assert step.max_tokens == 65 and step.max_len == 65 and step.last.tolist() == [64, 65] and step.positions.tolist() == list(range(65)) + [0]
    with pytest.raises(MemoryError, match="2 more blocks"):
        s.extend({"x": 64, "y": 64})
    assert s.length("x") == 65 and s.free_blocks == 1
    step = s.extend({"x": 63, "y": 63})
    assert s.free_blocks == 1 and step.cu_tokens is None and step.max_len == 128
    with pytest.raises(ValueError, match="at least one"):
        s.extend({"x": 0})
    held = s.blocks("x")
    s.drop("x")
    assert s.free_blocks == 3 and s.extend({"z": 128}) and sorted(s.blocks("z")) == sorted(held)
