"""The rotation tables of a decoder layer's attention through casts and moves of the module."""
import torch

from latentq_llm_amd.kv_cache import CachedAttention, rotation_tables


def test_a_cast_leaves_the_tables_as_they_are():
    cos, sin = rotation_tables(20, 64, device="cpu")
    model = torch.nn.Sequential(CachedAttention(*(torch.nn.Linear(64, 64) for _ in range(4)), 1, 1, 64, cos, sin))
    for cast in (lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.float16), lambda m: m.bfloat16()):
        layer = cast(model)[0]
        assert layer.cos.dtype == layer.sin.dtype == torch.float32 and torch.equal(layer.cos, cos) and torch.equal(layer.sin, sin)
    assert layer.q_proj.weight.dtype == torch.bfloat16 and set(dict(layer.named_buffers())) == {"cos", "sin"}
    assert model.to("meta")[0].cos.is_meta and model[0].cos.dtype == torch.float32
    assert model.to_empty(device="cpu")[0].cos.device.type == "cpu"


def test_without_tables():
    layer = CachedAttention(*(torch.nn.Linear(64, 64) for _ in range(4)), 1, 1, 64).to(torch.bfloat16)
    assert layer.cos is None and layer.sin is None
