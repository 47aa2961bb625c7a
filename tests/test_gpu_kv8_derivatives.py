"""The 8-bit cache's operators have no derivative: a gradient or a tangent that would be lost is refused, whichever operand it belongs to."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from tests import kv8_ref as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def operands():
    names = ("k_codes", "v_codes", "k_scale", "v_scale")
    cos, sin = (torch.from_numpy(x).cuda() for x in ref.tables(10, 64))
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    k = q[:, :2].contiguous()
    return dict(zip(names, ref.Cache(3, 2, 64, seed=1).tensors())), dict(block_table=i32([[1]]), seq_lens=i32([3])), dict(k=k, v=k.clone(), q=q, cos=cos, sin=sin)


def calls(cache, where, new):
    from latentq_llm_amd import ops
    return {"append": (lambda o: ops.kv8_append(o["k"], o["v"], **{n: o[n] for n in cache}, **where, q=o["q"], cos=o["cos"], sin=o["sin"]), (*new, "k_scale", "v_scale")),
            "attention": (lambda o: ops.kv8_attention(o["q"], **{n: o[n] for n in cache}, **where), ("q", "k_scale", "v_scale")),
            "read": (lambda o: ops.kv8_read(**{n: o[n] for n in cache}, blocks=i32([1])), ("k_scale", "v_scale"))}


@pytest.mark.parametrize("name", ["append", "attention", "read"])
def test_gradients(hip_lib, name):
    cache, where, new = operands()
    call, floats = calls(cache, where, new)[name]
    for n in floats:
        with pytest.raises(RuntimeError, match=f"no backward, and {n} requires"):
            call({**cache, **new, n: {**cache, **new}[n].clone().requires_grad_()})
        with torch.no_grad():
            call({**cache, **new, n: {**cache, **new}[n].clone().requires_grad_()})
    call({**cache, **new})


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["append", "attention", "read"])
def test_tangents(hip_lib, name, grad):
    cache, where, new = operands()
    call, floats = calls(cache, where, new)[name]
    with torch.set_grad_enabled(grad), fwAD.dual_level():
        for n in floats:
            t = {**cache, **new}[n]
            with pytest.raises(RuntimeError, match=f"no derivative, and {n} has a tangent"):
                call({**cache, **new, n: fwAD.make_dual(t.clone(), torch.ones_like(t))})
        before = [t.clone() for t in cache.values()]
        inside = call({**cache, **new})  # operands without one: as outside
    after = [t.clone() for t in cache.values()]
    for t, b in zip(cache.values(), before):
        t.copy_(b)
    outside = call({**cache, **new})
    for a, b in zip(inside if isinstance(inside, tuple) else (inside,), outside if isinstance(outside, tuple) else (outside,)):
        assert torch.equal(a, b)
    assert all(torch.equal(a, t) for a, t in zip(after, cache.values()))
