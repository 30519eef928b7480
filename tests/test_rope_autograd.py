"""Rope.apply and autograd: nothing that requires a gradient goes through it unnoticed."""
import pytest


def test_refuses_what_requires_a_gradient(drkv_lib):
    import torch
    from deusridet_b200 import DrkvError, Rope
    rope = Rope(head_dim=64, dtype="bf16", device=-1)
    pos = torch.arange(4, dtype=torch.int32)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    leaf = x.clone().requires_grad_()
    for args in (dict(q=leaf), dict(k=leaf), dict(q=x, k=leaf * 2), dict(q=x, out_q=leaf), dict(q=leaf, out_q=leaf), dict(k=leaf, inverse=True)):
        with pytest.raises(ValueError, match="autograd"):
            rope.apply(pos, **args)
    with torch.no_grad(), pytest.raises(DrkvError):                  # past the checks: this rotation has no device
        rope.apply(pos, leaf, out_q=torch.empty_like(x), stream=0)
    with pytest.raises(DrkvError):
        rope.apply(pos, leaf.detach(), out_q=torch.empty_like(x), stream=0)


@pytest.mark.gpu
def test_without_gradients_and_by_the_transpose(drkv_lib):
    import torch
    from deusridet_b200 import Rope
    rope = Rope(head_dim=64, rotary_dim=48, dtype="f16", device=0)
    pos = torch.tensor([3, 70000, 5], device="cuda", dtype=torch.int32)
    x = torch.randn(3, 2, 64, device="cuda", dtype=torch.float16).requires_grad_()
    with torch.no_grad():
        y, _ = rope.apply(pos, x)
        back, _ = rope.apply(pos, y, inverse=True)
    assert not y.requires_grad
    with torch.inference_mode():
        again, _ = rope.apply(pos, x)
    assert torch.equal(again, y)
    # the transpose undoes a rotation; two roundings to fp16 of values no larger than |x0| + |x1|
    size = x.detach().abs().float().amax(-1, keepdim=True) * 2
    assert ((back.float() - x.detach().float()).abs() <= 2 * 2.0 ** -11 * size * 1.5).all()
