"""What Rope refuses besides sizes: tensors that require a gradient, devices that are not there."""
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


@pytest.mark.gpu
def test_a_refused_device_leaves_no_error_behind(drkv_lib):
    """Launches that are checked by the last error (the merge of partials) do not report an earlier call's."""
    import torch
    from deusridet_b200 import DrkvError, PagedKVEngine, Rope, capi
    eng = PagedKVEngine(num_layers=1, num_q_heads=4, num_kv_heads=1, head_dim=64, page_size=16, rotary_dim=0, max_pages=8, max_seqs=1, device=0)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 20)
    eng.set_seq_len(0, 20)
    eng.sync_block_table()
    x = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    part = torch.zeros(eng.partial_floats(), device="cuda")
    eng.attend_partial(0, 0, 0, 20, x, part, 0.1)
    with pytest.raises(DrkvError) as err:
        Rope(head_dim=64, device=torch.cuda.device_count())
    assert err.value.code == capi.ERR_NO_DEVICE
    eng.combine_partials(1, part, torch.empty_like(x))
    torch.cuda.synchronize()
    eng.check_kernels()
    eng.close()
