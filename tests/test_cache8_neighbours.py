"""What a write to the 8-bit pool leaves alone: other slots, other layers, a fork's parent; and the size of a page's file."""
import numpy as np
import pytest

from tests.test_cache8 import _engine, _fill, _pool, _rows_of, _shuffle, _special_rows, _torch_dtype

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page,rot", [(64, 16, 0), (128, 48, 0), (256, 16, 64), (64, 32, 16)])
@pytest.mark.parametrize("how", ["chunk", "batch", "inject"])
def test_only_the_tokens_slots_change(drkv_lib, d, page, rot, how):
    """Bytes and exponents of every slot that no token was written to are those of before."""
    import torch
    start, n, h = 5, 2 * page + 3, 3
    eng = _engine(hq=6, hkv=h, d=d, page=page, dtype="bf16", layers=2, pages=12, seqs=2, per_seq=5, rot=rot)
    _shuffle(eng, d)
    for s in range(2):
        eng.seq_create()
        assert eng.ensure_blocks_for_range(s, 0, 4 * page)
        eng.set_seq_len(s, 4 * page)
    eng.sync_block_table()
    noise = torch.randint(-128, 128, eng.pool_tensor().view(torch.int8).shape, device="cuda", dtype=torch.int8)
    eng.pool_tensor().view(torch.int8).copy_(noise)
    torch.cuda.synchronize()
    before = _pool(eng)
    k, v = (torch.nan_to_num(_special_rows(n, h, d, _torch_dtype("bf16"), i), posinf=2.0, neginf=-2.0) for i in (1, 2))
    if how == "chunk":
        eng.append_rope_chunk(1, 1, start, n, k, v)
    elif how == "batch":
        pos = torch.arange(start, start + n, device="cuda", dtype=torch.int32)
        eng.append_rope(1, n, torch.ones_like(pos), pos, k, v)
    else:
        eng.inject(1, start, n, torch.stack([torch.stack([k, v])] * 2).contiguous())
    torch.cuda.synchronize()
    after = _pool(eng)
    pg, slot = _rows_of(eng, 1, 4 * page, page)
    written = np.zeros(before[1].shape, dtype=bool)                  # [layer, page, plane, head, slot]
    layers = (0, 1) if how == "inject" else (1,)
    for layer in layers:
        written[layer, pg[start:start + n], :, :, slot[start:start + n]] = True
    assert written.sum() == len(layers) * n * 2 * h
    assert np.array_equal(after[0][~written], before[0][~written]) and np.array_equal(after[1][~written], before[1][~written])
    # the noise was no token: what was written differs from it in every row
    assert (after[0][written] != before[0][written]).any(-1).all()
    eng.check_kernels()
    eng.close()


@pytest.mark.parametrize("pool_dtype", ["bf16", "f16"])
def test_parent_of_a_fork(drkv_lib, tmp_path, pool_dtype):
    """A fork writes behind the common tokens and over the last of them: the parent reads what it read before."""
    import torch
    t = _torch_dtype(pool_dtype)
    eng = _engine(hq=4, hkv=2, d=64, page=16, dtype=pool_dtype, layers=2, pages=12, seqs=3, per_seq=16, stream_evict=True)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 70)
    eng.set_seq_len(0, 70)
    eng.sync_block_table()
    for layer in (0, 1):
        _fill(eng, [70], pool_dtype, 8 + layer, layer=layer)
    flat, child_flat = torch.empty(2, 2, 70, 2, 64, device="cuda", dtype=t), torch.empty(2, 2, 71, 2, 64, device="cuda", dtype=t)
    eng.extract(0, 0, 70, flat)
    child = eng.seq_fork(0)
    assert eng.ensure_blocks_for_range(child, 68, 3)
    eng.sync_block_table()
    assert eng.table(child)[4] != eng.table(0)[4] and list(eng.table(child)[:4]) == list(eng.table(0)[:4])
    new = torch.ones(3, 2, 64, device="cuda", dtype=t)
    for layer in (0, 1):
        eng.append_rope_chunk(layer, child, 68, 3, new, new)
    parent = torch.empty_like(flat)
    eng.extract(0, 0, 70, parent)
    eng.extract(child, 0, 71, child_flat)
    torch.cuda.synchronize()
    assert torch.equal(parent, flat)
    assert torch.equal(child_flat[:, :, :68], flat[:, :, :68]) and (child_flat[:, :, 68:] == 1).all()
    assert not (flat[:, :, 68:] == 1).all(-1).any()                  # a row of ones is no token of the parent
    # a page's file: every layer's K and V rows of 64 + 1 bytes, known as soon as there is a tier
    assert eng.tier_stats()["page_file_bytes"] == 0
    eng.tier_enable(str(tmp_path))
    assert eng.tier_stats()["page_file_bytes"] == 2 * 2 * 2 * 16 * 65
    eng.seq_release(child, discard=True)
    assert eng.evict_blocks(0, 3) == 3
    import os
    sizes = [os.path.getsize(os.path.join(base, f)) for base, _, files in os.walk(tmp_path) for f in files]
    assert sizes == [2 * 2 * 2 * 16 * 65] * 3
    eng.close()
