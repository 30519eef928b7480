"""Prefill over the 8-bit pool is the prefill over a 16-bit pool that holds the values its rows stand for."""
import math

import pytest

from tests.test_cache8 import _engine, _fill, _shuffle, _torch_dtype

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d,grp,page,n,m", [("bf16", 128, 4, 16, 700, 300), ("f16", 128, 4, 16, 700, 129), ("f16", 64, 8, 48, 300, 300),
                                                  ("bf16", 256, 6, 32, 257, 1)])
def test_same_bits_as_a_16_bit_pool(drkv_lib, dtype, d, grp, page, n, m):
    import torch
    from deusridet_b200 import PagedKVEngine
    t, hkv, per = _torch_dtype(dtype), 2, -(-n // page)
    eight = _engine(hq=grp * hkv, hkv=hkv, d=d, page=page, dtype=dtype, pages=per + 4, seqs=1, per_seq=per)
    sixteen = PagedKVEngine(num_layers=1, num_q_heads=grp * hkv, num_kv_heads=hkv, head_dim=d, page_size=page, dtype=dtype, rotary_dim=0,
                            max_pages=per + 4, max_seqs=1, max_pages_per_seq=per, device=0)
    for e in (eight, sixteen):
        _shuffle(e, 3)
        e.seq_create()
        assert e.ensure_blocks_for_range(0, 0, n)
        e.set_seq_len(0, n)
        e.sync_block_table()
    _fill(eight, [n], dtype, 11, spread=2)
    flat = torch.empty(1, 2, n, hkv, d, device="cuda", dtype=t)
    eight.extract(0, 0, n, flat)
    sixteen.inject(0, 0, n, flat)
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(m, grp * hkv, d, generator=g, device="cuda").to(t)
    outs = []
    for e in (eight, sixteen):
        out = torch.zeros_like(q)
        e.attend_prefill_chunk(0, 0, n - m, m, q, out, 1.0 / math.sqrt(d))
        torch.cuda.synchronize()
        e.check_kernels()
        outs.append(out)
        e.close()
    assert outs[0].any() and torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))
