"""The 8-bit K/V pool: bookkeeping and refusals on the CPU; bytes, attention, prefill, fork, tier and graphs on the GPU."""
import ctypes as C
import math

import numpy as np
import pytest

from tests import cache8_helpers as R


def _engine(hq=8, hkv=2, d=128, page=16, dtype="bf16", layers=1, pages=64, seqs=4, per_seq=0, device=0, rot=0, **kw):
    from deusridet_b200 import PagedKVEngine
    return PagedKVEngine(num_layers=layers, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=page, dtype=dtype, kv_dtype="e4m3",
                         rotary_dim=rot, rope_theta=1e4, max_pages=pages, max_seqs=seqs, max_pages_per_seq=per_seq, device=device, **kw)


# ---- CPU ----------------------------------------------------------------------------------------------------------------
def test_e4m3_oracle_agrees_with_torch():
    import torch
    assert np.array_equal(R.E4M3[:0x7f], torch.arange(0x7f, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
    rng = np.random.default_rng(0)
    y = np.concatenate([rng.standard_normal(5000) * 100, rng.standard_normal(5000) * 0.01, [448.0, 0.0, 2.0 ** -10, 3 * 2.0 ** -10]])
    y = np.clip(y.astype(np.float32), -448, 448)
    assert np.array_equal(R.round_e4m3(y.astype(np.float64)), torch.from_numpy(y).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_geometry_and_offsets_without_device(drkv_lib):
    from deusridet_b200 import capi
    eng = _engine(hq=8, hkv=2, d=64, page=48, layers=3, pages=10, device=-1)
    assert eng.geom.dtype == capi.BF16_KV_E4M3
    plane, exps = 2 * 48 * 64, 2 * 48
    block = 2 * (plane + exps)
    assert eng.total_bytes() == 3 * 10 * block
    assert eng.k_offset(2, 3) == (2 * 10 + 3) * block and eng.v_offset(2, 3) == eng.k_offset(2, 3) + plane
    s = eng.seq_create()
    assert eng.ensure_blocks_for_range(s, 0, 100) and eng.free_count() == 7
    eng.set_seq_len(s, 100)
    f = eng.seq_fork(s)
    assert eng.ensure_blocks_for(f, 100)
    assert eng.stats()["cow_bytes"] == 4 * 64 * 2 * 2 * 3            # 4 slots, K and V, 2 heads, 3 layers, one byte each
    budget = _engine(hq=8, hkv=2, d=64, page=48, layers=3, pages=0, device=-1, budget_bytes=5 * 3 * block + 7)
    assert budget.max_blocks() == 5


def test_refusals_without_device(drkv_lib):
    from deusridet_b200 import DrkvError, PagedKVEngine, capi
    with pytest.raises(ValueError):
        PagedKVEngine(num_layers=1, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16, kv_dtype="int4", max_pages=8, device=-1)
    h = C.c_void_p()
    for bad in (-1, 4):
        g = capi.Geometry(1, 8, 2, 128, 16, bad, 128, 1e4)
        assert drkv_lib.drkv_create(C.byref(g), C.byref(capi.Config(0, 8, 1, 0, -1, 0)), C.byref(h)) == capi.ERR_INVALID
    eng = _engine(device=-1)
    for call in (lambda: eng.scorer_enable(0.9), lambda: eng.set_prefill_on_decode_kernel(True)):
        with pytest.raises(DrkvError) as err:
            call()
        assert err.value.code == capi.ERR_INVALID
    eng.set_prefill_on_decode_kernel(False)
    eng.scorer_disable()
    g = capi.Geometry(1, 8, 2, 128, 16, capi.BF16_KV_E4M3, 0, 1e4)
    assert drkv_lib.drkv_k_cache_write_batch(C.byref(g), 8, 8, 8, 8, 0, 0, 1, 4, None) == capi.ERR_INVALID
    assert drkv_lib.drkv_k_extract_kv(C.byref(g), 8, 8, 8, 0, 1, 4, None) == capi.ERR_INVALID
    assert drkv_lib.drkv_append_rope_chunk(eng.h, 0, 0, 0, 1, 8, 8, None) == capi.ERR_NO_DEVICE
    assert drkv_lib.drkv_select_pages(eng.h, 0, 1, 8, 8, 16, 8, 1, 0, 0, 8, None) == capi.ERR_NO_DEVICE
    assert drkv_lib.drkv_attend_selected(eng.h, 0, 1, 8, 8, 16, 8, 1, 8, 8, 1.0, None) == capi.ERR_NO_DEVICE
    assert drkv_lib.drkv_page_bounds_enable(eng.h, None) == capi.ERR_NO_DEVICE
    assert drkv_lib.drkv_page_bounds(eng.h) is None and drkv_lib.drkv_page_bound_exponents(None) is None


# ---- GPU ----------------------------------------------------------------------------------------------------------------
def _torch_dtype(dtype):
    import torch
    return torch.bfloat16 if dtype == "bf16" else torch.float16


def _half_step(dtype):
    import torch
    return torch.finfo(_torch_dtype(dtype)).eps / 2


def _weight_step(dtype):
    return 2.0 ** -11 if dtype == "bf16" else 2.0 ** -21


def _pool(eng):
    """Pool bytes as [layer, page, ...]: K, V [head, slot, dim] values and exponents [head, slot]."""
    g = eng.geom
    n, h, p, d = eng.max_blocks(), g.num_kv_heads, g.page_size, g.head_dim
    raw = eng.pool_tensor().cpu().numpy().view(np.uint8).reshape(g.num_layers, n, -1)
    plane = h * p * d
    rows = raw[:, :, :2 * plane].reshape(g.num_layers, n, 2, h, p, d)
    return rows, raw[:, :, 2 * plane:].reshape(g.num_layers, n, 2, h, p).astype(int) - 127


def _shuffle(eng, seed):
    rng = np.random.default_rng(seed)
    n = eng.free_count()
    pages = [eng.alloc_block() for _ in range(n)]
    for p in rng.permutation(n):
        eng.free_block(pages[int(p)])


def _rows_of(eng, seq, n, page):
    t = eng.table(seq)
    return np.array([t[i // page] for i in range(n)]), np.arange(n) % page


def _special_rows(n, h, d, t, seed):
    """Rows over many exponents, and rows of the values where a quantiser can go wrong."""
    import torch
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, h, d)) * 2.0 ** rng.integers(-12, 12, (n, h, 1))
    x[0, 0] = 0.0
    x[1 % n, 0, :4] = [1.75, -1.75, 0.0, 1.0]                        # maximum exactly 448 * 2^-8
    x[2 % n, 0] = np.linspace(-1, 1, d)
    x[2 % n, 0, 0] = -1.7578125                                     # a step above 1.75
    x[3 % n, 0] = 1e-6
    x[4 % n, 0, 0], x[4 % n, 0, 1], x[4 % n, 0, 2] = np.inf, -np.inf, np.nan
    x[5 % n, 0, 1:] = 2.0 ** -24
    x[6 % n, 0] = 65504.0
    x[7 % n, 0] = -0.0
    return torch.from_numpy(x).to(t).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d,page,rot", [(64, 16, 0), (128, 48, 0), (256, 16, 64), (128, 16, 128), (64, 32, 16)])
def test_written_bytes_and_flat_copies(drkv_lib, dtype, d, page, rot):
    """Chunk append, batch append and inject leave the formula's bytes; extract returns their values; holes read as zero."""
    import torch
    t = _torch_dtype(dtype)
    n, h = 5 * page + 7, 3
    eng = _engine(hq=6, hkv=h, d=d, page=page, dtype=dtype, layers=2, pages=24, seqs=3, per_seq=8, rot=rot, stream_evict=True)
    _shuffle(eng, d)
    for _ in range(3):
        eng.seq_create()
    for s in range(3):
        assert eng.ensure_blocks_for_range(s, 0, n)
        eng.set_seq_len(s, n)
    eng.sync_block_table()
    k, v = _special_rows(n, h, d, t, 1), _special_rows(n, h, d, t, 2)
    if rot:
        k = torch.nan_to_num(k, nan=1.0, posinf=2.0, neginf=-2.0)   # a rotation mixes pairs: finite keys here
    before = _pool(eng)
    eng.append_rope_chunk(1, 1, 0, n, k, v)
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    eng.append_rope(1, n, torch.full_like(pos, 2), pos, k, v)       # the tokens as a batch, into sequence 2
    torch.cuda.synchronize()
    kd, vd = k.double().cpu().numpy(), v.double().cpu().numpy()
    if rot:                                                          # fp32 angles, products and sums, as append_rope_kernel's
        half = rot // 2
        freq = (1.0 / np.power(np.float32(1e4), (np.float32(2) * np.arange(half, dtype=np.float32)) / np.float32(rot))).astype(np.float32)
        angle = (np.arange(n, dtype=np.float32)[:, None] * freq[None, :]).astype(np.float32).astype(np.float64)[:, None, :]
        c, s = np.cos(angle).astype(np.float32).astype(np.float64), np.sin(angle).astype(np.float32).astype(np.float64)
        x0, x1 = kd[..., :half].copy(), kd[..., half:rot].copy()
        kd[..., :half] = (x0 * c - (x1 * s).astype(np.float32)).astype(np.float32)
        kd[..., half:rot] = (x1 * c + (x0 * s).astype(np.float32)).astype(np.float32)
    rows, exps = _pool(eng)
    for seq in (1, 2):
        pg, slot = _rows_of(eng, seq, n, page)
        for plane, want in ((0, kd), (1, vd)):
            b, e = R.quantise(want)
            got_b, got_e = rows[1, pg, plane, :, slot], exps[1, pg, plane, :, slot]
            if rot and plane == 0:
                # powf on the host may differ by a unit in the last place from numpy's, and with it an angle: what moves is
                # at most one step of a value that lay next to a border
                assert (got_e != e).mean() < 0.01 and (got_b != b).mean() < 0.002
                assert np.nanmax(np.abs(R.E4M3[got_b] - R.E4M3[b])[got_e == e]) <= 32
                continue
            assert np.array_equal(got_e, e)
            nan = np.isnan(R.E4M3[b])
            assert np.array_equal(got_b[~nan], b[~nan]) and np.isnan(R.E4M3[got_b[nan]]).all()
    assert np.array_equal(rows[1][:, 1], rows[1][:, 1]) and np.array_equal(rows[0], before[0][0])     # layer 0 untouched
    # flat copies
    assert eng.evict_blocks(1, 1) == 1
    eng.sync_block_table()
    start, m = 3, n - 5
    flat = torch.empty(2, 2, m, h, d, device="cuda", dtype=t)
    eng.extract(1, start, m, flat)
    torch.cuda.synchronize()
    got = flat.double().cpu().numpy()
    hole = (np.arange(start, start + m) // page) == 0
    assert not got[:, :, hole].any() and not got[0].any()
    pg, slot = _rows_of(eng, 2, n, page)
    for plane in (0, 1):
        val = R.E4M3[rows[1, pg, plane, :, slot]] * 2.0 ** exps[1, pg, plane, :, slot][..., None].astype(float)
        # fp16 has steps of 2^-24 at least, a rotated row's values may be finer: extract rounds to the nearest
        val = np.clip(val, -65504, 65504).astype(np.float16).astype(float) if dtype == "f16" else val
        np.testing.assert_array_equal(got[1, plane][~hole], val[start:start + m][~hole])
    src = torch.cat([_special_rows(m, h, d, t, 10 + i)[None] for i in range(4)]).view(2, 2, m, h, d)
    eng.inject(2, start, m, src)
    torch.cuda.synchronize()
    rows, exps = _pool(eng)
    pg, slot = _rows_of(eng, 2, n, page)
    for layer in (0, 1):
        for plane in (0, 1):
            b, e = R.quantise(src[layer, plane].double().cpu().numpy())
            nan = np.isnan(R.E4M3[b])
            at = slice(start, start + m)
            assert np.array_equal(exps[layer, pg[at], plane, :, slot[at]], e)
            assert np.array_equal(rows[layer, pg[at], plane, :, slot[at]][~nan], b[~nan])
    eng.check_kernels()
    eng.close()


def _fill(eng, lens, dtype, seed, layer=0, spread=3):
    """Appends random K and V of unlike sizes per row; returns their stored values per sequence."""
    import torch
    g, t = eng.geom, _torch_dtype(dtype)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s, n in enumerate(lens):
        kv = []
        for _ in range(2):
            x = torch.randn(max(n, 1), g.num_kv_heads, g.head_dim, generator=gen, device="cuda")
            x = x * 2.0 ** torch.randint(-spread, spread + 1, (max(n, 1), g.num_kv_heads, 1), generator=gen, device="cuda")
            kv.append(x.to(t))
        if n:
            eng.append_rope_chunk(layer, s, 0, n, kv[0], kv[1])
        out.append([R.stored_values(x.double().cpu().numpy()) for x in kv])
    return out


def _check_decode(out, before, q, stored, lens, hkv, scale, dtype, visible=None):
    got, qd = out.double().cpu().numpy(), q.double().cpu().numpy()
    grp = q.shape[1] // hkv
    for b, n in enumerate(lens):
        for h in range(hkv):
            rows = slice(h * grp, (h + 1) * grp)
            see = np.arange(n) if visible is None else visible(b, h, n)
            if len(see) == 0:
                assert np.array_equal(got[b, rows], before.double().cpu().numpy()[b, rows]), (b, h)
                continue
            want, pv, mag = R.attend(qd[b, rows], stored[b][0][see, h], stored[b][1][see, h], scale)
            tol = R.attend_tolerance(want, pv, mag, _half_step(dtype), _weight_step(dtype))
            err = np.abs(got[b, rows] - want)
            assert (err <= tol).all(), (b, h, n, float((err / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("grp,hkv,page", [(1, 3, 16), (4, 2, 48), (6, 2, 16), (8, 1, 32), (12, 1, 16), (16, 2, 64)])
def test_decode_against_64_bits(drkv_lib, dtype, d, grp, hkv, page):
    import torch
    lens = [1, 0, 15, 16, 17, 33, 700, 64, 1500, 2]
    per = -(-1600 // page)
    eng = _engine(hq=grp * hkv, hkv=hkv, d=d, page=page, dtype=dtype, pages=len(lens) * per, seqs=len(lens), per_seq=per, stream_evict=True)
    _shuffle(eng, 5)
    for s, n in enumerate(lens):
        eng.seq_create()
        assert eng.ensure_blocks_for_range(s, 0, max(n, 1))
        eng.set_seq_len(s, n)
    # what an earlier owner may have left behind the last token: NaN bytes, largest exponents
    eng.pool_tensor().fill_(-1)
    eng.sync_block_table()
    stored = _fill(eng, lens, dtype, d + grp)
    gone = -(-700 // page) // 2 if page < 700 else 0
    assert eng.evict_blocks(6, gone) == gone                        # holes at the front of sequence 6
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(len(lens), grp * hkv, d, generator=g, device="cuda").to(_torch_dtype(dtype))
    q[3] *= 100.0
    q[4, 0] = 0.0
    out = torch.full_like(q, 7.0)
    before = out.clone()
    rows = torch.arange(len(lens), device="cuda", dtype=torch.int32)
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    scale = 1.0 / math.sqrt(d)
    eng.attend_decode(0, len(lens), rows, kv_len, max(lens), q, out, scale)
    torch.cuda.synchronize()
    eng.check_kernels()
    holes = lambda b, h, n: np.arange(gone * page if b == 6 else 0, n)
    _check_decode(out, before, q, stored, lens, hkv, scale, dtype, holes)
    # another order of the batch and another split of the work: a sequence alone gives the same values within tolerance
    one = torch.full_like(q[8:9], 7.0)
    eng.attend_decode(0, 1, rows[8:9], kv_len[8:9], 1500, q[8:9].contiguous(), one, scale)
    _check_decode(one, one, q[8:9], stored[8:9], lens[8:9], hkv, scale, dtype)
    # an upper bound of the lengths cuts what is beyond it; a row out of range reads nothing
    out.fill_(7.0)
    eng.attend_decode(0, len(lens), rows, kv_len, 20, q, out, scale)
    _check_decode(out, before, q, [[x[:20] for x in s] for s in stored], [min(n, 20) for n in lens], hkv, scale, dtype,
                  lambda b, h, n: np.arange(min(n, gone * page) if b == 6 else 0, n))
    out.fill_(7.0)
    eng.attend_decode(0, 2, torch.tensor([-1, len(lens)], device="cuda", dtype=torch.int32), kv_len[6:8], 700, q[:2], out[:2], scale)
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    eng.check_kernels()
    eng.close()


@pytest.mark.gpu
def test_one_long_call_and_many_short_ones(drkv_lib):
    """Appends, flat copies out and in: the same bytes whether a CTA takes one token or a hundred."""
    import torch
    n, d = 90001, 128
    one, many = (_engine(hq=1, hkv=1, d=d, page=16, dtype="bf16", pages=5700, seqs=1, per_seq=5700, rot=32) for _ in range(2))
    for e in (one, many):
        e.seq_create()
        assert e.ensure_blocks_for_range(0, 0, n)
        e.set_seq_len(0, n)
        e.sync_block_table()
        e.pool_tensor().zero_()
    g = torch.Generator(device="cuda").manual_seed(12)
    k, v = (torch.randn(n, 1, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    one.append_rope_chunk(0, 0, 0, n, k, v)
    for a in range(0, n, 701):
        b = min(n, a + 701)
        many.append_rope_chunk(0, 0, a, b - a, k[a:b].contiguous(), v[a:b].contiguous())
    torch.cuda.synchronize()
    assert torch.equal(one.pool_tensor(), many.pool_tensor())
    flat = torch.empty(1, 2, n, 1, d, device="cuda", dtype=torch.bfloat16)
    one.extract(0, 0, n, flat)
    for a in range(0, n, 14001):
        b = min(n, a + 14001)
        part = torch.empty(1, 2, b - a, 1, d, device="cuda", dtype=torch.bfloat16)
        many.extract(0, a, b - a, part)
        torch.cuda.synchronize()
        assert torch.equal(part, flat[:, :, a:b])
    one.pool_tensor().zero_()
    one.inject(0, 0, n, flat)
    many.pool_tensor().zero_()
    for a in range(0, n, 14001):
        b = min(n, a + 14001)
        many.inject(0, a, b - a, flat[:, :, a:b].contiguous())
    torch.cuda.synchronize()
    assert torch.equal(one.pool_tensor(), many.pool_tensor())
    # A stored row quantises to the values it has, if not to its bytes: a maximum between 224 and 232 times 2^e was rounded to
    # 224 * 2^e = 448 * 2^(e - 1), and then e - 1 with doubled codes holds the same row.
    again = torch.empty_like(flat)
    one.extract(0, 0, n, again)
    torch.cuda.synchronize()
    assert torch.equal(again, flat)
    one.close()
    many.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq,grp,hkv,d", [(1, 4, 1, 256), (6, 8, 2, 128), (16, 8, 2, 128), (12, 8, 2, 128), (40, 8, 2, 128), (5, 16, 1, 256),
                                             (37, 16, 1, 256), (20, 4, 8, 64), (300, 4, 2, 64)])
def test_pieces_of_every_number(drkv_lib, n_seq, grp, hkv, d):
    """From hundreds of pieces a row to two, few rows and many: every way of merging them; entries of one table row."""
    import torch
    n = 1900
    eng = _engine(hq=grp * hkv, hkv=hkv, d=d, page=16, dtype="bf16", pages=128, seqs=1, per_seq=120)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n)
    eng.sync_block_table()
    stored = _fill(eng, [n], "bf16", 9, spread=1)[0]
    g = torch.Generator(device="cuda").manual_seed(n_seq)
    lens = [n - 37 * (i % 40) - i % 16 for i in range(n_seq)]
    q = torch.randn(n_seq, grp * hkv, d, generator=g, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    rows = torch.zeros(n_seq, device="cuda", dtype=torch.int32)
    eng.attend_decode(0, n_seq, rows, torch.tensor(lens, device="cuda", dtype=torch.int32), n, q, out, 1.0 / math.sqrt(d))
    torch.cuda.synchronize()
    eng.check_kernels()
    some = sorted(set(range(0, n_seq, max(1, n_seq // 12))) | {n_seq - 1})
    _check_decode(out[some], out[some], q[some], [stored for _ in some], [lens[i] for i in some], hkv, 1.0 / math.sqrt(d), "bf16")
    eng.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_of_unlike_size(drkv_lib, dtype):
    """One value row is 2^20 times the others and has next to no weight; one query row is tiny, one large."""
    import torch
    t = _torch_dtype(dtype)
    eng = _engine(hq=4, hkv=1, d=128, dtype=dtype, pages=16, seqs=1)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 100)
    eng.set_seq_len(0, 100)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(100, 1, 128, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(1, 4, 128, generator=g, device="cuda")
    k[37] = -8.0 * q[0].mean(0)                                     # e^-40 or so of the others' weight
    v[37] = v[37].sign() * 30000.0
    v[:37] *= 2.0 ** -5
    q[0, 1] *= 2.0 ** -12
    q[0, 2] *= 2.0 ** 6
    k, v, q = k.to(t), v.to(t), q.to(t)
    eng.append_rope_chunk(0, 0, 0, 100, k, v)
    out = torch.zeros_like(q)
    one = torch.tensor([100], device="cuda", dtype=torch.int32)
    eng.attend_decode(0, 1, one - 100, one, 100, q, out, 0.3)
    stored = [[R.stored_values(x.double().cpu().numpy()) for x in (k, v)]]
    _check_decode(out, out, q, stored, [100], 1, 0.3, dtype)
    eng.close()


@pytest.mark.gpu
@pytest.mark.parametrize("d,rot,hkv,page,n_seq", [(128, 0, 2, 16, 4), (256, 64, 4, 16, 3), (64, 64, 2, 48, 4), (128, 128, 1, 32, 5),
                                                  (64, 16, 8, 16, 330)])
def test_step_appends_and_attends(drkv_lib, d, rot, hkv, page, n_seq):
    """append_attend_decode = append at kv_len - 1, then attention, to the bit; planned passes too; captured, replayed."""
    import torch
    lens = ([17, 1, 200, 48, 33] + [1 + 7 * i % 60 for i in range(n_seq)])[:n_seq]
    per = -(-210 // page)
    eng, ref = (_engine(hq=4 * hkv, hkv=hkv, d=d, page=page, dtype="bf16", layers=2, pages=n_seq * 5 + 16, seqs=n_seq, per_seq=per, rot=rot)
                for _ in range(2))
    for e in (eng, ref):
        for s, n in enumerate(lens):
            e.seq_create()
            assert e.ensure_blocks_for_range(s, 0, n + 2)
            e.set_seq_len(s, n)
        e.sync_block_table()
        _fill(e, [n - 1 for n in lens], "bf16", 3, layer=1)
    g = torch.Generator(device="cuda").manual_seed(4)
    new = [torch.randn(n_seq, hkv, d, generator=g, device="cuda").bfloat16() for _ in range(2)]
    new[0][0, 0, 3], new[1][1, 0, 5] = float("inf"), 0.0
    q = torch.randn(n_seq, 4 * hkv, d, generator=g, device="cuda").bfloat16()
    rows = torch.arange(n_seq, device="cuda", dtype=torch.int32)
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    want, out, planned = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))

    def reference():
        ref.append_rope(1, n_seq, rows, kv_len - 1, new[0], new[1])
        ref.attend_decode(1, n_seq, rows, kv_len, 210, q, want, 0.1)
        torch.cuda.synchronize()
    reference()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        eng.append_attend_decode(1, n_seq, rows, kv_len, 210, new[0], new[1], q, out, 0.1, torch.cuda.current_stream())
    graph.replay()
    torch.cuda.synchronize()
    assert same(out, want) and torch.equal(eng.pool_tensor(), ref.pool_tensor())
    kv_len += 1                                                      # the replay reads the lengths of its own time
    reference()
    graph.replay()
    torch.cuda.synchronize()
    assert same(out, want) and torch.equal(eng.pool_tensor(), ref.pool_tensor())
    info = eng.plan_decode(list(range(n_seq)), [n + 1 for n in lens])
    assert info["n_families"] == 0
    eng.attend_decode_planned(1, q, planned, 0.1)
    eng.append_attend_decode_planned(1, new[0], new[1], q, planned, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(eng.pool_tensor(), ref.pool_tensor())
    # the plan's bound of the lengths is its own, and with it the split of the keys: the same values but for rounding
    finite = torch.isfinite(out).all(-1)
    assert ((planned - out).abs().amax(-1)[finite] <= 2.0 ** -6 * out.abs().amax(-1)[finite]).all()
    eng.check_kernels()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,grp,page", [("bf16", 128, 4, 16), ("f16", 256, 6, 16), ("bf16", 64, 8, 48)])
def test_prefill_over_the_pool(drkv_lib, dtype, d, grp, page):
    """A chunk over earlier tokens, two sequences in one call (a fork sharing pages with its parent), stale NaN behind."""
    import torch
    t, hkv = _torch_dtype(dtype), 2
    eng = _engine(hq=grp * hkv, hkv=hkv, d=d, page=page, dtype=dtype, layers=2, pages=64, seqs=3, per_seq=20)
    _shuffle(eng, 1)
    n, m = 230, 90
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n - 35)
    eng.pool_tensor().fill_(-1)
    eng.sync_block_table()
    stored = _fill(eng, [n], dtype, 6, layer=1, spread=1)[0]
    child = eng.seq_fork(0)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(7)
    qs = [torch.randn(m, grp * hkv, d, generator=g, device="cuda").to(t) for _ in range(2)]
    outs = [torch.zeros_like(x) for x in qs]
    starts = [n - m, n - m - 35]
    scale = 1.0 / math.sqrt(d)
    eng.attend_prefill_batch(1, [0, child], starts, [m, m], qs, outs, scale)
    torch.cuda.synchronize()
    eng.check_kernels()
    for i in range(2):
        for tok in (0, 1, 15, 16, 63, m - 1):
            end = starts[i] + tok + 1
            for h in range(hkv):
                rows = slice(h * grp, (h + 1) * grp)
                want, pv, mag = R.attend(qs[i][tok, rows].double().cpu().numpy(), stored[0][:end, h], stored[1][:end, h], scale)
                # the prefill kernel rounds P to the storage type
                tol = R.attend_tolerance(want, pv, mag, _half_step(dtype), _half_step(dtype))
                err = np.abs(outs[i][tok, rows].double().cpu().numpy() - want)
                assert (err <= tol).all(), (i, tok, h, float((err / tol).max()))
    one = torch.zeros_like(qs[0])
    eng.attend_prefill_chunk(1, 0, starts[0], m, qs[0], one, scale)
    torch.cuda.synchronize()
    assert torch.equal(one, outs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("page,hkv,d,n,m", [(128, 5, 256, 43, 43), (128, 8, 64, 130, 2), (64, 3, 128, 1, 1)])
def test_prefill_of_few_large_pages(drkv_lib, page, hkv, d, n, m):
    """Pages that several CTAs expand, the last one only in part visible."""
    import torch
    eng = _engine(hq=hkv, hkv=hkv, d=d, page=page, dtype="bf16", pages=4, seqs=2, per_seq=2)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n)
    eng.pool_tensor().fill_(-1)
    eng.sync_block_table()
    stored = _fill(eng, [n], "bf16", 3, spread=1)[0]
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(m, hkv, d, generator=g, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    scale = 1.0 / math.sqrt(d)
    eng.attend_prefill_batch(0, [0], [n - m], [m], [q], [out], scale)
    torch.cuda.synchronize()
    eng.check_kernels()
    for t in range(m):
        end = n - m + t + 1
        for h in range(hkv):
            want, pv, mag = R.attend(q[t, h:h + 1].double().cpu().numpy(), stored[0][:end, h], stored[1][:end, h], scale)
            tol = R.attend_tolerance(want, pv, mag, _half_step("bf16"), _half_step("bf16"))
            assert (np.abs(out[t, h:h + 1].double().cpu().numpy() - want) <= tol).all(), (t, h)
    eng.close()


@pytest.mark.gpu
def test_prefill_pages_shared_out_of_step(drkv_lib):
    """One page at different places of two sequences' tables, whole for one and the tail of the other, in one call."""
    import torch
    eng = _engine(hq=4, hkv=1, d=64, page=16, dtype="bf16", pages=8, seqs=3, per_seq=4)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 48)
    eng.set_seq_len(0, 48)
    eng.sync_block_table()
    stored = _fill(eng, [48], "bf16", 1, spread=1)[0]
    other = eng.seq_create()
    pages = [int(p) for p in eng.table(0)[:3]]
    eng.adopt(other, [pages[2], pages[0]], 20)                       # its last page holds 4 tokens of the parent's first 16
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(2)
    qs = [torch.randn(4, 4, 64, generator=g, device="cuda").bfloat16() for _ in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    eng.attend_prefill_batch(0, [0, other], [44, 16], [4, 4], qs, outs, 0.125)
    torch.cuda.synchronize()
    order = [np.arange(48), np.concatenate([np.arange(32, 48), np.arange(16)])]
    for i, start in enumerate((44, 16)):
        for t in range(4):
            see = order[i][:start + t + 1]
            want, pv, mag = R.attend(qs[i][t].double().cpu().numpy(), stored[0][see, 0], stored[1][see, 0], 0.125)
            tol = R.attend_tolerance(want, pv, mag, _half_step("bf16"), _half_step("bf16"))
            assert (np.abs(outs[i][t].double().cpu().numpy() - want) <= tol).all(), (i, t)
    # a NaN in a slot that the parent sees and the other's last page hides: the parent's answer is that of a call of its own
    block = eng.pool_tensor().reshape(8, -1)[pages[0]]
    for plane in (0, 1):
        block[(plane * 16 + 9) * 32:(plane * 16 + 10) * 32] = -1
    alone = torch.zeros_like(outs[0])
    eng.attend_prefill_chunk(0, 0, 44, 4, qs[0], alone, 0.125)
    assert not torch.equal(alone, outs[0])
    for first, second in ((0, other), (other, 0)):
        again = {0: torch.zeros_like(outs[0]), other: torch.zeros_like(outs[1])}
        slot = {0: 0, other: 1}
        eng.attend_prefill_batch(0, [first, second], [(44, 16)[slot[x]] for x in (first, second)], [4, 4],
                                 [qs[slot[x]] for x in (first, second)], [again[first], again[second]], 0.125)
        torch.cuda.synchronize()
        assert torch.equal(again[0].view(torch.int16), alone.view(torch.int16))
    eng.close()


@pytest.mark.gpu
def test_more_sequences_than_one_launch(drkv_lib):
    """1030 rows of a batch over three sequences: two launches, every row as a batch of one gives it but for the split."""
    import torch
    lens = [40, 7, 100]
    eng = _engine(hq=4, hkv=2, d=64, page=16, dtype="f16", pages=16, seqs=3, per_seq=8)
    for s, n in enumerate(lens):
        eng.seq_create()
        assert eng.ensure_blocks_for_range(s, 0, n)
        eng.set_seq_len(s, n)
    eng.sync_block_table()
    stored = _fill(eng, lens, "f16", 1)
    n = 1030
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn(n, 4, 64, generator=g, device="cuda").half()
    rows = torch.arange(n, device="cuda", dtype=torch.int32) % 3
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)[rows.long()].contiguous()
    out = torch.zeros_like(q)
    eng.attend_decode(0, n, rows, kv_len, 100, q, out, 0.1)
    torch.cuda.synchronize()
    some = [0, 1, 2, 500, 1021, 1022, 1023, 1024, 1025, 1026, 1029]
    _check_decode(out[some], out[some], q[some], [stored[i % 3] for i in some], [lens[i % 3] for i in some], 2, 0.1, "f16")
    eng.close()


@pytest.mark.gpu
def test_fork_copy_on_write_and_tier(drkv_lib, tmp_path):
    """A fork's write leaves the parent's page alone; pages that went to files and back hold the same bytes."""
    import torch
    eng = _engine(hq=4, hkv=2, d=64, page=16, dtype="f16", layers=2, pages=12, seqs=3, per_seq=16, stream_evict=True)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 70)
    eng.set_seq_len(0, 70)
    eng.sync_block_table()
    for layer in (0, 1):
        _fill(eng, [70], "f16", 8 + layer, layer=layer)
    flat = torch.empty(2, 2, 70, 2, 64, device="cuda", dtype=torch.float16)
    eng.extract(0, 0, 70, flat)
    child = eng.seq_fork(0)
    assert eng.ensure_blocks_for(child, 70)                          # copies the tail page
    eng.sync_block_table()
    assert eng.table(child)[4] != eng.table(0)[4]
    new = torch.ones(1, 2, 64, device="cuda", dtype=torch.float16)
    eng.append_rope_chunk(0, child, 70, 1, new, new)
    again = torch.empty(2, 2, 71, 2, 64, device="cuda", dtype=torch.float16)
    eng.extract(child, 0, 71, again)
    torch.cuda.synchronize()
    assert torch.equal(again[:, :, :70], flat) and (again[0, :, 70] == 1).all()
    eng.extract(0, 0, 70, again[:, :, :70].contiguous())
    eng.seq_release(child, discard=True)
    eng.tier_enable(str(tmp_path))
    assert eng.tier_stats()["page_file_bytes"] == 0 or eng.tier_stats()["page_file_bytes"] == 2 * 2 * 2 * 16 * 65
    assert eng.evict_blocks(0, 3) == 3
    eng.pool_tensor()[:100] = 0x2222                                 # what the freed pages held is gone
    assert eng.ensure_blocks_for_range(0, 0, 70)
    eng.sync_block_table()
    back = torch.empty_like(flat)
    eng.extract(0, 0, 70, back)
    torch.cuda.synchronize()
    assert torch.equal(back, flat)
    assert eng.tier_stats()["page_file_bytes"] == 2 * 2 * 2 * 16 * 65
    eng.close()


@pytest.mark.gpu
def test_refusals_on_device(drkv_lib):
    import torch
    from deusridet_b200 import DrkvError, capi
    eng = _engine(pages=8, seqs=1)
    x = torch.zeros(16, 8, 128, device="cuda", dtype=torch.bfloat16)
    one = torch.ones(1, device="cuda", dtype=torch.int32)
    part = torch.zeros(eng.partial_floats(), device="cuda")
    for call in (lambda: eng.attend_partial(0, 0, 0, 4, x, part, 1.0), lambda: eng.exchange_create(2, 0),
                 lambda: eng.append_rope_chunk(0, 0, 2 ** 31 - 4, 16, x, x), lambda: eng.extract(0, 2 ** 31 - 4, 16, x),
                 lambda: eng.append_rope(1, 1, one, one, x, x), lambda: eng.attend_decode(0, 1, one, one, -1, x, x, 1.0),
                 lambda: eng.append_rope_chunk(0, 1, 0, 1, x, x), lambda: eng.append_rope_chunk(0, 0, 0, 1, x.data_ptr() + 2, x),
                 lambda: eng.append_rope(0, 1, one, one, x, x.data_ptr() + 8), lambda: eng.extract(0, 0, 1, x.data_ptr() + 8),
                 lambda: eng.inject(0, 0, 1, x.data_ptr() + 2), lambda: eng.attend_decode(0, 1, one, one, 16, x.data_ptr() + 2, x, 1.0),
                 lambda: eng.append_attend_decode(0, 1, one, one, 16, x, x, x, x.data_ptr() + 4, 1.0)):
        with pytest.raises(DrkvError) as err:
            call()
        assert err.value.code == capi.ERR_INVALID
    eng.attend_decode(0, 0, one, one, 16, x, x, 1.0)
    eng.append_rope_chunk(0, 0, 0, 0, x, x)
    eng.extract(0, 0, 0, x)
    eng.check_kernels()
