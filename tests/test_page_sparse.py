"""Page bounds, page selection and attention over listed pages, on both kinds of pool, against numpy in 64 bits; and a long
decode run of all of it together with the rotary operator."""
import math

import numpy as np
import pytest

from tests import cache8_helpers as R
from tests.test_cache8 import _check_decode, _half_step, _shuffle, _torch_dtype

pytestmark = pytest.mark.gpu


def _engine(pool, hq, hkv, d, page, dtype, pages, seqs, per_seq, layers=1, **kw):
    from deusridet_b200 import PagedKVEngine
    return PagedKVEngine(num_layers=layers, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, page_size=page, dtype=dtype,
                         kv_dtype=pool, rotary_dim=0, max_pages=pages, max_seqs=seqs, max_pages_per_seq=per_seq, device=0, **kw)


def _start(eng, lens, room=None, seed=1):
    _shuffle(eng, seed)
    for s, n in enumerate(lens):
        eng.seq_create()
        assert eng.ensure_blocks_for_range(s, 0, max(room or n, 1))
        eng.set_seq_len(s, n)
    eng.sync_block_table()


def _rows(n, hkv, d, t, gen):
    """Keys with an offset, channels of unlike size."""
    import torch
    spread = torch.exp(torch.randn(hkv, d, generator=gen, device="cuda"))
    return ((torch.randn(n, hkv, d, generator=gen, device="cuda") + 0.5) * spread).to(t)


def _stored(x, pool):
    x = x.double().cpu().numpy()
    return R.stored_values(x) if pool else x


def _check_bounds(eng, layer, seq, k, page, skip=()):
    """Every page of the sequence has exactly the bounds of its keys k [n, hkv, d]."""
    b, e = (t.cpu().numpy() for t in eng.page_bounds())
    table = eng.table(seq)
    for lp in range(-(-len(k) // page)):
        if lp in skip or table[lp] < 0:
            continue
        for h in range(k.shape[1]):
            hi, lo, ex = R.bounds(k[lp * page:(lp + 1) * page, h])
            assert e[layer, table[lp], h] == ex, (seq, lp, h)
            assert np.array_equal(b[layer, table[lp], h, 0], hi) and np.array_equal(b[layer, table[lp], h, 1], lo), (seq, lp, h)


def _page_bounds_of(k, page):
    hi, lo, ex = zip(*(R.bounds(k[p * page:(p + 1) * page]) for p in range(-(-len(k) // page))))
    return np.array(hi), np.array(lo), np.array(ex)


@pytest.mark.parametrize("pool", [None, "e4m3"])
@pytest.mark.parametrize("dtype,d,page", [("bf16", 128, 16), ("f16", 64, 48), ("bf16", 256, 32)])
def test_bounds_follow_every_write(drkv_lib, tmp_path, pool, dtype, d, page):
    """Chunks cut anywhere, batches, decode steps, inject, fork and copy on write, storage tier: the bounds of one pass."""
    import torch
    t, hkv, n = _torch_dtype(dtype), 2, 5 * page - 3
    eng = _engine(pool, 4, hkv, d, page, dtype, 32, 4, 8, layers=2, stream_evict=True)
    eng.page_bounds_enable()
    _start(eng, [n, n, n], room=n + 5)
    g = torch.Generator(device="cuda").manual_seed(d + page)
    k, v = _rows(n + 4, hkv, d, t, g), _rows(n + 4, hkv, d, t, g)
    k[3, 0, 5], k[page + 1, 1, 0], k[7, :, :] = 0.0, -60000.0, 0.0
    ks = _stored(k, pool)
    # sequence 0: uneven chunks; sequence 1: token by token in batches, many tokens of a page in one call; 2: injected
    cuts = [0, 1, 3, page, page + 5, 3 * page + 1, n]
    for a, b in zip(cuts, cuts[1:]):
        eng.append_rope_chunk(1, 0, a, b - a, k[a:b].contiguous(), v[a:b].contiguous())
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    for a, b in ((0, 5), (5, 2 * page + 2), (2 * page + 2, n)):
        # within a batch the order of the tokens does not matter
        perm = a + torch.randperm(b - a, generator=g, device="cuda")
        eng.append_rope(1, b - a, torch.ones(b - a, device="cuda", dtype=torch.int32), pos[perm].contiguous(), k[perm], v[perm])
    flat = torch.stack([torch.stack([k[:n], v[:n]])] * 2).contiguous()
    eng.inject(2, 0, n, flat)
    torch.cuda.synchronize()
    for seq in range(3):
        _check_bounds(eng, 1, seq, ks[:n], page)
    _check_bounds(eng, 0, 2, ks[:n], page)
    # a decode step's token widens its page
    q = torch.randn(3, 4, d, generator=g, device="cuda").to(t)
    rows = torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32)
    lens = torch.full_like(rows, n + 1)
    rep = lambda x: x[n:n + 1].expand(3, hkv, d).contiguous()
    eng.append_attend_decode(1, 3, rows, lens, n + 1, rep(k), rep(v), q, torch.zeros_like(q), 0.1)
    for s in range(3):
        eng.set_seq_len(s, n + 1)
    torch.cuda.synchronize()
    for seq in range(3):
        _check_bounds(eng, 1, seq, ks[:n + 1], page)
    eng.plan_decode([0, 1], [n + 2, n + 2])
    eng.append_attend_decode_planned(1, k[n + 1:n + 2].expand(2, hkv, d).contiguous(), v[n + 1:n + 2].expand(2, hkv, d).contiguous(),
                                     q[:2].contiguous(), torch.zeros_like(q[:2]), 0.1)
    for s in range(2):
        eng.set_seq_len(s, n + 2)
    torch.cuda.synchronize()
    for seq in range(2):
        _check_bounds(eng, 1, seq, ks[:n + 2], page)
    # a fork's copy takes the bounds along and widens its own
    child = eng.seq_fork(0)
    assert eng.ensure_blocks_for(child, n + 2)
    eng.sync_block_table()
    assert eng.table(child)[4] != eng.table(0)[4]
    big = k[n + 2:n + 3] * 4
    eng.append_rope_chunk(1, child, n + 2, 1, big, big)
    torch.cuda.synchronize()
    _check_bounds(eng, 1, 0, ks[:n + 2], page)
    _check_bounds(eng, 1, child, np.concatenate([ks[:n + 2], _stored(big, pool)]), page)
    # pages that come back from storage, under other ids
    eng.tier_enable(str(tmp_path))
    eng.seq_release(child, discard=True)
    assert eng.evict_blocks(1, 3) == 3
    grab = [eng.alloc_block() for _ in range(eng.free_count() - 3)]
    assert eng.ensure_blocks_for_range(1, 0, n)
    eng.sync_block_table()
    torch.cuda.synchronize()
    _check_bounds(eng, 1, 1, ks[:n + 2], page)
    for p in grab:
        eng.free_block(p)
    # a recycled page starts anew at its slot 0, whatever it held
    eng.seq_release(2, discard=True)
    s = eng.seq_create()
    assert eng.ensure_blocks_for_range(s, 0, page)
    eng.set_seq_len(s, 2)
    eng.sync_block_table()
    small = (k[:2] * 0.01).contiguous()
    eng.append_rope_chunk(1, s, 0, 2, small, small)
    torch.cuda.synchronize()
    _check_bounds(eng, 1, s, _stored(small, pool), page)
    # scanned whole: every slot of the full pages
    eng.page_bounds_enable()
    torch.cuda.synchronize()
    _check_bounds(eng, 1, 0, ks[:n + 2], page, skip=(4,))
    eng.check_kernels()
    eng.close()


@pytest.mark.parametrize("pool", [None, "e4m3"])
def test_bounds_of_a_long_chunk(drkv_lib, pool):
    """So many pages that a warp takes one each, begun inside a page; appended, then scanned."""
    import torch
    n, hkv, d, page = 19203, 8, 64, 16
    eng = _engine(pool, 8, hkv, d, page, "bf16", 1210, 1, 1205)
    eng.page_bounds_enable()
    _start(eng, [n])
    g = torch.Generator(device="cuda").manual_seed(4)
    k = _rows(n, hkv, d, torch.bfloat16, g)
    eng.append_rope_chunk(0, 0, 0, 5, k[:5].contiguous(), k[:5].contiguous())
    eng.append_rope_chunk(0, 0, 5, n - 5, k[5:].contiguous(), k[5:].contiguous())
    torch.cuda.synchronize()
    ks = _stored(k, pool)
    _check_bounds(eng, 0, 0, ks, page)
    bounds, exponents = eng.page_bounds()
    bounds.zero_()
    exponents.zero_()
    eng.page_bounds_enable()
    torch.cuda.synchronize()
    _check_bounds(eng, 0, 0, ks[:n // page * page], page)
    eng.check_kernels()
    eng.close()


def test_bounds_of_extreme_keys(drkv_lib):
    """Zeros, the smallest and largest values, infinities and NaN."""
    import torch
    eng = _engine(None, 2, 1, 64, 16, "bf16", 8, 1, 4)
    eng.page_bounds_enable()
    _start(eng, [64])
    k = torch.zeros(64, 1, 64, device="cuda", dtype=torch.bfloat16)
    k[16:32, 0, 0], k[16:32, 0, 1] = 2.0 ** -133, -(2.0 ** -130)
    k[20, 0, 2] = 2.0 ** -100
    k[32, 0, 0], k[33, 0, 0], k[32, 0, 1] = 3.3e38, -3.3e38, 1e-30
    k[48, 0, 0], k[49, 0, 1], k[50, 0, 2], k[48:64, 0, 3] = math.inf, -math.inf, math.nan, math.nan
    k[51, 0, 2] = -5.0
    eng.append_rope_chunk(0, 0, 0, 64, k, k)
    torch.cuda.synchronize()
    _check_bounds(eng, 0, 0, k[:48].double().cpu().numpy(), 16)
    b, e = (t.cpu().numpy() for t in eng.page_bounds())
    p = eng.table(0)[3]
    assert e[0, p, 0] == 121 and list(b[0, p, 0, 0, :5]) == [127, 0, 0, 0, 0] and list(b[0, p, 0, 1, :5]) == [0, -127, -1, 0, 0]
    eng.close()


def _selection(q, k, page, n, resident, top, first, last):
    return R.select(R.page_scores(q, *_page_bounds_of(k[:n], page)), resident, top, first, last)


@pytest.mark.parametrize("pool", [None, "e4m3"])
@pytest.mark.parametrize("dtype,d,grp,hkv,page", [("bf16", 128, 4, 2, 16), ("f16", 64, 1, 3, 48), ("bf16", 256, 6, 2, 16),
                                                  ("f16", 128, 16, 1, 32), ("bf16", 64, 9, 2, 16)])
def test_select_and_attend(drkv_lib, pool, dtype, d, grp, hkv, page):
    import torch
    t = _torch_dtype(dtype)
    lens = [1, 0, 16, 17, 1100, 5 * page, 777, 1100]
    per = -(-1100 // page)
    eng = _engine(pool, grp * hkv, hkv, d, page, dtype, len(lens) * per, len(lens), per, stream_evict=True)
    eng.page_bounds_enable()
    _start(eng, lens)
    g = torch.Generator(device="cuda").manual_seed(grp)
    ks, vs = [], []
    for s, n in enumerate(lens):
        k, v = _rows(max(n, 1), hkv, d, t, g), _rows(max(n, 1), hkv, d, t, g)
        if s == 7:
            k = k[:page].repeat(per, 1, 1)[:n].contiguous()         # every full page the same: ties
        if n:
            eng.append_rope_chunk(0, s, 0, n, k, v)
        ks.append(_stored(k, pool))
        vs.append(_stored(v, pool))
    assert eng.evict_blocks(4, 3) == 3                              # holes where the first pages would be
    eng.sync_block_table()
    q = torch.randn(len(lens), grp * hkv, d, generator=g, device="cuda").to(t)
    q[6] *= 1e-3
    if dtype == "bf16":                                             # exponents at the ends of fp32, heads far apart
        q[4, 0], q[4, -1] = q[4, 0] * 1e-25, q[4, -1] * 1e-36
        q[7] *= 1e25
    rows = torch.arange(len(lens), device="cuda", dtype=torch.int32)
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    scale = 1.0 / math.sqrt(d)
    for top, first, last in ((1, 0, 0), (1, 1, 0), (4, 1, 2), (7, 0, 1), (20, 2, 3), (per + 3, 1, 1)):
        sel = torch.full((len(lens), hkv, top), 99, device="cuda", dtype=torch.int32)
        eng.select_pages(0, len(lens), rows, kv_len, 1100, q, top, first, last, sel)
        got = sel.cpu().numpy()
        qd = q.double().cpu().numpy()
        for b, n in enumerate(lens):
            resident = np.array([not (b == 4 and p < 3) for p in range(-(-n // page))], dtype=bool)
            for h in range(hkv):
                want = _selection(qd[b, h * grp:(h + 1) * grp], ks[b][:, h], page, n, resident, top, first, last) if n else []
                assert list(got[b, h]) == want + [-1] * (top - len(want)), (b, h, top)
        out = torch.full_like(q, 3.0)
        before = out.clone()
        eng.attend_selected(0, len(lens), rows, kv_len, 1100, sel, top, q, out, scale)

        def visible(b, h, n):
            keep = np.zeros(n, dtype=bool)
            for p in got[b, h]:
                if p >= 0:
                    keep[p * page:(p + 1) * page] = True
            return np.flatnonzero(keep)
        weight_step = 2.0 ** -11 if pool and dtype == "bf16" else 2.0 ** -17
        _check_sparse(out, before, q, ks, vs, lens, hkv, scale, dtype, visible, weight_step)
    # all pages listed is dense attention: both within their bounds of the 64-bit result (the split of the keys over warps
    # differs, a list counts whole pages and no holes, so the bits may)
    dense = torch.full_like(q, 3.0)
    eng.attend_decode(0, len(lens), rows, kv_len, 1100, q, dense, scale)
    _check_sparse(dense, before, q, ks, vs, lens, hkv, scale, dtype, visible, weight_step)
    eng.check_kernels()
    eng.close()


def _check_sparse(out, before, q, ks, vs, lens, hkv, scale, dtype, visible, weight_step):
    got, qd = out.double().cpu().numpy(), q.double().cpu().numpy()
    grp = q.shape[1] // hkv
    for b, n in enumerate(lens):
        for h in range(hkv):
            rows = slice(h * grp, (h + 1) * grp)
            see = visible(b, h, n)
            if len(see) == 0:
                assert np.array_equal(got[b, rows], before.double().cpu().numpy()[b, rows])
                continue
            want, pv, mag = R.attend(qd[b, rows], ks[b][see, h], vs[b][see, h], scale)
            tol = R.attend_tolerance(want, pv, mag, _half_step(dtype), weight_step)
            err = np.abs(got[b, rows] - want)
            assert (err <= tol).all(), (b, h, float((err / tol).max()))


@pytest.mark.parametrize("pool", [None, "e4m3"])
def test_lists_of_the_callers_own(drkv_lib, pool):
    """Any order, a page twice, entries out of range, none at all; only the first ceil(kv_len / page_size) are read."""
    import torch
    page, hkv, grp, d, n = 16, 2, 4, 128, 100
    eng = _engine(pool, 8, hkv, d, page, "f16", 16, 1, 10)
    _start(eng, [n])
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = _rows(n, hkv, d, torch.float16, g), _rows(n, hkv, d, torch.float16, g)
    eng.append_rope_chunk(0, 0, 0, n, k, v)
    q = torch.randn(1, 8, d, generator=g, device="cuda").half()
    one = torch.tensor([n], device="cuda", dtype=torch.int32)
    ks, vs = _stored(k, pool), _stored(v, pool)
    for lists in ([[6, 0, 3], [2, 2, 5]], [[-1, 9, 4], [2 ** 31 - 1, -2 ** 31, 0]], [[-1, -1, -1], [7, 8, 1000000]],
                  [[5, 4, 3, 2, 1, 0, 6, 6, 6], [0, -1, 0, -1, 0, -1, 1, 2, 3]]):
        sel = torch.tensor([lists], device="cuda", dtype=torch.int64).to(torch.int32)
        out = torch.full_like(q, 3.0)
        before = out.clone()
        eng.attend_selected(0, 1, one - n, one, n, sel, len(lists[0]), q, out, 0.1)

        def visible(b, h, n):
            return np.array([i for p in lists[h][:7] if 0 <= p < 7 for i in range(p * page, min(n, (p + 1) * page))], dtype=int)
        _check_sparse(out, before, q, [ks], [vs], [n], hkv, 0.1, "f16", visible, 2.0 ** -17)
    eng.check_kernels()
    eng.close()


def test_many_pages_and_long_lists(drkv_lib):
    """More pages than the selection keeps in shared memory; scores that differ in their last bits only."""
    import torch
    page, n_pages, d = 16, 12500, 64
    n = page * n_pages - 5
    eng = _engine("e4m3", 2, 1, d, page, "bf16", n_pages, 1, n_pages)
    eng.page_bounds_enable()
    _start(eng, [n])
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randint(-3, 4, (n, 1, d), generator=g, device="cuda").bfloat16()
    eng.append_rope_chunk(0, 0, 0, n, k, k)
    q = torch.randint(-2, 3, (1, 2, d), generator=g, device="cuda").bfloat16()
    one = torch.tensor([n], device="cuda", dtype=torch.int32)
    kd = k[:, 0].double().cpu().numpy()
    pad = np.concatenate([kd, np.repeat(kd[-1:], page * n_pages - n, 0)]).reshape(n_pages, page, d)
    hi, lo = pad.max(1), pad.min(1)
    e = R.exponent_for(np.maximum(np.abs(hi), np.abs(lo)).max(1), 127.0, -126, 121)
    unit = 2.0 ** e[:, None].astype(float)
    scores = R.page_scores(q[0].double().cpu().numpy(), np.ceil(hi / unit), np.floor(lo / unit), e)
    for top in (1, 300, 12499, 12500):
        sel = torch.empty(1, 1, top, device="cuda", dtype=torch.int32)
        eng.select_pages(0, 1, one - n, one, n, q, top, 1 if top > 1 else 0, 1, sel)
        assert sel.cpu().numpy().ravel().tolist() == R.select(scores, np.ones(n_pages, bool), top, 1 if top > 1 else 0, 1)
    eng.close()


def test_refusals(drkv_lib):
    import torch
    from deusridet_b200 import DrkvError, capi
    eng = _engine(None, 4, 1, 64, 16, "bf16", 8, 1, 4)
    one = torch.ones(1, device="cuda", dtype=torch.int32)
    x, sel = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(8, device="cuda", dtype=torch.int32)
    with pytest.raises(DrkvError) as err:
        eng.select_pages(0, 1, one, one, 16, x, 4, 1, 1, sel)
    assert err.value.code == capi.ERR_STATE
    with pytest.raises(DrkvError):
        eng.page_bounds()
    eng.page_bounds_enable()
    for call in (lambda: eng.select_pages(1, 1, one, one, 16, x, 4, 1, 1, sel), lambda: eng.select_pages(0, 1, one, one, 16, x, 0, 0, 0, sel),
                 lambda: eng.select_pages(0, 1, one, one, 16, x, 4, 3, 2, sel), lambda: eng.select_pages(0, 1, one, one, 16, x, 4, -1, 2, sel),
                 lambda: eng.select_pages(0, 1, one, one, 16, x, 2, 2 ** 31 - 1, 2 ** 31 - 1, sel),
                 lambda: eng.select_pages(0, 1, one, one, -1, x, 4, 1, 1, sel), lambda: eng.select_pages(0, 1, one, one, 16, None, 4, 1, 1, sel),
                 lambda: eng.select_pages(0, 1, one, one, 16, x.data_ptr() + 2, 4, 1, 1, sel),
                 lambda: eng.attend_selected(0, 1, one, one, 16, sel, 4, x.data_ptr() + 2, x, 1.0),
                 lambda: eng.attend_selected(0, 1, one, one, 16, sel, 4, x, x.data_ptr() + 8, 1.0),
                 lambda: eng.attend_selected(0, 1, one, one, 16, None, 4, x, x, 1.0),
                 lambda: eng.attend_selected(0, 1, one, one, 16, sel, 0, x, x, 1.0), lambda: eng.attend_selected(0, -1, one, one, 16, sel, 4, x, x, 1.0)):
        with pytest.raises(DrkvError) as err:
            call()
        assert err.value.code == capi.ERR_INVALID
    sel.fill_(5)
    eng.select_pages(0, 0, one, one, 16, x, 4, 1, 1, sel)
    assert (sel == 5).all()
    eng.select_pages(0, 1, one, one, 0, x, 4, 1, 1, sel)             # no key within the bound of the lengths
    assert sel.tolist() == [-1] * 4 + [5] * 4
    eng.close()


@pytest.mark.parametrize("pool,dtype", [(None, "bf16"), ("e4m3", "f16")])
def test_long_decode_run(drkv_lib, pool, dtype):
    """As a server uses them: rotate q and k at scaled far positions, append, choose pages, attend; captured once and
    replayed over steps, then checked against 64 bits from the rotation on."""
    import torch
    from deusridet_b200 import Rope
    from tests.test_rope import expected_frequencies, rotate64
    t, page, hq, hkv, d, steps = _torch_dtype(dtype), 16, 8, 2, 128, 20
    lens0, top = [500, 37, 260], 6
    kw = dict(factor=8.0, original_context=4096, beta_fast=32.0, beta_slow=1.0)
    rope = Rope(head_dim=d, rotary_dim=64, layout="pairs", dtype=dtype, scaling="ramp", theta=1e6, device=0, **kw)
    freq, a = expected_frequencies(64, 1e6, "ramp", **kw)
    eng = _engine(pool, hq, hkv, d, page, dtype, 128, 3, 40)
    eng.page_bounds_enable()
    _start(eng, lens0, room=600)
    g = torch.Generator(device="cuda").manual_seed(8)
    far = 200000
    ks, vs = [], []
    for s, n in enumerate(lens0):
        k, v = _rows(n, hkv, d, t, g), _rows(n, hkv, d, t, g)
        _, kr = rope.apply(far + torch.arange(n, device="cuda", dtype=torch.int32), None, k)
        eng.append_rope_chunk(0, s, 0, n, kr, v)
        ks.append([_stored(kr, pool)])
        vs.append([_stored(v, pool)])
    qkv = torch.zeros(3, (hq + 2 * hkv) * d, device="cuda", dtype=t)
    q_in, k_in = qkv[:, :hq * d].unflatten(1, (hq, d)), qkv[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    q, k, v = torch.zeros(3, hq, d, device="cuda", dtype=t), torch.zeros(3, hkv, d, device="cuda", dtype=t), torch.zeros(3, hkv, d, device="cuda", dtype=t)
    pos, kv_len = torch.zeros(3, device="cuda", dtype=torch.int32), torch.zeros(3, device="cuda", dtype=torch.int32)
    sel, out = torch.zeros(3, hkv, top, device="cuda", dtype=torch.int32), torch.zeros(3, hq, d, device="cuda", dtype=t)
    rows = torch.arange(3, device="cuda", dtype=torch.int32)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        st = torch.cuda.current_stream()
        rope.apply(pos, q_in, k_in, out_q=q, out_k=k, stream=st)
        v.copy_(qkv[:, (hq + hkv) * d:].unflatten(1, (hkv, d)))
        eng.append_rope(0, 3, rows, kv_len - 1, k, v, st)
        eng.select_pages(0, 3, rows, kv_len, 600, q, top, 1, 2, sel, st)
        eng.attend_selected(0, 3, rows, kv_len, 600, sel, top, q, out, 0.09, st)
    for step in range(steps):
        n_now = [n + step + 1 for n in lens0]
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        kv_len.copy_(torch.tensor(n_now, dtype=torch.int32))
        pos.copy_(kv_len - 1 + far)
        graph.replay()
        torch.cuda.synchronize()
        for s in range(3):
            ks[s].append(_stored(k[s:s + 1], pool))
            vs[s].append(_stored(v[s:s + 1], pool))
        want, mag = rotate64(q_in.double().cpu().numpy(), pos.cpu().numpy(), freq, a, "pairs", False)
        assert (np.abs(q.double().cpu().numpy() - want) <= np.abs(want) * _half_step(dtype) * 1.001 + 2.0 ** -25 + 1e-6 * a * mag).all()
        if step % 5:
            continue
        kk, vv = [np.concatenate(x) for x in ks], [np.concatenate(x) for x in vs]
        got, qd = sel.cpu().numpy(), q.double().cpu().numpy()
        for s, n in enumerate(n_now):
            for h in range(hkv):
                pick = _selection(qd[s, h * 4:(h + 1) * 4], kk[s][:, h], page, n, np.ones(-(-n // page), bool), top, 1, 2)
                assert list(got[s, h]) == pick + [-1] * (top - len(pick)), (step, s, h)

        def visible(b, h, n):
            return np.array([i for p in got[b, h] if p >= 0 for i in range(p * page, min(n, (p + 1) * page))], dtype=int)
        _check_sparse(out, out, q, kk, vv, n_now, hkv, 0.09, dtype, visible, 2.0 ** -17)
    eng.check_kernels()
    eng.close()
