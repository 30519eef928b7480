"""The 8-bit pool where rows of one head differ in size by as much as the types can hold; refused calls that leave nothing behind."""
import math

import numpy as np
import pytest

from tests import cache8_helpers as R
from tests.test_cache8 import _engine, _half_step, _torch_dtype, _weight_step

pytestmark = pytest.mark.gpu


def _values(t, n, d, gap, gen):
    """Rows of size one, or as small as the type has room for below 2^gap of them; sizes differ by up to 4 from row to row."""
    import torch
    x = torch.randint(1, 8, (n, 1, d), generator=gen, device="cuda").float() * torch.randint(0, 2, (n, 1, d), generator=gen, device="cuda").mul(2).sub(1)
    x = x * 2.0 ** torch.randint(0, 3, (n, 1, 1), generator=gen, device="cuda")
    return x * (2.0 ** -24 if t is torch.float16 and gap > 24 else 2.0 ** -8)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gap", [22, 24, 30, 33, 38])
@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("n,n_seq,d,grp", [(100, 1, 128, 4), (1500, 1, 64, 4), (1500, 96, 128, 4), (700, 150, 256, 2), (300, 40, 64, 9)])
def test_values_far_apart(drkv_lib, dtype, gap, where, n, n_seq, d, grp):
    """One value row is 2^gap times the others.  The first head looks at it; to the others its weight is e^-60 (it must leave
    them alone), e^-28 or about 2^-gap (its share is of the size of theirs).  By one warp, by pieces of many, by whole stretches."""
    import torch
    t = _torch_dtype(dtype)
    eng = _engine(hq=grp, hkv=1, d=d, page=16, dtype=dtype, pages=100, seqs=1)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(gap)
    v = _values(t, n, d, gap, g)
    at = {"first": 0, "middle": n // 2 + 3, "last": n - 1}[where]
    v[at] = v[at].abs().clamp(max=float(v.abs().min()) * 2) * 2.0 ** gap * v[at].sign()
    k = torch.randn(n, 1, d, generator=g, device="cuda") * 0.5
    k[:, 0, 0] = 0.0
    k[at] = 0.0
    k[at, 0, 0] = 8.0
    q = torch.randn(n_seq, grp, d, generator=g, device="cuda") * 0.5
    scale = 1.0 / math.sqrt(d)
    far = [60.0, 28.0, gap * math.log(2.0)]
    for b in range(n_seq):
        for h in range(grp):
            q[b, h, 0] = (20.0 if h == 0 else -far[(b + h) % 3]) / (8.0 * scale)
    k, v, q = k.to(t), v.to(t), q.to(t)
    eng.append_rope_chunk(0, 0, 0, n, k, v)
    lens = [n - (i % 7 if where == "first" else 0) for i in range(n_seq)]
    kv_len = torch.tensor(lens, device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 7.0)
    eng.attend_decode(0, n_seq, torch.zeros_like(kv_len), kv_len, n, q, out, scale)
    torch.cuda.synchronize()
    eng.check_kernels()
    ks, vs = (R.stored_values(x.double().cpu().numpy())[:, 0] for x in (k, v))
    got, qd = out.double().cpu().numpy(), q.double().cpu().numpy()
    for b in range(0, n_seq, max(1, n_seq // 8)):
        want, pv, mag = R.attend(qd[b], ks[:lens[b]], vs[:lens[b]], scale)
        tol = R.attend_tolerance(want, pv, mag, _half_step(dtype), _weight_step(dtype))
        err = np.abs(got[b] - want)
        assert (err <= tol).all(), (b, float((err / tol).max()))
    eng.close()


@pytest.mark.parametrize("n,n_seq,d", [(60, 1, 128), (1500, 3, 256), (1300, 120, 64)])
def test_weight_on_a_row_of_nothing(drkv_lib, n, n_seq, d):
    """The key with nearly all the weight has zeros for values, or values 2^100 below the rest: the others make the result,
    down to weights that fp32 does not hold beside 1; and rows above 2^100."""
    import torch
    eng = _engine(hq=4, hkv=1, d=d, page=16, dtype="bf16", pages=100, seqs=1)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = (torch.randn(n, 1, d, generator=g, device="cuda") for _ in range(2))
    k[:, 0, 0] = 0.0
    k[n // 3] = 0.0
    k[n // 3, 0, 0] = 8.0
    q = torch.randn(n_seq, 4, d, generator=g, device="cuda")
    scale = 1.0 / math.sqrt(d)
    for h, x in enumerate((30.0, 60.0, 80.0, 95.0)):
        q[:, h, 0] = x / (8.0 * scale)
    kv_len = torch.full((n_seq,), n, device="cuda", dtype=torch.int32)
    for sink, rest in ((0.0, 1.0), (2.0 ** -100, 1.0), (1.0, 2.0 ** 110), (2.0 ** -60, 2.0 ** 60)):
        vv = v * rest
        vv[n // 3] = v[n // 3] * sink
        k16, v16, q16 = k.bfloat16(), vv.bfloat16(), q.bfloat16()
        eng.append_rope_chunk(0, 0, 0, n, k16, v16)
        out = torch.full_like(q16, 7.0)
        eng.attend_decode(0, n_seq, torch.zeros_like(kv_len), kv_len, n, q16, out, scale)
        torch.cuda.synchronize()
        ks, vs = (R.stored_values(x.double().cpu().numpy())[:, 0] for x in (k16, v16))
        got, qd = out.double().cpu().numpy(), q16.double().cpu().numpy()
        for b in range(0, n_seq, max(1, n_seq // 5)):
            want, pv, mag = R.attend(qd[b], ks, vs, scale)
            # attend_tolerance's terms without its floor for fp16 (taking 2^-25 off its sum again would leave multiples of
            # 2^-77, results here go down to 2^-130); below bf16's normal range results may vanish
            tol = np.abs(want) * _half_step("bf16") + 2.0 ** -126 + pv * (_weight_step("bf16") + 2.0 ** -18 + 2 * 2.0 ** -20 * mag)
            err = np.abs(got[b] - want)
            assert (err <= tol).all(), (sink, rest, b, float((err / tol).max()))
    eng.check_kernels()
    eng.close()


@pytest.mark.parametrize("n,d,grp", [(2, 128, 4), (5, 64, 7), (40, 256, 2), (900, 128, 8)])
def test_weights_of_bf16_outputs(drkv_lib, n, d, grp):
    """Weights of up to eight heads a group go into the product with 22 bits: what is off is the output's rounding."""
    import torch
    eng = _engine(hq=grp, hkv=1, d=d, page=16, dtype="bf16", pages=64, seqs=1)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = (torch.randn(n, 1, d, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(150, grp, d, generator=g, device="cuda").bfloat16()
    eng.append_rope_chunk(0, 0, 0, n, k, v)
    kv_len = torch.full((150,), n, device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 7.0)
    eng.attend_decode(0, 150, torch.zeros_like(kv_len), kv_len, n, q, out, 0.5 / math.sqrt(d))
    torch.cuda.synchronize()
    ks, vs = (R.stored_values(x.double().cpu().numpy())[:, 0] for x in (k, v))
    got, qd = out.double().cpu().numpy(), q.double().cpu().numpy()
    for b in range(150):
        want, pv, mag = R.attend(qd[b], ks, vs, 0.5 / math.sqrt(d))
        assert (np.abs(got[b] - want) <= R.attend_tolerance(want, pv, mag, _half_step("bf16"), 2.0 ** -21)).all(), b
    eng.check_kernels()
    eng.close()


def test_refused_steps_leave_the_cache(drkv_lib):
    """A decode step with a bad pointer writes no token and widens no bounds, by batch and by plan."""
    import torch
    from deusridet_b200 import DrkvError, capi
    eng = _engine(hq=8, hkv=2, d=128, page=16, dtype="bf16", pages=8, seqs=1)
    eng.page_bounds_enable()
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 20)
    eng.set_seq_len(0, 20)
    eng.sync_block_table()
    eng.pool_tensor().zero_()
    eng.page_bounds_enable()
    x = torch.ones(2, 8, 128, device="cuda", dtype=torch.bfloat16)
    rows, kv_len = torch.zeros(1, device="cuda", dtype=torch.int32), torch.full((1,), 20, device="cuda", dtype=torch.int32)
    eng.plan_decode([0], [20])
    before = [t.clone() for t in (eng.pool_tensor(), *eng.page_bounds())]
    off = x.data_ptr() + 4
    for ptrs in ((x, x, x, off), (x, x, off, x), (off, x, x, x), (x, off, x, x)):
        for call in (lambda: eng.append_attend_decode(0, 1, rows, kv_len, 20, *ptrs, 1.0), lambda: eng.append_attend_decode_planned(0, *ptrs, 1.0)):
            with pytest.raises(DrkvError) as err:
                call()
            assert err.value.code == capi.ERR_INVALID
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(before, (eng.pool_tensor(), *eng.page_bounds())))
    eng.append_attend_decode(0, 1, rows, kv_len, 20, x, x, x, torch.empty_like(x), 1.0)
    torch.cuda.synchronize()
    assert not torch.equal(before[0], eng.pool_tensor()) and not torch.equal(before[1], eng.page_bounds()[0])
    eng.close()


def test_lists_over_one_vast_page(drkv_lib):
    """A list counts whole pages: 1 024 sequences of twenty keys on a page of 2^25 tokens are 2^31 groups of 16, more than a
    launch counts."""
    import torch
    from deusridet_b200 import PagedKVEngine
    eng = PagedKVEngine(num_layers=1, num_q_heads=1, num_kv_heads=1, head_dim=64, page_size=2 ** 25, dtype="f16", rotary_dim=0,
                        max_pages=4, max_seqs=1, max_pages_per_seq=1, device=0)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, 20)
    eng.set_seq_len(0, 20)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(20, 1, 64, generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn(1024, 1, 64, generator=g, device="cuda").half()
    eng.append_rope_chunk(0, 0, 0, 20, k, v)
    kv_len = torch.full((1024,), 20, device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 7.0)
    zeros = torch.zeros_like(kv_len)
    eng.attend_selected(0, 1024, zeros, kv_len, 20, zeros, 1, q, out, 0.125)
    torch.cuda.synchronize()
    eng.check_kernels()
    kd, vd, qd, got = (x.double().cpu().numpy() for x in (k[:, 0], v[:, 0], q[:, 0], out[:, 0]))
    want, pv, mag = R.attend(qd, kd, vd, 0.125)
    assert (np.abs(got - want) <= R.attend_tolerance(want, pv, mag, _half_step("f16"), 2.0 ** -21)).all()
    eng.close()


def test_smallest_keys_and_large_queries(drkv_lib):
    """Keys whose exponent byte is 0 (their row's largest is at most 448 * 2^-127) against queries that make scores of them."""
    import torch
    n, d = 40, 64
    eng = _engine(hq=2, hkv=1, d=d, page=16, dtype="bf16", pages=8, seqs=1)
    eng.seq_create()
    assert eng.ensure_blocks_for_range(0, 0, n)
    eng.set_seq_len(0, n)
    eng.sync_block_table()
    g = torch.Generator(device="cuda").manual_seed(3)
    k = (torch.randint(1, 28, (n, 1, d), generator=g, device="cuda") * 2.0 ** -126).bfloat16()
    v = torch.randn(n, 1, d, generator=g, device="cuda").bfloat16()
    q = (torch.randn(1, 2, d, generator=g, device="cuda") * 2.0 ** 119).bfloat16()
    eng.append_rope_chunk(0, 0, 0, n, k, v)
    kv_len = torch.full((1,), n, device="cuda", dtype=torch.int32)
    out = torch.full_like(q, 7.0)
    eng.attend_decode(0, 1, kv_len - n, kv_len, n, q, out, 0.25)
    torch.cuda.synchronize()
    e = R.quantise(k.double().cpu().numpy())[1]
    assert (e == -127).all()
    ks, vs = (R.stored_values(x.double().cpu().numpy())[:, 0] for x in (k, v))
    want, pv, mag = R.attend(q[0].double().cpu().numpy(), ks, vs, 0.25)
    assert (mag > 1).all()
    err = np.abs(out[0].double().cpu().numpy() - want)
    assert (err <= R.attend_tolerance(want, pv, mag, _half_step("bf16"), _weight_step("bf16"))).all()
    eng.close()
