"""Page scores at the ends of fp32."""
import pytest

from tests.test_page_sparse import _engine, _start

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_size,k_size,order", [(2.0 ** 100, 2.0 ** 100, "first"), (2.0 ** 30, 2.0 ** 120, "first"), (2.0 ** 100, 1.0, "best"),
                                                 (2.0 ** -60, 2.0 ** 60, "best"), (2.0 ** -100, 2.0 ** -100, "first")])
def test_scores_beyond_fp32_tie(drkv_lib, q_size, k_size, order):
    """Pages of rising keys: the last are the best, unless every score is infinite, or too small for any."""
    import torch
    page, n_pages, d, top = 16, 40, 64, 5
    eng = _engine(None, 2, 1, d, page, "bf16", n_pages, 1, n_pages)
    eng.page_bounds_enable()
    _start(eng, [page * n_pages])
    k = torch.ones(n_pages, page, 1, d, device="cuda") * torch.arange(1, n_pages + 1, device="cuda").view(-1, 1, 1, 1)
    k = (k * k_size).bfloat16().view(-1, 1, d)
    eng.append_rope_chunk(0, 0, 0, page * n_pages, k, k)
    q = torch.full((1, 2, d), q_size, device="cuda").bfloat16()
    n = torch.full((1,), page * n_pages, device="cuda", dtype=torch.int32)
    sel = torch.full((1, 1, top), 9, device="cuda", dtype=torch.int32)
    eng.select_pages(0, 1, n - page * n_pages, n, page * n_pages, q, top, 0, 0, sel)
    assert sel.flatten().tolist() == (list(range(top)) if order == "first" else list(range(n_pages - top, n_pages)))
    eng.check_kernels()
    eng.close()


@pytest.mark.parametrize("pool,n_seq,hkv,d,page", [(None, 64, 8, 64, 16), ("e4m3", 100, 3, 128, 32)])
def test_bounds_of_the_step_are_in_its_scores(drkv_lib, pool, n_seq, hkv, d, page):
    """Append, selection and attention back to back in one graph, keys of every step of another size: what a step writes is
    what its selection sees, as when every launch is waited for."""
    import torch
    n0, steps, top = 150, 30, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    size = torch.exp2(torch.randint(-2, 6, (steps, n_seq, hkv, 1), generator=g, device="cuda").float())
    ks = (torch.randn(steps, n_seq, hkv, d, generator=g, device="cuda") * size).bfloat16()
    qs = torch.randn(steps, n_seq, 4 * hkv, d, generator=g, device="cuda").bfloat16()
    first = torch.randn(n_seq, n0, hkv, d, generator=g, device="cuda").bfloat16()
    per = -(-(n0 + steps) // page)
    seen = []
    for captured in (True, False):
        eng = _engine(pool, 4 * hkv, hkv, d, page, "bf16", n_seq * per, n_seq, per)
        eng.page_bounds_enable()
        _start(eng, [n0] * n_seq, room=n0 + steps)
        for s in range(n_seq):
            eng.append_rope_chunk(0, s, 0, n0, first[s], first[s])
        rows = torch.arange(n_seq, device="cuda", dtype=torch.int32)
        pos, kv_len, k, q = torch.zeros_like(rows), torch.zeros_like(rows), torch.zeros_like(ks[0]), torch.zeros_like(qs[0])
        sel, out = torch.zeros(n_seq, hkv, top, device="cuda", dtype=torch.int32), torch.zeros_like(q)
        wait = (lambda: None) if captured else torch.cuda.synchronize

        def step(st):
            eng.append_rope(0, n_seq, rows, pos, k, k, st)
            wait()
            eng.select_pages(0, n_seq, rows, kv_len, n0 + steps, q, top, 0, 0, sel, st)
            wait()
            eng.attend_selected(0, n_seq, rows, kv_len, n0 + steps, sel, top, q, out, 0.1, st)
        torch.cuda.synchronize()
        if captured:
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=side):
                step(torch.cuda.current_stream())
        for i in range(steps):
            pos.fill_(n0 + i)
            kv_len.fill_(n0 + i + 1)
            k.copy_(ks[i])
            q.copy_(qs[i])
            torch.cuda.synchronize()
            graph.replay() if captured else step(torch.cuda.current_stream())
            torch.cuda.synchronize()
            seen.append((sel.clone(), out.clone()))
        eng.check_kernels()
        eng.close()
    for (a, x), (b, y) in zip(seen[:steps], seen[steps:]):
        assert torch.equal(a, b) and torch.equal(x.view(torch.int16), y.view(torch.int16))
