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
