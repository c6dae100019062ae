"""The row limit of kv_plan on the GPU, with results written out by hand."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("rows,want,num,n_new,held,n_free", [
    (10, [8, 5, 2], 3, [8, 0, 0], [1, 0, 0], 2),            # the second does not fit, and the third waits behind it
    (10, [8, 2, 5], 3, [8, 2, 0], [1, 1, 0], 1),            # exactly full
    (10, [30, 1, 1], 3, [0, 0, 0], [0, 0, 0], 3),           # more than a step has rows for holds up all
    (10, [-1, 11, 1], 3, [0, 0, 0], [0, 0, 0], 3),
    (10, [11, 0, 0], 3, [0, 0, 0], [0, 0, 0], 3),
    (100, [33, 60, 7], 3, [33, 0, 0], [2, 0, 0], 1),        # pages: 2 of 3, then 2 more than are left; so has the third
    (40, [33, 300, 7], 3, [33, 0, 7], [2, 0, 1], 0),        # what outgrows its table (128) is not counted, neither pages nor rows
    (0, [1, 1, 1], 3, [0, 0, 0], [0, 0, 0], 3)])
def test_rows_that_do_not_fit(gpu, rows, want, num, n_new, held, n_free):
    from tokamak_amd import attn
    cache = attn.KvCache.empty(3, 4, num, 1, 64, page=32, device=gpu)
    pages = attn.KvPages.all_free(cache)
    plan = attn.kv_plan(cache, pages, i32(want, gpu), rows=rows, start=i32([0, 0, 0], gpu))
    assert plan.n_new.tolist() == n_new and cache.kv_len.tolist() == n_new
    assert pages.held.tolist() == held and pages.n_free.tolist() == [n_free]
    assert plan.row_start.tolist() == [0, n_new[0], n_new[0] + n_new[1], sum(n_new)]
    assert plan.seq.tolist() == [b for b, n in enumerate(n_new) for _ in range(n)] + [-1] * (rows - sum(n_new))


def test_what_does_not_lack_pages_waits_for_rows(gpu):
    """Sequences that hold their pages already wait behind one whose rows do not fit, and go on past one whose pages are
    missing."""
    from tokamak_amd import attn
    cache = attn.KvCache.empty(3, 4, 2, 1, 64, page=32, device=gpu)
    pages = attn.KvPages.all_free(cache)
    assert attn.kv_plan(cache, pages, i32([0, 3, 4], gpu), rows=10).n_new.tolist() == [0, 3, 4]
    assert attn.kv_plan(cache, pages, i32([11, 1, 1], gpu), rows=10).n_new.tolist() == [0, 1, 1]      # no page is free
    assert cache.kv_len.tolist() == [0, 4, 5]
    assert attn.kv_plan(cache, pages, i32([0, 11, 1], gpu), rows=10).n_new.tolist() == [0, 0, 0]
    assert cache.kv_len.tolist() == [0, 4, 5] and pages.held.tolist() == [0, 1, 1]
