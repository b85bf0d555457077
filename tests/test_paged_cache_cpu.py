"""CPU tests of PagedCache's bookkeeping (pages, lengths, refusals): host work, on CPU tensors."""
import pytest
import torch


@pytest.fixture(scope="module")
def PagedCache():
    import __graft_entry__
    __graft_entry__._load_builder().build()
    from fourierattention_b200 import PagedCache as P
    return P


def make(P, **kw):
    d = dict(num_layers=1, num_kv_heads=1, head_dim=64, batch=3, max_tokens=40, page_size=16, device="cpu")
    d.update(kw)
    return P(**d)


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(page_size=20), dict(head_dim=80), dict(batch=0), dict(max_tokens=0),
                                dict(num_pages=0), dict(dtype=torch.float32)])
def test_refused_sizes(PagedCache, kw):
    with pytest.raises(ValueError):
        make(PagedCache, **kw)


def test_steps_take_pages_and_keep_tables(PagedCache):
    c = make(PagedCache)
    assert c.num_pages == 12 and c.max_pages == 3
    c.plan([17, 0, 16])
    c.begin_step(1, 33)
    assert c.lengths == [17, 0, 16] and c.kv_lens.tolist() == [17, 0, 16] and c.cu_seqlens.tolist() == [0, 17, 17, 33]
    used = c._pages[0] + c._pages[2]
    assert [len(p) for p in c._pages] == [2, 0, 1] and len(set(used)) == 3
    assert c.page_table[0, :2].tolist() == c._pages[0] and c.page_table[2, 0] == c._pages[2][0]
    c.begin_step(3, 1)
    assert c.cu_seqlens is None and c.kv_lens.tolist() == [18, 1, 17] and [len(p) for p in c._pages] == [2, 1, 2]
    c.begin_step(3, 2)
    assert c.cu_seqlens.tolist() == [0, 2, 4, 6] and c.get_seq_length() == 20
    c.truncate(0, 3)
    assert c.lengths[0] == 3 and len(c._pages[0]) == 1 and c.kv_lens.tolist() == [3, 3, 19]
    h = torch.arange(12.0).view(1, 6, 2)
    assert c.last_rows(h)[:, 0].tolist() == [[2, 3], [6, 7], [10, 11]]
    c.reset()
    assert sorted(c._free) == list(range(12))


def test_refusals_leave_the_state(PagedCache):
    c = make(PagedCache, num_pages=3)
    with pytest.raises(ValueError):
        c.plan([1, 2])
    with pytest.raises(ValueError):
        c.plan([0, 0, 0])
    with pytest.raises(ValueError):
        c.begin_step(2, 1)
    c.plan([5, 5, 5])
    with pytest.raises(ValueError):
        c.begin_step(3, 5)
    c.begin_step(1, 15)
    with pytest.raises(ValueError, match="holds"):
        c.begin_step(3, 36)
    with pytest.raises(RuntimeError, match="pages"):
        c.begin_step(3, 12)
    assert c.lengths == [5, 5, 5] and c.kv_lens.tolist() == [5, 5, 5] and c._free == []
    with pytest.raises(ValueError):
        c.truncate(0, 6)
    with pytest.raises(NotImplementedError):
        c.update(None, None, 0)


def test_prefix(PagedCache):
    c = make(PagedCache)
    with pytest.raises(RuntimeError):
        c.share_prefix(0)
    c.plan([20, 0, 0])
    c.begin_step(1, 20)
    ids = list(c._pages[0])
    c.share_prefix(0)
    assert c.prefix_len == 20 and c.prefix_pages.tolist() == ids and c.lengths == [0, 0, 0] and c.kv_lens.tolist() == [0, 0, 0]
    c.begin_step(3, 4)
    assert not set(ids) & {p for q in c._pages for p in q} and c.get_seq_length() == 24
    with pytest.raises(RuntimeError):
        c.share_prefix(0)
    c.reset()
    assert sorted(c._free) == list(range(12)) and c.prefix_pages is None
    c.plan([1, 1, 0])
    c.begin_step(1, 2)
    with pytest.raises(RuntimeError, match="empty"):
        c.share_prefix(0)


@pytest.mark.parametrize("new", [[5, 0, 3], [0, 2, 0], [0, 0, 1], [2, 1, 0]])
def test_last_rows_of_idle_sequences(PagedCache, new):
    """A sequence without new tokens has no last row: it gets zeros, not a neighbour's (nor its NaN)."""
    c = make(PagedCache)
    c.plan(new)
    c.begin_step(1, sum(new))
    h = torch.arange(1.0, 1 + 2 * sum(new)).view(1, -1, 2)
    h[0, 0, 0] = float("nan")
    got, at = c.last_rows(h), 0
    assert tuple(got.shape) == (3, 1, 2)
    for b, n in enumerate(new):
        at += n
        want = h[0, at - 1] if n else torch.zeros(2)
        assert torch.equal(got[b, 0].nan_to_num(-1.0), want.nan_to_num(-1.0))


def test_a_cancelled_step_leaves_no_trace(PagedCache):
    c = make(PagedCache)
    with pytest.raises(RuntimeError, match="no step"):
        c.cancel_step()
    c.plan([17, 0, 16])
    c.begin_step(1, 33)
    pages, free = [list(p) for p in c._pages], sorted(c._free)
    for plan in ([3, 20, 0], None):
        if plan:
            c.plan(plan)
        c.begin_step(*((1, 23) if plan else (3, 1)))
        c.cancel_step()
        assert c.lengths == [17, 0, 16] and c.kv_lens.tolist() == [17, 0, 16] and c.planned == plan
        assert c._pages == pages and sorted(c._free) == free
        c._plan = None
    with pytest.raises(RuntimeError, match="no step"):
        c.cancel_step()
    c.begin_step(3, 1)
    assert c.kv_lens.tolist() == [18, 1, 17] and c.page_table[1, 0] == c._pages[1][0]
    c.truncate(0, 4)                                # what was done since cannot be taken back with it
    with pytest.raises(RuntimeError, match="no step"):
        c.cancel_step()


def test_what_a_captured_step_reads_stays_in_place(PagedCache):
    """Lengths, table and token offsets of a later step are where those of an earlier one were."""
    c = make(PagedCache)
    c.begin_step(3, 2)
    where = lambda: (c.kv_lens.data_ptr(), c.page_table.data_ptr(), c.cu_seqlens.data_ptr())
    first, held = where(), c.cu_seqlens
    c.begin_step(3, 1)
    assert c.cu_seqlens is None
    c.plan([4, 0, 2])
    c.begin_step(1, 6)
    assert where() == first and held.tolist() == [0, 4, 4, 6]
    c.reset()
    c.begin_step(3, 3)
    assert where() == first and held.tolist() == [0, 3, 6, 9]
