"""Page ids that are not the pool's, and a stack with too few pages."""
import numpy as np
import pytest
import torch

from oracle.tokens import POOL_EXHAUSTED, TokenPoolModel
from parakeet_b200 import TokenKVPool, _lib
from test_gpu_tokens import check_step, check_tables, grow, i32

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("trees", [True, False])
@pytest.mark.parametrize("batch", [3, 70])
@pytest.mark.parametrize("bad", [-1, -5, 40, 2 ** 27 + 1, 2 ** 30, 2 ** 31 - 1])
def test_a_bad_page_is_reported_by_the_step_that_reads_it(bad, batch, trees):
    """Its rows have no place (slot_map -1): append and acceptance leave them out."""
    pool = TokenKVPool(1, 2, 2, 64, batch, 64, num_pages=max(40, 2 * batch), page_size=16, device=DEV)
    bad = bad if bad != 40 else pool.num_pages
    slots = np.arange(batch)
    model = TokenPoolModel(batch, 64, pool.num_pages, 16)
    grow(pool, model, slots, np.full(batch, 10))
    pool.page_table[1, 0] = bad
    n = np.full(batch, 9)             # six rows in the page held, three in a new one
    rows = int(n.sum())
    parents = np.tile(np.arange(-1, 8), batch)
    step = pool.begin_step(i32(slots), i32(n), rows, i32(parents) if trees else None)
    assert pool.read_error() == _lib.PK_DEV_BAD_PAGE
    got = step.slot_map.cpu().numpy().reshape(batch, 9)
    assert (got[1, :6] == -1).all()
    got = np.delete(got, 1, 0)
    assert (got >= 0).all() and len(set(got.ravel())) == got.size
    pool.error.zero_()
    before = pool.kv.clone()
    k = torch.ones(rows, 2, 64, dtype=torch.bfloat16, device=DEV)
    pool.append(0, k, k, step)
    pool.end_step(step, i32(n - 1))
    table = pool.page_table.cpu().numpy()
    changed = set((pool.kv != before).flatten(1).any(1).nonzero()[:, 0].tolist())
    assert changed <= set(table[table >= 0].tolist())
    assert pool.lengths.tolist() == [19] * batch


@pytest.mark.parametrize("bad", [-1, 2 ** 24])
def test_a_move_of_a_bad_page_touches_no_other_requests_rows(bad):
    """Request 0's kept rows lie in a page that is none; request 1, whose first page is
    page 0, moves an accepted row into that page's first row in the same launch."""
    layers = 96
    order = np.array([3, 2, 1, 4, 5, 0])           # taken from the end: request 1 first
    for _ in range(10):
        pool = TokenKVPool(layers, 8, 8, 128, 2, 128, num_pages=6, page_size=64, device=DEV,
                           page_order=order)
        slots, n = i32([1, 0]), i32([64, 64])
        # the path 1, 2, .. 63 of every tree: each row moves up by one
        parents = i32(np.tile(np.concatenate([[-1, -1], np.arange(1, 63)]), 2))
        step = pool.begin_step(slots, n, 128, parents)
        assert pool.page_table[1, 0].item() == 0
        k = torch.randn(layers, 128, 8, 128, device=DEV).to(torch.bfloat16)
        pool.append(0, k, k, step)
        step.slot_map[64:] = bad << 6 if bad > 0 else -1
        pool.end_step(step, i32([63, 63]))
        assert pool.read_error() == _lib.PK_DEV_BAD_PAGE
        for plane in (0, 1):
            assert torch.equal(pool.kv[0, :, plane, :, :63], k[:, 1:64].transpose(1, 2))


@pytest.mark.parametrize("batch", [4, 80])
def test_requests_behind_one_that_found_too_few_pages_get_none(batch):
    """Pages go out in batch order and nobody overtakes: with 3 pages left and needs of
    4, 1, 0 and 1, only the request that needs none is served, and the pages stay."""
    pool = TokenKVPool(1, 1, 1, 64, batch, 128, num_pages=batch + 3, page_size=16, device=DEV)
    model = TokenPoolModel(batch, 128, batch + 3, 16)
    grow(pool, model, np.arange(batch), np.full(batch, 10))
    n = np.ones(batch, int)
    n[:4] = [60, 7, 1, 7]           # 4, 1, 0 and 1 more pages
    counts, rows = i32(n), int(n.sum())
    step = pool.begin_step(i32(np.arange(batch)), counts, rows)
    ref = model.begin_step(np.arange(batch), n, rows)
    check_step(step, ref)
    assert step.context.tolist()[:4] == [-1, -1, 10, -1]
    assert all(c == 10 for c in step.context.tolist()[4:])
    assert pool.read_error() == POOL_EXHAUSTED and int(pool.free_count) == 3
    model.error = POOL_EXHAUSTED
    check_tables(pool, model)
    # without the first one the others are
    pool.end_step(step, i32(np.full(batch, -1)))
    step = pool.begin_step(i32(np.arange(1, batch)), i32(n[1:]), int(n[1:].sum()))
    assert all(c == 10 for c in step.context.tolist()) and int(pool.free_count) == 1


@pytest.mark.parametrize("kind", [list, np.array, lambda o: torch.tensor(o)])
@pytest.mark.parametrize("order", [[0, 1, 2, 2], [0, 1, 2, 4], [-1, 0, 1, 2], [0, 1, 2], [0, 1, 2, 3, 3]])
def test_an_order_that_does_not_list_every_page_once_is_refused(order, kind):
    """Two requests would share a page."""
    args = dict(num_layers=1, num_heads=1, num_kv_heads=1, head_dim=64, num_slots=2, max_tokens=32,
                num_pages=4, page_size=16, device=DEV)
    with pytest.raises(ValueError, match="every page once"):
        TokenKVPool(**args, page_order=kind(order))
    pool = TokenKVPool(**args, page_order=kind([2, 0, 3, 1]))
    step = pool.begin_step(i32([0]), i32([20]), 20)
    pool.end_step(step, i32([19]))
    with pytest.raises(ValueError, match="every page once"):
        pool.reset(kind(order))
    assert pool.lengths.tolist() == [20, 0] and pool.page_table.tolist()[0] == [1, 3]
    pool.reset(kind([0, 1, 2, 3]))
    assert pool.free_pages.tolist() == [0, 1, 2, 3] and pool.lengths.tolist() == [0, 0]


@pytest.mark.parametrize("trees", [True, False])
@pytest.mark.parametrize("cut", ["release", "shorter", "reset"])
def test_a_step_is_not_ended_over_pages_given_back(cut, trees):
    """A request cut while its step is open (a client that left) keeps nothing of the
    step: its length never passes the pages it holds.  The others are ended."""
    pool = TokenKVPool(2, 2, 2, 64, 3, 200, page_size=16, device=DEV)
    slots, model = np.arange(3), TokenPoolModel(3, 200, pool.num_pages, 16)
    grow(pool, model, slots, np.array([30, 40, 50]))
    n = i32([20, 20, 20])
    # the path 1, 2, .. 19: rows are moved
    parents = i32(np.tile(np.concatenate([[-1, -1], np.arange(1, 19)]), 3)) if trees else None
    step = pool.begin_step(i32(slots), n, 60, parents)
    k = torch.randn(2, 60, 2, 64, device=DEV).to(torch.bfloat16)
    pool.append(0, k, k, step)
    if cut == "reset":
        pool.reset()
    else:
        pool.truncate(i32([1]), i32([0 if cut == "release" else 10]))
    before, held = pool.kv.clone(), pool.held.tolist()
    pool.end_step(step, i32([19, 19, 19]))
    kept = 19 if trees else 20
    assert pool.read_error() == _lib.PK_DEV_BAD_COUNT
    assert pool.lengths.tolist() == {"release": [30 + kept, 0, 50 + kept],
                                     "shorter": [30 + kept, 10, 50 + kept], "reset": [0, 0, 0]}[cut]
    assert pool.held.tolist() == held
    left = step.slot_map[20:40].long()
    for plane in (0, 1):
        assert torch.equal(pool.kv[left // 16, :, plane, :, left % 16],
                           before[left // 16, :, plane, :, left % 16])
    # the request goes on
    pool.error.zero_()
    start = pool.lengths[1].item()
    step = pool.begin_step(i32([1]), i32([3]), 3)
    assert step.context.tolist() == [start]
    pool.end_step(step, i32([2]))
    assert pool.lengths[1].item() == start + 3 and pool.read_error() == 0
