"""Token pools on the GPU: page tables, slot maps, masks, appended and kept rows
bit for bit against the numpy model, attention against float64.

Attention tolerance, per element, from the kernel's arithmetic: with A the
weighted mean of |v| and u = 2^-24, a score is off by at most scale * (dh + 2) *
u * sum |q||k| =: d, the maximum's product by as much again, exp2 by 2^-22, and
a weight thus by 2 d + 2^-21 relative (numerator and sum: twice that); adding n
keys adds n * u.  bf16 rounds each weight for the product and the result: 2^-8
A + 2^-8 |out| (bf16's half step is 2^-8), f32 the result: 2^-23 |out|."""
import numpy as np
import pytest
import torch

from oracle.tokens import TokenPoolModel, tree_attention
from parakeet_b200 import TokenKVPool, _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def random_tree(rng, counts, rows):
    parents = np.full(rows, -1, np.int32)
    r = 0
    for n in counts:
        for j in range(n):
            parents[r + j] = j - 1 if j and rng.random() < 0.6 else rng.integers(-1, j) if j else -1
        r += n
    return parents


def check_tables(pool, model):
    assert np.array_equal(pool.page_table.cpu().numpy(), model.table)
    assert np.array_equal(pool.lengths.cpu().numpy(), model.lengths)
    assert np.array_equal(pool.held.cpu().numpy(), model.held)
    n = int(pool.free_count.item())
    assert pool.free_pages.cpu().numpy()[:n].tolist() == [int(p) for p in model.stack]
    assert pool.read_error() == model.error


def check_step(step, ref):
    for name in ("row_start", "context", "row_request", "positions", "slot_map", "masks"):
        got, want = getattr(step, name), ref[name]
        if want is None:
            assert got is None
        else:
            assert np.array_equal(got.cpu().numpy(), want), name


def bound(out, ref, mean_abs, reach, dtype, n, dh):
    u = 2.0 ** -24
    d = reach[..., None] * (dh + 2) * u
    tol = mean_abs * (2 * (2 * d + 2.0 ** -21) + n * u)
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * mean_abs + 2.0 ** -8 * np.abs(ref) * 1.01
    else:
        tol = tol + 2.0 ** -23 * np.abs(ref)
    err = np.abs(out - ref)
    assert not np.isnan(err).any()
    assert (err <= tol).all(), f"{(err > tol).sum()} off, worst {np.max(err / tol):.3g} of the bound"


def grow(pool, model, slots, lengths):
    step = pool.begin_step(i32(slots), i32(lengths), int(np.sum(lengths)))
    ref = model.begin_step(slots, lengths, int(np.sum(lengths)))
    check_step(step, ref)
    pool.end_step(step, i32(np.asarray(lengths) - 1))
    model.end_step(ref, np.asarray(lengths) - 1)
    check_tables(pool, model)


@pytest.mark.parametrize("page,slots,trees,big", [(8, 5, True, False), (16, 70, True, True),
                                                  (32, 4, False, False), (16, 90, False, True)])
def test_tables_churn(page, slots, trees, big):
    """Random requests join, draft, keep a path, are cut and released; some are
    refused (no pages, bad slot, slot twice, count out of range, bad parents).
    More than 64 requests take the two-launch path."""
    rng = np.random.default_rng(page + slots)
    max_tokens, pages = 300, slots * 6
    order = rng.permutation(pages)
    pool = TokenKVPool(1, 4, 2, 64, slots, max_tokens, num_pages=pages, page_size=page, device=DEV,
                       page_order=order)
    model = TokenPoolModel(slots, max_tokens, pages, page, order)
    check_tables(pool, model)
    for it in range(25):
        B = int(rng.integers(66 if big else 1, slots + 1))
        s = rng.permutation(slots)[:B].astype(np.int32)
        n = rng.integers(0, 65 if trees else 120, B).astype(np.int32)
        if it % 5 == 1:
            s[int(rng.integers(B))] = -1 if it % 2 else slots
        if it % 5 == 2 and B > 1:
            s[-1] = s[0]
        if it % 5 == 3:
            n[int(rng.integers(B))] = -3 if it % 2 else 400
        total = int(np.maximum(n, 0).sum())
        rows = max(total + int(rng.integers(0, 9)) - (4 if it % 7 == 4 else 0), 0)
        parents = None
        if trees:
            parents = random_tree(rng, np.maximum(n, 0), max(rows, total))[:rows]
            if it % 6 == 5 and rows:
                parents[int(rng.integers(rows))] = 64
        step = pool.begin_step(i32(s), i32(n), rows, None if parents is None else i32(parents))
        ref = model.begin_step(s, n, rows, parents)
        check_step(step, ref)
        last = np.array([rng.integers(-1, max(x, 0)) if x > 0 else -1 for x in n], np.int32)
        if it % 8 == 6:
            last[0] = 64
        pool.end_step(step, i32(last))
        model.end_step(ref, last)
        check_tables(pool, model)
        who = rng.permutation(slots)[: int(rng.integers(1, slots + 1))].astype(np.int32)
        cut = np.where(rng.random(len(who)) < 0.4, 0,
                       (model.lengths[who] * rng.random(len(who))).astype(np.int32)).astype(np.int32)
        if it % 4 == 3:
            cut[0] = model.lengths[who[0]] + 1
        pool.truncate(i32(who), i32(cut))
        model.truncate(who, cut)
        check_tables(pool, model)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,heads,dh,layers", [(8, 1, 64, 3), (16, 4, 128, 1)])
def test_append_and_keep(dtype, page, heads, dh, layers):
    """Rows land at their slots (strided slices of a wider buffer, all layers in
    one call or one by one), the kept path moves behind the context in every
    layer, and nothing else of the pool changes."""
    rng = np.random.default_rng(dh)
    slots, pages = 9, 80
    order = rng.permutation(pages)
    pool = TokenKVPool(layers, heads, heads, dh, slots, 120, num_pages=pages, page_size=page,
                       dtype=dtype, device=DEV, page_order=order)
    pool.kv.copy_(torch.randn(pool.kv.shape, device=DEV))
    as_np = lambda t: t.float().cpu().numpy()   # noqa: E731
    model = TokenPoolModel(slots, 120, pages, page, order, kv=as_np(pool.kv).copy())
    for it in range(6):
        B = int(rng.integers(1, slots + 1))
        s = rng.permutation(slots)[:B]
        n = rng.integers(0, 20, B)
        rows = int(n.sum()) + 3
        parents = random_tree(rng, n, rows)
        step = pool.begin_step(i32(s), i32(n), rows, i32(parents))
        ref = model.begin_step(s, n, rows, parents)
        wide = torch.randn(layers, rows, 3 * heads * dh, device=DEV).to(dtype)
        k, v = wide[..., heads * dh:2 * heads * dh], wide[..., 2 * heads * dh:]
        if it % 2:
            pool.append(0, k, v, step)
        else:
            for layer in range(layers):
                pool.append(layer, k[layer], v[layer], step)
        for layer in range(layers):
            model.append(layer, as_np(k[layer]).reshape(rows, heads, dh),
                         as_np(v[layer]).reshape(rows, heads, dh), ref)
        assert np.array_equal(as_np(pool.kv), model.kv)
        last = np.array([rng.integers(-1, x) for x in n])
        pool.end_step(step, i32(last))
        model.end_step(ref, last)
        check_tables(pool, model)
        assert np.array_equal(as_np(pool.kv), model.kv)


CASES = [
    # (page, heads, kv heads, dh, context lengths, new tokens, tree)
    (16, 8, 8, 64, [300], [1], True),                       # a single token
    (16, 2, 2, 64, [0], [1], True),                         # the very first token
    (8, 4, 2, 64, [0, 1, 7, 8, 63, 64, 65], [1, 2, 3, 4, 5, 6, 7], True),
    (16, 8, 8, 64, [37, 0, 129, 250], [13, 64, 0, 1], True),
    (32, 16, 4, 128, [100, 31, 64], [16, 9, 33], True),     # row tiles of 64, a ragged last one
    (64, 5, 1, 128, [70, 5], [12, 64], True),               # a group of 5: rows not a power of two
    (256, 2, 1, 64, [500, 255], [40, 3], True),             # pages longer than a tile
    (16, 4, 4, 128, [2100, 17, 900], [7, 2, 20], True),     # keys split over CTAs and joined
    (16, 8, 2, 64, [1500], [64], True),
    (16, 4, 2, 64, [0, 40], [200, 77], False),              # chains: a prompt
    (16, 2, 2, 128, [600], [130], False),                   # a chain whose first rows see no last range
    (8, 2, 1, 64, [3, 0, 9], [1, 1, 1], False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, dtype):
    page, H, Hkv, dh, ctx, new, tree = CASES[case]
    rng = np.random.default_rng(case)
    B = len(ctx)
    max_tokens = max(c + n for c, n in zip(ctx, new))
    pages = sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + 3
    order = rng.permutation(pages)
    pool = TokenKVPool(2, H, Hkv, dh, B + 2, max_tokens, num_pages=pages, page_size=page,
                       dtype=dtype, device=DEV, page_order=order)
    model = TokenPoolModel(B + 2, max_tokens, pages, page, order)
    slots = rng.permutation(B + 2)[:B]
    # whatever a page held before has no part in a request: NaN everywhere first
    pool.kv.fill_(float("nan"))
    grow(pool, model, slots, ctx)
    pad = 3
    rows = sum(new) + pad
    parents = random_tree(rng, new, rows) if tree else None
    step = pool.begin_step(i32(slots), i32(new), rows, i32(parents) if tree else None)
    ref = model.begin_step(slots, new, rows, parents)
    check_step(step, ref)
    kv = torch.randn(pool.kv.shape, device=DEV).to(dtype)
    for b, s in enumerate(slots):     # the tokens that the request has
        for t in range(ctx[b] + new[b]):
            pg = int(model.table[s, t // page])
            pool.kv[pg, 1, :, :, t % page] = kv[pg, 1, :, :, t % page]
    q = torch.randn(rows, H, dh, device=DEV).to(dtype)
    out = torch.full((rows, H * dh), 7.0, dtype=dtype, device=DEV)
    got = pool.attention(1, q.reshape(rows, H * dh), step, out=out)
    assert got is out and pool.read_error() == 0
    got = got.reshape(rows, H, dh).double().cpu().numpy()
    want, mean_abs, reach = tree_attention(q.double().cpu().numpy(),
                                           np.nan_to_num(pool.kv.double().cpu().numpy()), 1, model,
                                           ref, parents, dh ** -0.5)
    used = sum(new)
    bound(got[:used], want[:used], mean_abs[:used], reach[:used], dtype, max_tokens, dh)
    assert (got[used:] == 7.0).all()                        # rows behind the last request
