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
    (16, 40, 1, 64, [50, 0, 333], [1, 2, 1], True),         # a token's heads over several row tiles
    (16, 160, 1, 128, [130, 700], [1, 3], True),            # of 128 rows too
    (32, 48, 2, 64, [70], [9], False),
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


def filled(rng, page, H, Hkv, dh, ctx, new, dtype, tree=True, num_pages=None, order=None, layers=1):
    """A pool whose requests have ``ctx`` tokens of random K and V, and a step of
    ``new`` more, all in place; the model and the step's arrays beside them."""
    B = len(ctx)
    most = max(c + n for c, n in zip(ctx, new))
    pages = num_pages or sum(-(-(c + n) // page) for c, n in zip(ctx, new)) + 1
    pool = TokenKVPool(layers, H, Hkv, dh, B, most, num_pages=pages, page_size=page, dtype=dtype,
                       device=DEV, page_order=order)
    model = TokenPoolModel(B, most, pages, page, order)
    slots = np.arange(B, dtype=np.int32)
    grow(pool, model, slots, np.asarray(ctx))
    rows = int(sum(new))
    parents = random_tree(rng, new, rows) if tree else None
    step = pool.begin_step(i32(slots), i32(new), rows, i32(parents) if tree else None)
    ref = model.begin_step(slots, new, rows, parents)
    if num_pages is None:
        pool.kv.copy_(torch.randn(pool.kv.shape, device=DEV).to(dtype))
    q = torch.randn(rows, H, dh, device=DEV).to(dtype)
    return pool, model, step, ref, parents, q


def reference(pool, model, ref, parents, q, layer=0, scale=None):
    dh = q.shape[-1]
    return tree_attention(q.double().cpu().numpy(), pool.kv.double().cpu().numpy(), layer, model, ref,
                          parents, scale or dh ** -0.5)


# one shape for each kernel: fp32, 16-row tiles (a team of warps, workers with cut row
# tiles), 128-row tiles
KERNELS = [(torch.float32, 8, 2, 64, [90, 700, 3], [6, 9, 12]),
           (torch.bfloat16, 4, 4, 64, [90, 130, 3], [6, 9, 12]),
           (torch.bfloat16, 2, 2, 128, [3000, 700, 3], [6, 9, 12]),
           (torch.bfloat16, 8, 2, 128, [90, 700, 3], [40, 9, 12]),
           (torch.bfloat16, 8, 1, 64, [2000, 61, 0], [20, 64, 5])]


@pytest.mark.parametrize("kernel", range(len(KERNELS)))
@pytest.mark.parametrize("what", ["nan key", "inf value", "nan value", "inf key"])
def test_a_tokens_bad_values_stay_with_the_rows_that_see_it(kernel, what):
    """An inf or NaN in a drafted token's K or V reaches the rows that descend from
    it; every other row is bit for bit what it is without it."""
    dtype, H, Hkv, dh, ctx, new = KERNELS[kernel]
    rng = np.random.default_rng(7 + kernel)
    pool, model, step, ref, parents, q = filled(rng, 16, H, Hkv, dh, ctx, new, dtype)
    clean = pool.attention(0, q, step).clone()
    victims = [(0, 2), (1, 0), (2, 3)]                    # (request, node)
    bad = float("nan") if "nan" in what else float("inf")
    for b, j in victims:
        at = int(ref["slot_map"][ref["row_start"][b] + j])
        pool.kv[at // 16, 0, 0 if "key" in what else 1, :, at % 16, 5::7] = bad
    out = pool.attention(0, q, step)
    masks = ref["masks"].view(np.uint64)
    seen = np.zeros(len(masks), bool)
    for b, j in victims:
        r0, r1 = ref["row_start"][b], ref["row_start"][b + 1]
        seen[r0:r1] |= (masks[r0:r1] >> np.uint64(j) & np.uint64(1)).astype(bool)
    assert seen.any() and not seen.all()
    keep = torch.tensor(~seen, device=DEV)
    assert torch.equal(out[keep], clean[keep])
    if "key" not in what:      # (an inf key may also give a row a weight of zero)
        assert not bool(out[~keep][..., 5::7].isfinite().any())
        others = [c for c in range(dh) if c % 7 != 5]
        assert torch.equal(out[~keep][..., others], clean[~keep][..., others])
    elif bad != bad:
        assert not bool(out[~keep].isfinite().any())
    assert pool.read_error() == 0


@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_an_infinite_value_of_the_context_reaches_its_rows_whatever_its_weight(kernel):
    """A context token whose weight is below fp32's range, with an infinite value."""
    dtype, H, Hkv, dh, ctx, new = KERNELS[kernel]
    rng = np.random.default_rng(70 + kernel)
    pool, model, step, ref, parents, q = filled(rng, 16, H, Hkv, dh, ctx, new, dtype)
    q = q.abs() + 1
    pool.kv[:, :, 0].abs_()
    clean = pool.attention(0, q, step).clone()
    page = int(model.table[0, 0])
    pool.kv[page, 0, 0, :, 5] = -200.0     # a score at least 400 below the others
    low = pool.attention(0, q, step).clone()
    pool.kv[page, 0, 1, :, 5, ::3] = float("inf")
    out = pool.attention(0, q, step)
    n = new[0]
    assert not bool(out[:n, :, ::3].isfinite().any())
    assert torch.equal(out[n:], clean[n:])
    rest = [c for c in range(dh) if c % 3]
    assert torch.equal(out[:n][..., rest], low[:n][..., rest])


@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_large_scores_scale_strides_and_repeatability(kernel):
    """Scores of hundreds (weights of 1 and 0), a given scale, queries out of a
    wider buffer, a strided output, and the same bits every time."""
    dtype, H, Hkv, dh, ctx, new = KERNELS[kernel]
    rng = np.random.default_rng(kernel)
    pool, model, step, ref, parents, _ = filled(rng, 8, H, Hkv, dh, ctx, new, dtype)
    rows = step.rows
    wide = (16 * torch.randn(rows, 3, H, dh, device=DEV)).to(dtype)
    q = wide[:, 1]
    buf = torch.full((rows, H, 2, dh), 3.0, dtype=dtype, device=DEV)
    out = pool.attention(0, q, step, scale=0.25, out=buf[:, :, 1])
    want, mean_abs, reach = reference(pool, model, ref, parents, q, scale=0.25)
    bound(out.double().cpu().numpy(), want, mean_abs, reach, dtype, max(ctx) + 64, dh)
    assert bool((buf[:, :, 0] == 3.0).all())
    for _ in range(3):
        assert torch.equal(pool.attention(0, q, step, scale=0.25), out)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements whose requests hold its last pages."""
    page, Hkv, dh = 16, 8, 128
    pages = 2 ** 31 // (2 * Hkv * page * dh) + 70
    rng = np.random.default_rng(0)
    order = np.concatenate([np.arange(pages - 60), rng.permutation(np.arange(pages - 60, pages))])
    for H, ctx, new in ((8, [200, 77], [5, 7]), (32, [300, 77], [30, 64])):
        pool, model, step, ref, parents, q = filled(rng, page, H, Hkv, dh, ctx, new, torch.bfloat16,
                                                    num_pages=pages, order=order)
        assert pool.kv.numel() > 2 ** 31
        tail = torch.randn(pool.kv[-60:].shape, device=DEV).to(torch.bfloat16)
        pool.kv[-60:] = tail
        k = torch.randn(step.rows, Hkv, dh, device=DEV).to(torch.bfloat16)
        v = torch.randn_like(k)
        pool.append(0, k, v, step)
        at = step.slot_map.long()
        assert torch.equal(pool.kv[at // page, 0, 0, :, at % page], k)
        assert torch.equal(pool.kv[at // page, 0, 1, :, at % page], v)
        out = pool.attention(0, q, step)
        small = pool.kv[-60:].double().cpu().numpy()
        shifted = TokenPoolModel(1, 1, 1, page)
        shifted.table = np.where(model.table >= 0, model.table - (pages - 60), -1)
        want, mean_abs, reach = tree_attention(q.double().cpu().numpy(), small, 0, shifted, ref,
                                               parents, dh ** -0.5)
        bound(out.double().cpu().numpy(), want, mean_abs, reach, torch.bfloat16, 400, dh)
        last = np.array([n - 1 for n in new])
        pool.end_step(step, i32(last))
        kept = [int(((int(ref["masks"][ref["row_start"][b] + last[b]])) & (2 ** 64 - 1)).bit_count())
                for b in range(2)]
        assert pool.lengths.tolist() == [c + k for c, k in zip(ctx, kept)]
        assert pool.read_error() == 0
        del pool, tail, step


@pytest.mark.parametrize("batch", [3000, 9000])
def test_tables_of_many_requests(batch):
    """More requests than the planning CTA has threads, and than eight times that."""
    rng = np.random.default_rng(batch)
    n = rng.integers(0, 6, batch).astype(np.int32)
    pages = int((-(-n // 8)).sum()) - 5          # a few requests find none left
    pool = TokenKVPool(1, 1, 1, 64, batch, 16, num_pages=pages, page_size=8, dtype=torch.float32,
                       device=DEV)
    model = TokenPoolModel(batch, 16, pages, 8)
    slots = rng.permutation(batch).astype(np.int32)
    rows = int(n.sum())
    parents = random_tree(rng, n, rows)
    step = pool.begin_step(i32(slots), i32(n), rows, i32(parents))
    ref = model.begin_step(slots, n, rows, parents)
    check_step(step, ref)
    last = np.where(n > 0, n - 1, -1)
    pool.end_step(step, i32(last))
    model.end_step(ref, last)
    check_tables(pool, model)
    cut = np.where(rng.random(batch) < 0.5, 0, model.lengths[slots]).astype(np.int32)
    pool.truncate(i32(slots), i32(cut))
    model.truncate(slots, cut)
    check_tables(pool, model)
    q = torch.randn(rows, 1, 64, device=DEV)
    step = pool.begin_step(i32(slots), i32(np.zeros(batch)), rows)   # rows of nobody
    out = torch.full_like(q, 5.0)
    pool.attention(0, q, step, out=out)
    assert bool((out == 5.0).all())


def test_empty_calls():
    pool = TokenKVPool(2, 4, 2, 64, 3, 100, page_size=16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    step = pool.begin_step(none, none, 4)
    assert step.row_start.tolist() == [0] and step.row_request.tolist() == [-1] * 4
    assert step.slot_map.tolist() == [-1] * 4
    kv = torch.ones(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    pool.append(0, kv, kv, step)
    out = torch.full((4, 4, 64), 2.0, dtype=torch.bfloat16, device=DEV)
    pool.attention(0, torch.ones_like(out), step, out=out)
    pool.end_step(step, none)
    pool.truncate(none, none)
    assert bool((out == 2.0).all()) and not bool(pool.kv.any()) and pool.read_error() == 0
    step = pool.begin_step(i32([1]), i32([0]), 0)
    assert step.context.tolist() == [0]
    pool.end_step(step, i32([-1]))
    assert pool.lengths.tolist() == [0, 0, 0] and int(pool.free_count) == pool.num_pages


@pytest.mark.parametrize("dtype,H,Hkv,dh", [(torch.float32, 4, 2, 64), (torch.bfloat16, 4, 4, 64),
                                            (torch.bfloat16, 8, 2, 128)])
def test_bad_table_entries_are_reported(dtype, H, Hkv, dh):
    """A page id outside the pool is an error bit, and the others' rows are right."""
    rng = np.random.default_rng(1)
    ctx, new = [40, 70], [12, 3]
    pool, model, step, ref, parents, q = filled(rng, 16, H, Hkv, dh, ctx, new, dtype)
    want = pool.attention(0, q, step).clone()
    for bad in (pool.num_pages, 2 ** 30, -5):
        held = pool.page_table.clone()
        pool.page_table[0, 1] = bad
        out = pool.attention(0, q, step)
        r0, r1 = int(ref["row_start"][1]), int(ref["row_start"][2])
        assert torch.equal(out[r0:r1], want[r0:r1])
        assert pool.read_error() == _lib.PK_DEV_BAD_PAGE
        pool.error.zero_()
        pool.page_table[0, 2] = min(bad, 2 ** 26)       # where request 0's new rows are
        again = pool.begin_step(i32([0, 1]), i32(new), sum(new), i32(parents))
        before = pool.kv.clone()
        k = torch.ones(sum(new), Hkv, dh, dtype=dtype, device=DEV)
        pool.append(0, k, k, again)
        pool.end_step(again, i32([n - 1 for n in new]))
        torch.cuda.synchronize()
        assert bad < 0 or pool.read_error() == _lib.PK_DEV_BAD_PAGE
        changed = (pool.kv != before).flatten(1).any(1).nonzero()[:, 0].tolist()
        assert set(changed) <= {0, *model.table[1].tolist(), *model.table[0].tolist()}
        pool.kv.copy_(before)
        pool.page_table.copy_(held)
        pool.lengths.copy_(i32(ctx))
        pool.error.zero_()


def test_a_whole_decode_captured_and_replayed():
    """Steps of drafting, attention, acceptance and cutting, captured once and
    replayed with other requests, counts, trees and acceptances: lengths and page
    tables live on the device.  The second layer reads the first one's output, as
    a model's would."""
    rng = np.random.default_rng(3)
    slots_n, B, rows, L, H, Hkv, dh, page = 7, 4, 40, 2, 4, 2, 64, 16
    pages, most = 60, 400
    order = rng.permutation(pages)
    pool = TokenKVPool(L, H, Hkv, dh, slots_n, most, num_pages=pages, page_size=page, device=DEV,
                       page_order=order)
    model = TokenPoolModel(slots_n, most, pages, page, order,
                           kv=np.zeros((pages, L, 2, Hkv, page, dh), np.float32))
    buf = dict(slots=i32(np.arange(B)), counts=i32(np.ones(B)), parents=i32(np.full(rows, -1)),
               last=i32(np.zeros(B)), cut=i32(np.zeros(B)),
               x=torch.zeros(rows, H * dh, dtype=torch.bfloat16, device=DEV))
    w = [(torch.randn(2 * Hkv * dh, H * dh, device=DEV) / 16).to(torch.bfloat16) for _ in range(L)]

    def decode():
        step = pool.begin_step(buf["slots"], buf["counts"], rows, buf["parents"])
        x = buf["x"]
        outs = []
        for layer in range(L):
            kv = x @ w[layer].t()
            pool.append(layer, kv[:, :Hkv * dh], kv[:, Hkv * dh:], step)
            x = pool.attention(layer, x, step, out=torch.zeros_like(x))
            outs.append((kv, x))
        pool.end_step(step, buf["last"])
        return step, outs

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    pool.reset(order)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step, outs = decode()
    torch.cuda.synchronize()
    pool.reset(order)
    pool.kv.zero_()
    for it in range(12):
        slots = rng.permutation(slots_n)[:B].astype(np.int32)
        n = rng.integers(0, 11, B).astype(np.int32)
        parents = random_tree(rng, n, rows)
        last = np.array([rng.integers(-1, k) for k in n], np.int32)
        for key, v in (("slots", slots), ("counts", n), ("parents", parents), ("last", last)):
            buf[key].copy_(i32(v))
        buf["x"].copy_(torch.randn(rows, H * dh, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        ref = model.begin_step(slots, n, rows, parents)
        check_step(step, ref)
        used = int(n.sum())
        x = buf["x"]
        for layer, (kv, got) in enumerate(outs):
            rows_np = kv.float().cpu().numpy().reshape(rows, 2, Hkv, dh)
            model.append(layer, rows_np[:, 0], rows_np[:, 1], ref)
            want, mean_abs, reach = tree_attention(x.double().cpu().numpy().reshape(rows, H, dh),
                                                   model.kv, layer, model, ref, parents, dh ** -0.5)
            bound(got.double().cpu().numpy().reshape(rows, H, dh)[:used], want[:used], mean_abs[:used],
                  reach[:used], torch.bfloat16, most, dh)
            assert not bool(got[used:].any())
            x = got
        model.end_step(ref, last)
        check_tables(pool, model)
        assert np.array_equal(pool.kv.float().cpu().numpy(), model.kv)
        if it % 4 == 3:
            who = rng.permutation(slots_n)[:3].astype(np.int32)
            keep = (model.lengths[who] // 2).astype(np.int32)
            pool.truncate(i32(who), i32(keep))
            model.truncate(who, keep)
            check_tables(pool, model)


def test_layers_on_two_streams_at_once():
    """The attention of two layers of one step, in two captured graphs replayed
    side by side and on two streams: each call has a workspace of its own."""
    rng = np.random.default_rng(5)
    for dtype, H, Hkv, dh, ctx, new in KERNELS[2:]:
        pool, model, step, ref, parents, q = filled(rng, 16, H, Hkv, dh, ctx, new, dtype, layers=2)
        want = [pool.attention(layer, q, step).clone() for layer in (0, 1)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        graphs, outs = [], []
        torch.cuda.synchronize()
        for layer, s in enumerate(streams):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
                outs.append(pool.attention(layer, q, step))
            graphs.append(g)
        for _ in range(20):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        got = []
        for layer, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(pool.attention(layer, q, step))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("nl", [1, 3])
def test_one_token_of_one_kv_head(dh, nl):
    """[nl, 1, dh] may be one row of nl layers or nl rows of one head: the step's
    rows say which."""
    pool = TokenKVPool(nl, 2, 1, dh, 2, 40, num_pages=4, page_size=8, device=DEV)
    k = torch.randn(nl, 1, dh, device=DEV).to(torch.bfloat16)
    v = torch.randn_like(k)
    step = pool.begin_step(i32([1]), i32([1]), 1)
    pool.append(0, k, v, step)
    page = pool.page_table.tolist()[1][0]
    assert torch.equal(pool.kv[page, :, 0, 0, 0], k[:, 0])
    assert torch.equal(pool.kv[page, :, 1, 0, 0], v[:, 0])
    out = pool.attention(nl - 1, torch.randn(1, 2 * dh, device=DEV).to(torch.bfloat16), step)
    assert torch.equal(out, v[nl - 1].repeat(1, 2))    # one key: its value
    pool.end_step(step, i32([0]))
    step = pool.begin_step(i32([1]), i32([3]), 3)
    rows = torch.randn(3, 1, dh, device=DEV).to(torch.bfloat16)
    pool.append(0, rows, rows, step)
    assert torch.equal(pool.kv[page, 0, 0, 0, 1:4], rows[:, 0])
    assert pool.read_error() == 0


@pytest.mark.parametrize("dtype,H,Hkv,dh,batch,most_ctx,most_new", [
    (torch.bfloat16, 8, 8, 64, 260, 5, 3), (torch.bfloat16, 16, 8, 128, 150, 20, 7),
    (torch.bfloat16, 32, 8, 64, 90, 40, 12), (torch.bfloat16, 8, 8, 128, 80, 9, 60),
    (torch.float32, 8, 8, 64, 120, 30, 4), (torch.bfloat16, 8, 8, 64, 30, 900, 4),
    (torch.bfloat16, 4, 4, 128, 20, 1400, 2), (torch.bfloat16, 2, 1, 128, 3, 2500, 8)])
def test_many_short_requests_and_few_long_ones(dtype, H, Hkv, dh, batch, most_ctx, most_new):
    """More row tiles than workers, a few whole ones each; a CTA's warps on one longer
    row tile; small shares of few row tiles."""
    rng = np.random.default_rng(batch)
    ctx = rng.integers(0, most_ctx + 1, batch).tolist()
    new = rng.integers(0, most_new + 1, batch).tolist()
    ctx[0], new[0] = most_ctx, most_new
    pool, model, step, ref, parents, q = filled(rng, 16, H, Hkv, dh, ctx, new, dtype)
    want, mean_abs, reach = reference(pool, model, ref, parents, q)
    out = torch.full_like(q, 7.0)
    pool.attention(0, q, step, out=out)
    bound(out.double().cpu().numpy(), want, mean_abs, reach, dtype, most_ctx + most_new, dh)
    assert pool.read_error() == 0


@pytest.mark.parametrize("kernel", range(len(KERNELS)))
def test_out_may_be_the_query(kernel):
    dtype, H, Hkv, dh, ctx, new = KERNELS[kernel]
    rng = np.random.default_rng(31 + kernel)
    pool, model, step, ref, parents, q = filled(rng, 16, H, Hkv, dh, ctx, new, dtype)
    want = pool.attention(0, q, step).clone()
    got = pool.attention(0, q, step, out=q)
    assert got.data_ptr() == q.data_ptr()
    for row, req in enumerate(step.row_request.tolist()):
        if req >= 0:
            assert torch.equal(got[row], want[row])


def test_python_refusals():
    pool = TokenKVPool(2, 4, 2, 64, 3, 100, page_size=16, device=DEV)
    other = TokenKVPool(2, 4, 2, 64, 3, 100, page_size=16, device=DEV)
    s, n = i32([0, 1]), i32([2, 3])
    with pytest.raises(TypeError):
        pool.begin_step(s.long(), n, 5)
    with pytest.raises(TypeError):
        pool.begin_step(s.cpu(), n, 5)
    with pytest.raises(ValueError):
        pool.begin_step(s, n[:1], 5)
    with pytest.raises(ValueError):
        pool.begin_step(s, n, -1)
    with pytest.raises(ValueError):
        pool.begin_step(s, n, 5, i32([0, 0]))
    with pytest.raises(ValueError):
        pool.begin_step(i32([[0, 1]]), n, 5)
    with pytest.raises(_lib.PKError):
        pool.begin_step(i32([0, 1, 2, 3]), i32([1, 1, 1, 1]), 4)       # more than the slots
    step = pool.begin_step(s, n, 5)
    kv = torch.zeros(5, 2, 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(5, 4, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (kv.float(), kv[:4], kv[:, :1], kv[..., :32], kv.transpose(1, 2)):
        with pytest.raises((TypeError, ValueError)):
            pool.append(0, bad, bad, step)
    with pytest.raises(ValueError):
        pool.append(0, kv, kv.repeat(1, 2, 1)[:, :2], step)            # other strides
    with pytest.raises(_lib.PKError):
        pool.append(2, kv, kv, step)
    with pytest.raises(_lib.PKError):
        pool.append(1, kv[None].repeat(2, 1, 1, 1), kv[None].repeat(2, 1, 1, 1), step)
    with pytest.raises((TypeError, ValueError)):
        pool.attention(0, q.half(), step)
    with pytest.raises(ValueError):
        pool.attention(0, q, step, out=q[:4])
    with pytest.raises(_lib.PKError):
        pool.attention(0, q, step, scale=0.0)
    with pytest.raises(_lib.PKError):
        pool.attention(-1, q, step)
    with pytest.raises(_lib.PKError):   # rows that are not 16-byte aligned
        pool.attention(0, torch.zeros(5 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(5, 4, 64),
                       step)
    with pytest.raises(ValueError):
        other.attention(0, q, step)
    with pytest.raises(ValueError):
        other.end_step(step, n - 1)
    pool.end_step(step, n - 1)
    for call in (lambda: pool.append(0, kv, kv, step), lambda: pool.attention(0, q, step),
                 lambda: pool.end_step(step, n - 1)):
        with pytest.raises(ValueError):
            call()
    assert pool.lengths.tolist() == [2, 3, 0]
    for bad in (dict(dtype=torch.float16), dict(head_dim=96), dict(page_size=12), dict(num_heads=3),
                dict(device="cpu"), dict(max_tokens=0)):
        args = dict(num_layers=1, num_heads=4, num_kv_heads=2, head_dim=64, num_slots=2, max_tokens=64,
                    device=DEV)
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            TokenKVPool(**{**args, **bad})
