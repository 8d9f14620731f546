"""Cases for the token-decoding operators: a page pool that grows with its
requests (page tables and slot maps from request lengths, append, acceptance),
attention of drafted token trees over it, and low-rank adapters of many
requests beside a shared projection.

Sizes follow the models and serving batches of this repository (d_model 512
and 1024, 8 heads of 64 or 128, feed-forward 2048 and 4096, 80 to 2048 streams,
16-row pages); the grouped-query and long-context cases are generic.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
TREE = 64          # most nodes of one drafted tree


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # 8 requests, drafts of up to 12 tokens: the bookkeeping of a latency-bound step
        dict(name="tables_small", op="tables", batch=8, nodes=12, context=200, page=16),
        # a full serving batch with trees of up to 64 drafts
        dict(name="tables_large", op="tables", batch=2048, nodes=64, context=2000, page=16),
        # one verification step's cache traffic (append, accept, roll back), one layer
        dict(name="cache_small", op="cache", batch=16, nodes=7, context=100, page=16, layers=1,
             kv_heads=8, dim=64),
        # the same over several layers of a wide model, 128 requests
        dict(name="cache_large", op="cache", batch=128, nodes=32, context=100, page=16, layers=4,
             kv_heads=8, dim=128),
        # one request, one token: plain decoding, latency only
        dict(name="tree_token", op="tree", batch=1, nodes=1, context=300, page=16, heads=8,
             kv_heads=8, dim=64, dtype="bf16"),
        # float32 pool (the parity mode), short transcripts
        dict(name="tree_f32", op="tree", batch=16, nodes=5, context=250, page=16, heads=8,
             kv_heads=8, dim=64, dtype="f32"),
        # 160 streams with ragged transcripts and trees of up to 13 drafts
        dict(name="tree_streams", op="tree", batch=160, nodes=13, context=500, page=16, heads=8,
             kv_heads=8, dim=64, dtype="bf16"),
        # grouped queries, ragged contexts of thousands of tokens, 32-node trees
        dict(name="tree_grouped", op="tree", batch=32, nodes=32, context=8000, page=16, heads=32,
             kv_heads=8, dim=128, dtype="bf16"),
        # one request with a long document: few rows, a long axis
        dict(name="tree_long", op="tree", batch=1, nodes=64, context=131000, page=16, heads=8,
             kv_heads=8, dim=128, dtype="bf16"),
        # 8 single rows, 8 customers: latency only
        dict(name="adapter_token", op="adapter", rows=8, inner=512, outer=512, rank=8, adapters=8,
             epilogue="store"),
        # 160 streams x 2 frames through the small model's first feed-forward projection
        dict(name="adapter_streams", op="adapter", rows=320, inner=512, outer=2048, rank=16,
             adapters=32, epilogue="silu"),
        # 480 streams x 14 frames through the large model's second one, added to the residual
        dict(name="adapter_large", op="adapter", rows=6720, inner=4096, outer=1024, rank=32,
             adapters=64, epilogue="residual"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def _draw_once(rng):
    op = rng.choice(["tables", "cache", "tree", "tree", "adapter", "adapter"])
    if op == "tables":
        return dict(op=op, batch=_log(rng, 1, 2048), nodes=_log(rng, 1, TREE),
                    context=_log(rng, 1, 2000), page=rng.choice([8, 16, 32, 64]))
    if op == "cache":
        return dict(op=op, batch=_log(rng, 1, 128), nodes=_log(rng, 1, TREE),
                    context=_log(rng, 1, 200), page=rng.choice([8, 16, 32]),
                    layers=_log(rng, 1, 4), kv_heads=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 128]))
    if op == "tree":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        kv = rng.choice([1, 2, 4, 8])
        big = dtype == "bf16"
        return dict(op=op, batch=_log(rng, 1, 256 if big else 32),
                    nodes=_log(rng, 1, TREE if big else 16),
                    context=_log(rng, 1, 131000 if big else 600),
                    page=rng.choice([8, 16, 16, 32, 64]),
                    heads=kv * rng.choice([1, 1, 2, 4, 5]), kv_heads=kv, dim=rng.choice([64, 128]),
                    dtype=dtype)
    return dict(op=op, rows=_log(rng, 1, 6720), inner=64 * rng.choice([1, 4, 8, 8, 10, 16, 32, 64]),
                outer=64 * rng.choice([3, 8, 8, 10, 16, 32]), rank=8 * _log(rng, 1, 8),
                adapters=_log(rng, 1, 64),
                epilogue=rng.choice(["store", "silu", "residual", "bias"]))


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def draw(rng):
    most = {}
    for c in listed():
        if c.get("dtype") != "f32":
            most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        case = _draw_once(rng)
        limit = most[case["op"]]
        if case["op"] == "tree":   # padded requests of the plain form fit too
            pad = case["batch"] * (case["context"] + case["nodes"])
            if pad * case["kv_heads"] * case["dim"] > 3e8 or \
                    pad * case["heads"] * case["nodes"] > 3e8:
                continue
        if _cost(case) <= limit:
            return case


def _spread(n, lo, hi):
    """n whole numbers from hi down to lo, the first always hi."""
    if n == 1:
        return [hi]
    return [hi - (hi - lo) * i // (n - 1) for i in range(n)]


def _lengths(case):
    """The cached tokens and the new rows of each request, before shuffling."""
    n = case["batch"]
    ctx = _spread(n, case["context"] // 8, case["context"])
    new = _spread(n, min(2, case["nodes"]), case["nodes"])
    return ctx, new[n // 2:] + new[:n // 2]


def work(case):
    if case["op"] == "adapter":
        m, k, n, r = (case[x] for x in ("rows", "inner", "outer", "rank"))
        used = min(case["adapters"], m)
        two = 2 if case["epilogue"] == "residual" else 1
        return {"bytes": 2 * (m * k + n * k + two * m * n + used * r * (k + n)) + 4 * m,
                "flops": 2 * m * n * k + 2 * m * r * (k + n)}
    ctx, new = _lengths(case)
    rows = sum(new)
    if case["op"] == "tables":
        pages = sum(-(-(c + n) // case["page"]) - -(-c // case["page"]) for c, n in zip(ctx, new))
        # in: parents, lengths, counts, slots; out: row starts, each row's request,
        # position, cache row and mask, the new page ids (popped, listed, given back)
        return {"bytes": rows * (4 + 4 + 4 + 4 + 8) + case["batch"] * 6 * 4 + pages * 12,
                "flops": rows * 8}
    esize = 4 if case.get("dtype") == "f32" else 2
    token = case["kv_heads"] * case["dim"] * 2 * esize
    if case["op"] == "cache":
        moved = sum(n // 2 for n in new)
        return {"bytes": case["layers"] * token * 2 * (rows + moved) + rows * 28,
                "flops": rows * 8}
    q = rows * case["heads"] * case["dim"]
    return {"bytes": sum(c + n for c, n in zip(ctx, new)) * token + 2 * q * esize,
            "flops": sum(4 * n * (c + 1) for c, n in zip(ctx, new)) * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ the inputs
def _randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype) * scale


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "parakeet-streaming_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import parakeet_b200
    return parakeet_b200


def _requests(case, g):
    """Request lengths in the seed's order, tree parents, and a pool whose page
    ids come in a random order: request b's pages in its table row slots[b]."""
    ctx, new = _lengths(case)
    B, page = case["batch"], case["page"]
    order = torch.randperm(B, generator=g, device=DEV)
    ctx, new = _ints(ctx)[order], _ints(new)[order]
    rows = int(new.sum())
    slots = torch.randperm(B + 3, generator=g, device=DEV)[:B].to(torch.int32)
    start = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    start[1:] = new.cumsum(0)
    row_request = torch.repeat_interleave(torch.arange(B, device=DEV), new.long())
    node = torch.arange(rows, device=DEV) - start.long()[row_request]
    # most drafts follow the one before, some branch off up to 3 nodes earlier
    back = torch.randint(0, 8, (rows,), generator=g, device=DEV)
    parents = torch.where(node == 0, node - 1, (node - 1 - (back - 4).clamp(min=0)).clamp(min=-1))
    most = case["context"] + case["nodes"]
    width = -(-most // page)
    held = (ctx + page - 1) // page
    need = (ctx + new + page - 1) // page
    pages = int(need.sum()) + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((B + 3, width), -1, dtype=torch.int32, device=DEV)
    first = held.cumsum(0) - held
    col = torch.arange(width, device=DEV)[None]
    k = (pages - 1 - (first[:, None] + col)).clamp(min=0)
    table[slots.long()] = torch.where(col < held[:, None], order[k], -1).to(torch.int32)
    lengths = torch.zeros(B + 3, dtype=torch.int32, device=DEV)
    lengths[slots.long()] = ctx
    heldt = torch.zeros_like(lengths)
    heldt[slots.long()] = held.to(torch.int32)
    top = (pages - held.sum(dtype=torch.int32)).reshape(1).to(torch.int32)
    return dict(ctx=ctx, counts=new, rows=rows, slots=slots, parents=parents.to(torch.int32),
                order=order, table=table, lengths=lengths, held=heldt, free=order.clone(), top=top,
                num_pages=pages, most=most)


def _pool(case, s, layers, heads, kv_heads, dim, dtype, kv=None):
    """The framework's pool in the same state: every request grown to its length."""
    pool = _package().TokenKVPool(layers, heads, kv_heads, dim, case["batch"] + 3, s["most"],
                                  num_pages=s["num_pages"], page_size=case["page"], dtype=dtype,
                                  device=DEV, page_order=s["order"])
    step = pool.begin_step(s["slots"], s["ctx"], int(s["ctx"].sum()))
    pool.end_step(step, s["ctx"] - 1)
    if kv is not None:
        pool.kv.copy_(kv)
    return pool


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "adapter":
        m, k, n, r, a = (case[x] for x in ("rows", "inner", "outer", "rank", "adapters"))
        return dict(case=case, x=_randn(g, m, k), weight=_randn(g, n, k, scale=k ** -0.5),
                    down=_randn(g, a, r, k, scale=k ** -0.5), up=_randn(g, a, n, r, scale=r ** -0.5),
                    scale=torch.rand(a, generator=g, device=DEV) + 0.5,
                    # one row in about `adapters` + 1 has none
                    ids=torch.randint(-1, a, (m,), generator=g, device=DEV).to(torch.int32),
                    residual=_randn(g, m, n), bias=_randn(g, n))
    s = _requests(case, g)
    s["case"] = case
    B = case["batch"]
    if case["op"] == "tables":
        if own:
            s["pool"] = _pool(case, s, 1, 1, 1, 64, torch.bfloat16)
        return s
    dtype = TYPES[case.get("dtype", "bf16")]
    layers, H, D = case.get("layers", 1), case["kv_heads"], case["dim"]
    shape = (s["num_pages"], layers, 2, H, case["page"], D)
    if case["op"] == "cache":
        s["kv"] = torch.zeros(shape, dtype=dtype, device=DEV)
        s["key"] = _randn(g, layers, s["rows"], H, D, dtype=dtype)
        s["value"] = _randn(g, layers, s["rows"], H, D, dtype=dtype)
        s["last"] = (torch.rand(B, generator=g, device=DEV) * (s["counts"] + 1)).to(torch.int32) - 1
        if own:
            s["pool"] = _pool(case, s, layers, H, H, D, dtype)
        return s
    s["kv"] = _randn(g, *shape, dtype=dtype)
    s["query"] = _randn(g, s["rows"], case["heads"], D, dtype=dtype)
    if own:   # the step's tables serve every layer of the model
        s["pool"] = _pool(case, s, layers, case["heads"], H, D, dtype, s["kv"])
        s["step"] = s["pool"].begin_step(s["slots"], s["counts"], s["rows"], s["parents"])
        del s["kv"]
    else:
        s["step"] = _begin(s)
    return s


# ------------------------------------------------------------------ the plain forms
def _begin(s):
    """Pages for each request's new rows off the free stack, in batch order, and
    each row's request, position (context + depth), cache row and ancestors."""
    page, slot = s["case"]["page"], s["slots"].long()
    counts, parents = s["counts"].long(), s["parents"].long()
    start = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    length, held = s["lengths"][slot].long(), s["held"][slot].long()
    need = (length + counts + page - 1) // page
    take = need - held
    first = take.cumsum(0) - take
    table = s["table"][slot]
    col = torch.arange(table.shape[1], device=DEV)[None]
    k = (s["top"].long() - 1 - (first[:, None] + col - held[:, None])).clamp(0, s["free"].numel() - 1)
    table = torch.where((col >= held[:, None]) & (col < need[:, None]), s["free"][k], table)
    s["table"][slot] = table
    s["held"][slot] = need.to(torch.int32)
    s["top"].sub_(take.sum())
    row = torch.arange(s["rows"], device=DEV)
    req = torch.searchsorted(start, row, right=True) - 1
    node = row - start[req]
    mask, hops = torch.ones_like(node) << node, (parents >= 0).long()
    jump = torch.where(parents >= 0, start[req] + parents, -1)
    for _ in range(6):       # ancestors and depths by doubling: at most 64 nodes
        live, at = jump >= 0, jump.clamp(min=0)
        mask = mask | torch.where(live, mask[at], 0)
        hops = hops + torch.where(live, hops[at], 0)
        jump = torch.where(live, jump[at], -1)
    where = length[req] + node
    slot_map = table[req, where // page].long() * page + where % page
    return dict(start=start.to(torch.int32), request=req.to(torch.int32),
                position=(length[req] + hops).to(torch.int32), slot_map=slot_map.to(torch.int32),
                mask=mask, length=length)


def _shrink(s, lengths):
    """The requests at `lengths` tokens: pages past the end back on the stack."""
    page, slot = s["case"]["page"], s["slots"].long()
    held = s["held"][slot].long()
    keep = (lengths + page - 1) // page
    give = held - keep
    first = give.cumsum(0) - give
    total = give.sum()
    table = s["table"][slot]
    col = torch.arange(table.shape[1], device=DEV)[None]
    back = (col >= keep[:, None]) & (col < held[:, None])
    at = s["top"].long() + total - 1 - (first[:, None] + col - keep[:, None])
    size = s["free"].numel()
    spare = torch.cat([s["free"], s["free"][:1]])     # the last place takes what is not given back
    spare[torch.where(back, at, size)] = table
    s["free"].copy_(spare[:size])
    s["table"][slot] = torch.where(back, -1, table)
    s["held"][slot] = keep.to(torch.int32)
    s["lengths"][slot] = lengths.to(torch.int32)
    s["top"].add_(total)


def _cache(s):
    """The step's rows into the pool, then those on the path to node last[b]
    (none for -1) behind the context in order of depth."""
    page, step, kv = s["case"]["page"], _begin(s), s["kv"]
    start, req = step["start"].long(), step["request"].long()
    row = torch.arange(s["rows"], device=DEV)
    node = row - start[req]
    last = s["last"].long()
    path = torch.where(last >= 0, step["mask"][(start[:-1] + last).clamp(min=0)], 0)
    on = (path[req] >> node) & 1
    before = on.cumsum(0) - on
    to = start[req] + before - before[start[req]]         # the path's row of each depth
    source = torch.cat([row, row[:1]])                    # the last place takes the others
    source[torch.where(on > 0, to, s["rows"])] = row
    source = source[:-1]
    at = step["slot_map"].long()
    kv[at // page, :, 0, :, at % page] = s["key"][:, source].transpose(0, 1)
    kv[at // page, :, 1, :, at % page] = s["value"][:, source].transpose(0, 1)
    count = torch.zeros_like(step["length"]).index_add_(0, req, on)
    s["lengths"][s["slots"].long()] = (step["length"] + count).to(torch.int32)
    return step


def _tree(s):
    """softmax(q k^T / sqrt(dim)) v over the request's context and the row's
    ancestors, itself among them; requests padded to the longest."""
    case, step = s["case"], s["step"]
    page, H, D = case["page"], case["kv_heads"], case["dim"]
    B, G = case["batch"], case["heads"] // case["kv_heads"]
    start, req = step["start"].long(), step["request"].long()
    node = torch.arange(s["rows"], device=DEV) - start[req]
    table = s["table"][s["slots"].long()].long().clamp(min=0)
    kv = s["kv"][table, 0].float()                        # [B, pages, 2, H, page, D]
    key, value = (kv[:, :, i].permute(0, 2, 1, 3, 4).reshape(B, H, -1, D) for i in (0, 1))
    n = case["nodes"]
    query = torch.zeros(B, n, H, G, D, device=DEV)
    query[req, node] = s["query"].float().view(-1, H, G, D)
    query = query.permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D)
    mask = torch.zeros(B, n, dtype=torch.int64, device=DEV)
    mask[req, node] = step["mask"]
    score = (query @ key.transpose(-1, -2)) * D ** -0.5   # [B, H, n * G, tokens]
    rel = torch.arange(key.shape[2], device=DEV)[None] - step["length"][:, None]
    bit = (mask[:, :, None] >> rel.clamp(0, TREE - 1)[:, None]) & 1
    ok = (rel < 0)[:, None] | ((rel >= 0) & (rel < TREE))[:, None] & (bit > 0)
    ok = ok[:, None, :, None].expand(B, 1, n, G, -1).reshape(B, 1, n * G, -1)
    score = score.masked_fill_(~ok, float("-inf"))
    score = score - score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = score.exp_()
    total = p.sum(-1, keepdim=True).clamp_(min=1e-30)
    out = (p @ value) / total
    out = out.view(B, H, n, G, D).permute(0, 2, 1, 3, 4)[req, node]
    return out.reshape(-1, case["heads"], D).to(TYPES[case["dtype"]])


def _adapter(s):
    """x W^T and, for rows with an adapter, scale (x A^T) B^T: both products over
    all adapters at once, the other adapters' columns zeroed in between."""
    case = s["case"]
    a, r = case["adapters"], case["rank"]
    x = s["x"].float()
    acc = x @ s["weight"].float().t()
    low = (x @ s["down"].float().view(a * r, -1).t()).view(-1, a, r)
    mine = s["ids"].long()[:, None] == torch.arange(a, device=DEV)[None]
    low = (low * torch.where(mine, s["scale"][None], 0.0)[:, :, None]).view(-1, a * r)
    acc = acc + low @ s["up"].float().transpose(1, 2).reshape(a * r, -1)
    if case["epilogue"] == "silu":
        acc = acc / (1 + (-acc).exp())
    elif case["epilogue"] == "residual":
        acc = s["residual"].float() + 0.5 * acc
    elif case["epilogue"] == "bias":
        acc = acc + s["bias"].float()
    return acc.to(torch.bfloat16)


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _run_own(s, op)
    if op == "adapter":
        return _adapter(s)
    if op == "tree":
        return _tree(s)
    if op == "tables":
        step, out = _begin(s), {}
    else:
        step = _cache(s)
        out = {"kv": s["kv"], "lengths": s["lengths"].clone()}
    _shrink(s, step["length"])            # the drafts dropped, their pages given back
    return dict(start=step["start"], request=step["request"], position=step["position"],
                slot_map=step["slot_map"], mask=step["mask"], table=s["table"], held=s["held"],
                free=s["free"], top=s["top"], **out)


def _run_own(s, op):
    if op == "adapter":
        p = sys.modules.get("parakeet_b200") or _package()
        e = s["case"]["epilogue"]
        plan = p.adapter_plan(s["ids"], s["case"]["adapters"])
        return p.adapter_gemm(s["x"], s["weight"], s["down"], s["up"], plan, scale=s["scale"],
                              epilogue=e, residual=s["residual"] if e == "residual" else None,
                              alpha=0.5 if e == "residual" else 1.0,
                              bias=s["bias"] if e == "bias" else None)
    pool = s["pool"]
    if op == "tree":
        return pool.attention(0, s["query"], s["step"])
    step = pool.begin_step(s["slots"], s["counts"], s["rows"], s["parents"])
    if op == "tables":
        out = {}
    else:
        pool.append(0, s["key"], s["value"], step)
        pool.end_step(step, s["last"])
        out = {"kv": pool.kv, "lengths": pool.lengths.clone()}
    pool.truncate(s["slots"], s["ctx"])
    return dict(start=step.row_start, request=step.row_request, position=step.positions,
                slot_map=step.slot_map, mask=step.masks, table=pool.page_table, held=pool.held,
                free=pool.free_pages, top=pool.free_count, **out)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] in ("tables", "cache"):
        return None            # whole numbers and copied rows
    s = prepare(case, seed)
    if case["op"] == "adapter":
        out = s["x"].double() @ s["weight"].double().T
        for a in range(case["adapters"]):
            m = (s["ids"] == a).nonzero()[:, 0]
            low = s["x"][m].double() @ s["down"][a].double().T
            out[m] += s["scale"][a].double() * (low @ s["up"][a].double().T)
        return {"store": lambda v: v, "silu": lambda v: v * torch.sigmoid(v),
                "residual": lambda v: s["residual"].double() + 0.5 * v,
                "bias": lambda v: v + s["bias"].double()}[case["epilogue"]](out)
    ctx, new, par = s["ctx"].tolist(), s["counts"].tolist(), s["parents"].tolist()
    G = case["heads"] // case["kv_heads"]
    out = torch.empty(s["rows"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    row = 0
    for b in range(case["batch"]):
        L, n = ctx[b], new[b]
        pages = s["table"][int(s["slots"][b])][: -(-(L + n) // case["page"])].long()
        kv = s["kv"][pages, 0]
        key, value = (kv[:, i].transpose(0, 1).flatten(1, 2)[:, :L + n] for i in (0, 1))
        see = torch.zeros(n, L + n, dtype=torch.bool)
        see[:, :L] = True
        for i in range(n):
            j = i
            while j >= 0:
                see[i, L + j] = True
                j = par[row + j]
        see = see.to(DEV)
        q = s["query"][row:row + n].double()
        for h in range(case["kv_heads"]):
            t = torch.einsum("igd,kd->gik", q[:, h * G:(h + 1) * G], key[h].double())
            t = (t / math.sqrt(case["dim"])).masked_fill(~see[None], -math.inf).softmax(-1)
            out[row:row + n, h * G:(h + 1) * G] = torch.einsum("gik,kd->igd", t, value[h].double())
        row += n
    return out
