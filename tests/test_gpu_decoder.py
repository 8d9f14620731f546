"""A text decoder's verification step as it would be run: adapters beside the
projections, K and V appended to a token pool, tree attention, the path accepted,
requests released - eager, and captured once and replayed on other requests.  Each
stage against float64 of the inputs that it got."""
import numpy as np
import pytest
import torch

from oracle.tokens import TokenPoolModel, tree_attention
from parakeet_b200 import TokenKVPool, adapter_gemm, adapter_plan
from test_gpu_adapters import check as check_projection
from test_gpu_adapters import reference as projection
from test_gpu_tokens import bound, check_step, check_tables, i32, random_tree

pytestmark = pytest.mark.gpu
DEV, BF = "cuda", torch.bfloat16


def weights(n, k, rank, adapters):
    rn = lambda *s, scale: (torch.randn(*s, device=DEV) * scale).to(BF)  # noqa: E731
    return dict(w=rn(n, k, scale=k ** -0.5), down=rn(adapters, rank, k, scale=k ** -0.5),
                up=rn(adapters, n, rank, scale=rank ** -0.5), scale=torch.rand(adapters, device=DEV) + 0.5)


# the 16-row attention kernel and one row tile of adapters; the 128-row one, several
# row tiles, sorted
@pytest.mark.parametrize("slots_n,B,most_new,group", [(9, 5, 12, 1), (12, 8, 40, 4)])
def test_a_verification_step_eager_and_captured(slots_n, B, most_new, group):
    torch.manual_seed(B)
    rng = np.random.default_rng(B)
    L, Hkv, dh, page, adapters, rank = 2, 2, 64, 16, 6, 16
    H = Hkv * group
    D, rows, most, pages = H * dh, B * most_new, 600, 260
    order = rng.permutation(pages)
    pools = [TokenKVPool(L, H, Hkv, dh, slots_n, most, num_pages=pages, page_size=page, device=DEV,
                         page_order=order) for _ in range(2)]
    model = TokenPoolModel(slots_n, most, pages, page, order,
                           kv=np.zeros((pages, L, 2, Hkv, page, dh), np.float32))
    qkv_w = [weights(D + 2 * Hkv * dh, D, rank, adapters) for _ in range(L)]
    out_w = [weights(D, D, rank, adapters) for _ in range(L)]
    buf = dict(slots=i32(np.arange(B)), counts=i32(np.ones(B)), parents=i32(np.full(rows, -1)),
               last=i32(np.zeros(B)), who=i32([0]), keep=i32([0]), ids=i32(np.full(rows, -1)),
               x=torch.zeros(rows, D, dtype=BF, device=DEV))

    def run(pool):
        plan = adapter_plan(buf["ids"], adapters)
        step = pool.begin_step(buf["slots"], buf["counts"], rows, buf["parents"])
        x, seen = buf["x"], []
        for layer in range(L):
            w = qkv_w[layer]
            qkv = adapter_gemm(x, w["w"], w["down"], w["up"], plan, scale=w["scale"])
            q, k, v = qkv.split([D, Hkv * dh, Hkv * dh], dim=1)
            pool.append(layer, k, v, step)
            y = pool.attention(layer, q, step, out=torch.zeros_like(x))
            w = out_w[layer]
            z = adapter_gemm(y, w["w"], w["down"], w["up"], plan, "residual", residual=x, alpha=0.5,
                             scale=w["scale"])
            seen.append((x, qkv, y, z))
            x = z
        pool.end_step(step, buf["last"])
        pool.truncate(buf["who"], buf["keep"])
        return step, seen

    run(pools[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        captured = run(pools[1])
    torch.cuda.current_stream().wait_stream(side)
    for p in pools:
        p.reset(order)
        p.kv.zero_()
    for it in range(8):
        slots = rng.permutation(slots_n)[:B].astype(np.int32)
        n = rng.integers(0, most_new + 1, B).astype(np.int32)
        parents = random_tree(rng, n, rows)
        last = np.array([rng.integers(-1, k) for k in n], np.int32)
        who = rng.permutation(slots_n)[:1].astype(np.int32)
        of_request = rng.integers(-1, adapters, B)
        ids = np.full(rows, -1, np.int32)
        ids[:n.sum()] = np.repeat(of_request, n)
        for key, v in (("slots", slots), ("counts", n), ("parents", parents), ("last", last),
                       ("who", who), ("keep", np.zeros(1)), ("ids", ids)):
            buf[key].copy_(i32(v))
        buf["x"].copy_(torch.randn(rows, D, device=DEV))
        step, seen = run(pools[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(seen, captured[1]):
            assert all(torch.equal(s, t) for s, t in zip(a, b))
        assert torch.equal(pools[0].kv, pools[1].kv)
        assert torch.equal(pools[0].page_table, pools[1].page_table)

        ref = model.begin_step(slots, n, rows, parents)
        check_step(step, ref)
        used = int(n.sum())
        for layer, (x, qkv, y, z) in enumerate(seen):
            check_projection(qkv, projection(dict(qkv_w[layer], x=x, ids=buf["ids"]), "store"))
            check_projection(z, projection(dict(out_w[layer], x=y, ids=buf["ids"], res=x), "residual", 0.5))
            kv = qkv[:, D:].float().cpu().numpy().reshape(rows, 2, Hkv, dh)
            model.append(layer, kv[:, 0], kv[:, 1], ref)
            want, mean_abs, reach = tree_attention(
                qkv[:, :D].double().cpu().numpy().reshape(rows, H, dh), model.kv, layer, model, ref,
                parents, dh ** -0.5)
            bound(y.double().cpu().numpy().reshape(rows, H, dh)[:used], want[:used], mean_abs[:used],
                  reach[:used], BF, most, dh)
            assert not bool(y[used:].any())
        model.end_step(ref, last)
        model.truncate(who, np.zeros(1, np.int32))
        for p in pools:
            check_tables(p, model)
