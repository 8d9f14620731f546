"""pk_adapter_gemm against float64 of the same bf16 operands.

Tolerance per element, with T = sum |x||w| + sum_r |s_r||up_r| the sum of the
absolute terms and B = sum_r |s_r||up_r|: S is rounded to bf16 (2^-8 of each
term), the result once more (2^-8); products of bf16 are exact in fp32 and adding
n of them is off by at most n 2^-24 T (K + rank terms; S's own sums add K 2^-24
sum_r (|x||down|)_r |up_r|).  SiLU's slope is below 1.1; its own evaluation
(__expf, a fast division) is within 2^-20 relative."""
import pytest
import torch

from parakeet_b200 import adapter_gemm, adapter_plan
from parakeet_b200.ops import gemm_error_word

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make(M, N, K, rank, n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(BF)  # noqa: E731
    return dict(x=rn(M, K), w=rn(N, K, scale=K ** -0.5), down=rn(n, rank, K, scale=K ** -0.5),
                up=rn(n, N, rank, scale=rank ** -0.5), res=rn(M, N), bias=rn(N),
                scale=torch.rand(n, generator=g, device="cuda") + 0.5,
                ids=torch.randint(-1, n, (M,), generator=g, device="cuda").to(torch.int32))


def reference(d, epilogue, alpha=1.0, scaled=True):
    """(result, tolerance) in float64."""
    x, w, u = d["x"].double(), d["w"].double(), 2.0 ** -24
    K, rank = w.shape[1], d["down"].shape[1]
    acc = x @ w.T
    terms = x.abs() @ w.abs().T
    low_terms = torch.zeros_like(acc)
    low_sums = torch.zeros_like(acc)
    for a in range(d["down"].shape[0]):
        m = (d["ids"] == a).nonzero()[:, 0]
        sc = d["scale"][a].double() if scaled else 1.0
        dn, up = d["down"][a].double(), d["up"][a].double()
        s = sc * (x[m] @ dn.T)
        acc[m] += s @ up.T
        low_terms[m] = s.abs() @ up.abs().T
        low_sums[m] = sc * (x[m].abs() @ dn.abs().T) @ up.abs().T
    tol = (K + rank) * u * (terms + low_terms) + K * u * low_sums + 2.0 ** -8 * low_terms
    if epilogue == "silu":
        out, tol = acc * torch.sigmoid(acc), 1.1 * tol
        tol = tol + 2.0 ** -20 * out.abs()
    elif epilogue.startswith("residual"):
        out, tol = d["res"].double() + alpha * acc, abs(alpha) * tol
        tol = tol + 2 * u * (d["res"].double().abs() + (alpha * acc).abs())
        if epilogue == "residual_relu":
            out = out.relu()
    elif epilogue == "bias":
        out = acc + d["bias"].double()
        tol = tol + 2 * u * out.abs()
    else:
        out = acc
    return out, tol + 2.0 ** -8 * (out.abs() + tol)


def check(got, want):
    out, tol = want
    err = (got.double() - out).abs()
    assert not bool(err.isnan().any())
    bad = err > tol
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float((err / tol).max()):.3g} of the bound")
    assert gemm_error_word("cuda") == 0


def run(d, epilogue="store", alpha=1.0, scaled=True, plan=None, **kw):
    plan = plan or adapter_plan(d["ids"], d["down"].shape[0])
    return adapter_gemm(d["x"], d["w"], d["down"], d["up"], plan, epilogue=epilogue,
                        residual=d["res"] if epilogue.startswith("residual") else None, alpha=alpha,
                        bias=d["bias"] if epilogue == "bias" else None,
                        scale=d["scale"] if scaled else None, **kw)


@pytest.mark.parametrize("M,N,K,rank,n", [
    (1, 64, 64, 8, 1), (8, 512, 512, 8, 8), (7, 192, 128, 16, 3), (127, 64, 640, 24, 5),
    (128, 128, 64, 64, 2), (129, 128, 192, 72, 130), (300, 640, 512, 128, 7), (320, 2048, 512, 16, 32),
    (1000, 1024, 1024, 32, 64), (6720, 1024, 1024, 32, 64), (2500, 4096, 256, 16, 300),
    (4096, 256, 320, 40, 1), (2500, 2048, 2048, 16, 40), (2305, 2048, 2048, 72, 5)])
def test_store(M, N, K, rank, n):
    d = make(M, N, K, rank, n, M + N + K)
    check(run(d), reference(d, "store"))


@pytest.mark.parametrize("epilogue,alpha", [("silu", 1.0), ("residual", 0.5), ("residual_relu", -2.0),
                                            ("bias", 1.0)])
@pytest.mark.parametrize("M,N,K", [(33, 192, 128), (700, 512, 512), (5000, 2048, 256),
                                   (2400, 2048, 2048)])
def test_epilogues(M, N, K, epilogue, alpha):
    d = make(M, N, K, 16, 9, M + len(epilogue))
    check(run(d, epilogue, alpha), reference(d, epilogue, alpha))


@pytest.mark.parametrize("kind", ["none", "one", "first", "last", "sorted", "each", "tiles"])
def test_id_patterns(kind):
    """No row with an adapter; one adapter for all; a single row; adapters in
    order; a different one on every row; segments ending on tile borders."""
    M, n = 384, 400
    d = make(M, 128, 128, 16, n, 5)
    ids = torch.full((M,), -1, dtype=torch.int32)
    if kind == "one":
        ids[:] = 399
    elif kind == "first":
        ids[0] = 0
    elif kind == "last":
        ids[-1] = 7
    elif kind == "sorted":
        ids = (torch.arange(M) // 50).int()
    elif kind == "each":
        ids = torch.randperm(M).int()
    elif kind == "tiles":
        ids = (torch.arange(M) // 128).int()
    d["ids"] = ids.cuda()
    check(run(d, scaled=False), reference(d, "store", scaled=False))


@pytest.mark.parametrize("K,N,rank", [(1024, 64, 16), (64, 128, 8), (512, 128, 72), (2048, 320, 128)])
@pytest.mark.parametrize("M", [128, 100, 256])
def test_an_adapter_a_row(M, K, N, rank):
    """As many pairs in a tile as it has rows; K split over 8, 1, 8 and 4 CTAs a tile."""
    d = make(M, N, K, rank, 260, M + rank)
    d["ids"] = torch.randperm(260)[:M].int().cuda()
    check(run(d, "silu"), reference(d, "silu"))


@pytest.mark.parametrize("M,N,K", [(200, 128, 128), (100, 128, 512), (2400, 2048, 2048), (2500, 256, 64)])
def test_adapters_do_not_reach_other_rows(M, N, K):
    """Inf and NaN in an adapter's weights, or in a row, stay with that adapter's
    rows and that row."""
    d = make(M, N, K, 16, 6, 3)
    d["ids"] = (torch.arange(M) % 7 - 1).int().cuda()
    clean = run(d)
    d["down"][2, 3, 5] = float("nan")
    d["up"][4] = float("inf")
    d["x"][11] = float("nan")
    out = run(d)
    other = (d["ids"] != 2) & (d["ids"] != 4)
    other[11] = False
    assert torch.equal(out[other], clean[other])
    assert not bool(out[11].isfinite().any()) and not bool(out[d["ids"] == 2].isfinite().any())
    assert not bool(out[d["ids"] == 4].isfinite().any())


def test_strides_out_and_leading_shape():
    """Rows of wider buffers, a given ``out``, [B, T, K] inputs; R may be C."""
    d = make(60, 256, 128, 16, 4, 9)
    wide = torch.randn(60, 3 * 128, device="cuda").to(BF)
    d["x"] = wide[:, 128:256]
    plan = adapter_plan(d["ids"], 4)
    want = reference(d, "residual", 0.5)
    out = d["res"].clone()
    got = adapter_gemm(d["x"].view(4, 15, 128) if d["x"].is_contiguous() else
                       d["x"].unflatten(0, (4, 15)), d["w"], d["down"], d["up"], plan,
                       epilogue="residual", residual=out, alpha=0.5, scale=d["scale"], out=out)
    assert got.shape == (4, 15, 256) and got.data_ptr() == out.data_ptr()
    check(got.reshape(60, 256), want)


def test_graph_replay_with_other_ids():
    """Plan and product captured together; a replay sorts the ids it finds."""
    d = make(500, 512, 256, 16, 12, 21)
    run(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        out = run(d, "silu")
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2):
        new = make(500, 512, 256, 16, 12, 100 + seed)
        d["ids"].copy_(new["ids"])
        d["x"].copy_(new["x"])
        g.replay()
        torch.cuda.synchronize()
        check(out, reference(d, "silu"))


def test_a_devices_first_call_is_not_captured():
    """The GEMMs' error word is made by the first call; made under capture, each
    replay would clear it."""
    from parakeet_b200 import ops
    d = make(20, 64, 64, 8, 3, 4)
    want = run(d)
    word = ops._gemm_error.pop(d["x"].device)
    try:
        g = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="first"):
            with torch.cuda.graph(g):
                run(d)
    finally:
        ops._gemm_error[d["x"].device] = word
    torch.cuda.synchronize()
    assert torch.equal(run(d), want)


def test_the_ids_may_change_after_the_plan():
    d = make(300, 128, 128, 16, 6, 8)
    plan = adapter_plan(d["ids"], 6)
    want = reference(d, "store")
    d["ids"].fill_(1 << 30)
    check(run(d, plan=plan), want)


def test_bad_ids_are_reported_and_left_without():
    from parakeet_b200 import _lib, ops
    d = make(50, 64, 64, 8, 3, 2)
    d["ids"][3], d["ids"][7] = 3, -2
    out = run(d)
    err = ops._gemm_error[d["x"].device]
    assert int(err.item()) == _lib.PK_DEV_BAD_SLOT
    err.zero_()
    d["ids"][3] = d["ids"][7] = -1
    check(out, reference(d, "store"))


def test_refusals():
    d = make(16, 64, 64, 8, 3, 2)
    plan = adapter_plan(d["ids"], 3)
    args = (d["x"], d["w"], d["down"], d["up"], plan)
    for bad in (dict(epilogue="gelu"), dict(epilogue="bias"), dict(epilogue="residual"),
                dict(scale=d["scale"].double()), dict(scale=d["scale"][:2]),
                dict(out=torch.empty(16, 32, device="cuda", dtype=BF)),
                dict(epilogue="residual", residual=d["res"][:8])):
        with pytest.raises(ValueError):
            adapter_gemm(*args, **bad)
    with pytest.raises(ValueError):
        adapter_gemm(d["x"].float(), *args[1:])
    with pytest.raises(ValueError):
        adapter_gemm(d["x"][:8], *args[1:])
    with pytest.raises(ValueError):
        adapter_gemm(d["x"], d["w"], d["down"][:2], d["up"], plan)
    with pytest.raises(ValueError):
        adapter_gemm(d["x"], d["w"], d["down"], d["up"].transpose(1, 2), plan)
    with pytest.raises(ValueError):
        adapter_plan(d["ids"].long(), 3)
    with pytest.raises(ValueError):
        adapter_plan(d["ids"], 0)


@pytest.mark.parametrize("kind", ["random", "sorted", "one"])
def test_more_rows_than_the_plan_holds_in_registers(kind):
    """9,000 rows: the plan's loop past 8 rows a thread, with and without resorting."""
    d = make(9000, 128, 64, 8, 40, 17)
    if kind == "sorted":
        d["ids"] = torch.where(d["ids"] < 0, 40, d["ids"]).sort().values.int()
        d["ids"][d["ids"] == 40] = -1
    elif kind == "one":
        d["ids"][:] = 3
    check(run(d), reference(d, "store"))


def test_two_streams_at_once():
    """The same plan under two products on two streams, eager and captured."""
    d = [make(300, 256, 512, 16, 5, s) for s in (1, 2)]
    d[1]["ids"] = d[0]["ids"]
    plan = adapter_plan(d[0]["ids"], 5)
    want = [run(x, plan=plan).clone() for x in d]
    streams = [torch.cuda.Stream() for _ in d]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, s in zip(d, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            outs.append(run(x, plan=plan))
        graphs.append(g)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    got = []
    for x, s in zip(d, streams):
        with torch.cuda.stream(s):
            got.append(run(x, plan=plan))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_rows():
    d = make(4, 64, 64, 8, 3, 1)
    plan = adapter_plan(d["ids"][:0], 3)
    out = adapter_gemm(d["x"][:0], d["w"], d["down"], d["up"], plan)
    assert out.shape == (0, 64)


def test_same_bits_every_time():
    for M, N, K in ((8, 512, 512), (700, 512, 512), (2400, 2048, 2048)):
        d = make(M, N, K, 16, 9, M)
        plan = adapter_plan(d["ids"], 9)
        first = run(d, plan=plan)
        for _ in range(3):
            assert torch.equal(run(d, plan=adapter_plan(d["ids"], 9)), first)
