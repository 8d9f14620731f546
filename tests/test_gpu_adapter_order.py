"""The plan's order of rows is a function of the ids alone: stable, so that which rows
of an adapter lie on which side of a tile's border, and with it the order in which a
split product adds a row's terms, is the same every time."""
import numpy as np
import pytest
import torch

from parakeet_b200 import adapter_plan
from test_gpu_adapters import check, make, reference, run

pytestmark = pytest.mark.gpu


def ids_of(kind, rows, adapters, seed):
    rng = np.random.default_rng(seed)
    ids = rng.integers(-1, adapters, rows)
    if kind == "few":            # long segments over many tiles
        ids = rng.choice(rng.integers(0, adapters, 3), rows)
    elif kind == "blocks":       # requests of a few rows each
        ids = np.repeat(rng.integers(-1, adapters, rows // 7 + 1), 7)[:rows]
    elif kind == "falling":
        ids = (np.arange(rows)[::-1] * adapters) // rows
    return ids.astype(np.int32)


@pytest.mark.parametrize("kind", ["random", "few", "blocks", "falling"])
@pytest.mark.parametrize("rows,adapters", [
    (129, 2), (200, 6), (1000, 1), (1023, 64), (1025, 300), (6720, 64), (8192, 33), (8193, 5),
    (9001, 2000), (40000, 64), (33333, 8192), (1048576, 17)])
def test_rows_keep_their_order_within_an_adapter(rows, adapters, kind):
    ids = ids_of(kind, rows, adapters, rows + adapters)
    plan = adapter_plan(torch.from_numpy(ids).cuda(), adapters)
    tiles = -(-rows // 128)
    order = plan.block[:tiles * 128].cpu().numpy()
    want = np.argsort(np.where(ids < 0, adapters, ids), kind="stable")
    assert np.array_equal(order[:rows], want)
    assert (order[rows:] == rows).all()


@pytest.mark.parametrize("M,N,K,n", [(200, 128, 128, 6), (200, 512, 512, 3), (300, 128, 512, 5),
                                     (300, 512, 1024, 40), (700, 512, 512, 2), (1100, 64, 2048, 90)])
def test_split_products_of_several_row_tiles_give_the_same_bits(M, N, K, n):
    """Plans of the same ids made while the GPU is busy with something else."""
    d = make(M, N, K, 16, n, M + N)
    first = run(d)
    check(first, reference(d, "store"))
    busy = torch.randn(2048, 2048, device="cuda")
    side = torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(side):
            for _ in range(4):
                busy = busy @ busy * 1e-2
        assert torch.equal(run(d), first)
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows,adapters", [(700, 5), (9500, 2000), (9500, 8192)])
def test_bad_ids_among_many_rows(rows, adapters):
    """They count as none, and are reported wherever they are."""
    from parakeet_b200 import _lib, ops
    device = torch.device("cuda", torch.cuda.current_device())
    for at in (0, 31, 32, rows // 2, rows - 1):
        for bad in (-2, adapters, 2 ** 31 - 1, -2 ** 31):
            ids = ids_of("random", rows, adapters, at)
            ids[at] = bad
            plan = adapter_plan(torch.from_numpy(ids).cuda(), adapters)
            want = np.argsort(np.where((ids < 0) | (ids >= adapters), adapters, ids), kind="stable")
            assert np.array_equal(plan.block[:rows].cpu().numpy(), want)
            err = ops._gemm_error[device]
            assert int(err.item()) == _lib.PK_DEV_BAD_SLOT
            err.zero_()
    adapter_plan(torch.from_numpy(ids_of("random", rows, adapters, 1)).cuda(), adapters)
    assert int(ops._gemm_error[device].item()) == 0
