"""Chains (prompts, plain decoding) at lengths where row tiles are cut over several
workers, behind the diagonal too, against float64 on the GPU; tolerance as in
test_gpu_tokens."""
import numpy as np
import pytest
import torch

from test_gpu_tokens import bound, filled

pytestmark = pytest.mark.gpu

CASES = [
    # (dtype, query heads, K/V heads, dim, page, context lengths, new tokens)
    (torch.bfloat16, 8, 8, 64, 16, [0], [2500]),            # one prompt: 128-row tiles
    (torch.bfloat16, 8, 2, 128, 32, [700, 0], [1300, 2049]),
    (torch.bfloat16, 1, 1, 64, 8, [4000], [16]),            # 16-row tiles, keys cut
    (torch.bfloat16, 2, 1, 128, 64, [9000, 3, 130], [7, 8, 1]),
    (torch.float32, 2, 1, 64, 16, [100, 0], [900, 1100]),
    (torch.float32, 2, 2, 128, 16, [3000], [5]),
    # a prompt beside requests of one token: the 16-row kernel for all of them
    (torch.bfloat16, 2, 2, 64, 16, [0] + [40 * i for i in range(1, 128)], [1000] + [1] * 127),
    (torch.bfloat16, 4, 2, 128, 16, [37] + [300] * 90, [600] + [1] * 90),
]


def float64(pool, model, ref, q):
    """Outputs, mean |v| and the largest sum of |q||k|, request by request."""
    rows, H, dh = q.shape
    Hkv, page = pool.num_kv_heads, pool.page_size
    G, scale = H // Hkv, dh ** -0.5
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    mean_abs, reach = torch.empty_like(out), torch.empty(rows, H, dtype=torch.float64, device=q.device)
    for b, slot in enumerate(ref["slots"]):
        c, n, r0 = int(ref["context"][b]), int(ref["counts"][b]), int(ref["row_start"][b])
        pages = torch.tensor(model.table[slot][:-(-(c + n) // page)], device=q.device).long()
        kv = pool.kv[pages, 0].double()
        key, value = (kv[:, i].permute(1, 0, 2, 3).reshape(Hkv, -1, dh)[:, :c + n] for i in (0, 1))
        see = torch.ones(n, c + n, dtype=torch.bool, device=q.device).tril(c)
        for h in range(H):
            x = q[r0:r0 + n, h].double()
            p = (x @ key[h // G].T * scale).masked_fill(~see, -torch.inf).softmax(-1)
            out[r0:r0 + n, h] = p @ value[h // G]
            mean_abs[r0:r0 + n, h] = p @ value[h // G].abs()
            reach[r0:r0 + n, h] = (x.abs() @ key[h // G].abs().T * scale).masked_fill(~see, 0).amax(-1)
    return [t.cpu().numpy() for t in (out, mean_abs, reach)]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_long_chains(case):
    dtype, H, Hkv, dh, page, ctx, new = CASES[case]
    rng = np.random.default_rng(case)
    pool, model, step, ref, _, q = filled(rng, page, H, Hkv, dh, ctx, new, dtype, tree=False)
    got = torch.full_like(q, 7.0)
    pool.attention(0, q, step, out=got)
    bound(got.double().cpu().numpy(), *float64(pool, model, ref, q), dtype,
          max(c + n for c, n in zip(ctx, new)), dh)
    assert torch.equal(pool.attention(0, q, step), got)
    assert pool.read_error() == 0
