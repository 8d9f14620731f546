"""Low-rank adapters of many requests beside a shared projection.

``ops.gemm`` whose rows may each belong to a request with an adapter of its own
(a customer's vocabulary, a speaker's accent) - all of them in one call, the
shared weight read once.  The ids of a step's rows are sorted once
(``adapter_plan``) and serve every projection of the step::

    plan = adapter_plan(ids, num_adapters)          # int32 [M], -1 = no adapter
    h = adapter_gemm(x, w1, down1, up1, plan, epilogue="silu")
    y = adapter_gemm(h, w2, down2, up2, plan, epilogue="residual", residual=x, alpha=0.5)
"""
from __future__ import annotations

import torch

from ._lib import PK_ADAPTER_MAX_RANK, lib
from .ops import GEMM_EPILOGUES, _gemm_error, _launch, _rows, _stream


_BF16 = torch.bfloat16


_plan_words: dict = {}   # (rows, adapters): a plan's size


def _error_word(device) -> int:
    """Address of the device's error word, which the GEMMs share."""
    err = _gemm_error.get(device)
    if err is None:
        if torch.cuda.is_current_stream_capturing():   # a replay would clear it again
            raise RuntimeError("a device's first adapter call cannot be captured: make one before")
        # (another thread may have made it meanwhile: one word a device)
        err = _gemm_error.setdefault(device, torch.zeros(1, dtype=torch.int32, device=device))
    return err.data_ptr()


class AdapterPlan:
    """The rows of a step sorted by adapter (``adapter_plan``)."""

    __slots__ = ("rows", "num_adapters", "block")

    def __init__(self, rows, num_adapters, block):
        self.rows, self.num_adapters, self.block = rows, num_adapters, block


def adapter_plan(ids: torch.Tensor, num_adapters: int) -> AdapterPlan:
    """ids int32 [M] on the device: each row's adapter in [0, num_adapters), or
    -1 (``num_adapters`` is 1 at least).  An id out of range counts as -1 and sets PK_DEV_BAD_SLOT in the GEMMs'
    error word (``ops.gemm_error_word``)."""
    if ids.dtype is not torch.int32 or not ids.is_cuda or ids.dim() != 1 or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous int32 [M] CUDA tensor")
    rows, dev, L = ids.shape[0], ids.device, lib()
    words = _plan_words.get((rows, num_adapters))
    if words is None:
        words = L.pk_adapter_plan_words(rows, num_adapters)
        if words < 0:
            raise ValueError(f"{rows} rows or {num_adapters} adapters: out of range")
        if len(_plan_words) >= 256:
            _plan_words.clear()
        _plan_words[rows, num_adapters] = words
    block = ids.new_empty(words)
    _launch(dev, L.pk_adapter_plan, ids.data_ptr(), rows, num_adapters, block.data_ptr(),
            _error_word(dev), _stream(dev))
    return AdapterPlan(rows, num_adapters, block)


def _operand(t, shape, dtype, dev, name):
    if t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or \
            t.get_device() != dev.index:
        raise ValueError(f"{name} must be a contiguous {dtype} {shape} tensor on {dev}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")


def _plain_rows(t):
    """[rows, width] that ops._rows would leave as it is."""
    row, col = t.stride()
    return col == 1 and row % 8 == 0 and row >= t.shape[1] and t.data_ptr() % 16 == 0


def adapter_gemm(a: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                 plan: AdapterPlan, epilogue: str = "store", residual: torch.Tensor | None = None,
                 alpha: float = 1.0, bias: torch.Tensor | None = None,
                 scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """epilogue(acc) with acc[m] = a[m] weight^T + scale[i] (a[m] down[i]^T) up[i]^T
    for row m's adapter i, a[m] weight^T for rows without one; epilogues,
    ``residual``, ``alpha``, ``bias`` and ``out`` as in ``ops.gemm`` (``out`` may be the
    residual, and shares nothing with ``a``).

    a [..., K], weight [N, K], down [num_adapters, rank, K], up [num_adapters, N,
    rank], bf16; K and N multiples of 64, rank a multiple of 8 up to 128; scale
    float32 [num_adapters] or None.  The plan's rows are those of ``a`` flattened.

    Sums are float32, added in an order that the plan's ids alone give.  The low-rank
    scale[i] (a[m] down[i]^T) is rounded to bf16 before its product with ``up``, as the
    tensor cores take it: off by 2^-8 of each term at most, beside the result's own
    rounding."""
    dev, shape = a.device, a.shape
    N, K = weight.shape if weight.dim() == 2 else (0, 0)
    ldw, wcol = weight.stride() if K else (0, 0)
    if a.dtype is not _BF16 or weight.dtype is not _BF16 or not a.is_cuda or weight.device != dev \
            or shape[-1] != K or wcol != 1:
        raise ValueError("adapter_gemm needs bf16 operands a [..., K] and weight [N, K], rows "
                         "contiguous, on one CUDA device")
    n = plan.num_adapters
    rank = down.shape[1] if down.dim() == 3 else 0
    _operand(down, (n, rank, K), _BF16, dev, "down")
    _operand(up, (n, N, rank), _BF16, dev, "up")
    sc = None
    if scale is not None:
        _operand(scale, (n,), torch.float32, dev, "scale")
        sc = scale.data_ptr()
    flat = len(shape) == 2
    a2 = a
    lda, col = a.stride() if flat else (0, 0)
    ap = a.data_ptr()
    if col != 1 or lda % 8 or lda < K or ap % 16:
        a2 = _rows(a, K)
        ap, lda = a2.data_ptr(), a2.stride(0)
    M = a2.shape[0]
    if plan.rows != M or plan.block.device != dev:
        raise ValueError(f"the plan is for {plan.rows} rows on {plan.block.device}, a has {M} on {dev}")
    if out is None:
        out = a.new_empty((M, N))
    elif not out.is_contiguous() or out.numel() != M * N or out.dtype is not _BF16 or \
            out.device != dev:
        raise ValueError("out must be a contiguous [M, N] tensor of a's type and device")
    epi = GEMM_EPILOGUES.get(epilogue)
    if epi is None:
        raise ValueError(f"epilogue {epilogue!r}: one of {sorted(GEMM_EPILOGUES)}")
    r, ldr, b = None, 0, None
    if epilogue == "residual" or epilogue == "residual_relu":
        if residual is None or residual.dtype is not _BF16 or residual.device != dev or \
                residual.shape[-1] != N or residual.numel() != M * N:
            raise ValueError(f"the residual epilogue needs a bf16 residual of {M} x {N}")
        r2 = residual if residual.dim() == 2 and _plain_rows(residual) else _rows(residual, N)
        r, ldr = r2.data_ptr(), r2.stride(0)
    elif epilogue == "bias":
        if bias is None:
            raise ValueError("the bias epilogue needs a bias")
        _operand(bias, (N,), _BF16, dev, "bias")
        b = bias.data_ptr()
    if rank == 0 or rank > PK_ADAPTER_MAX_RANK:
        raise ValueError(f"rank {rank}: a multiple of 8 up to {PK_ADAPTER_MAX_RANK}")
    # (rows padded to 128 of K and of rank; a buffer of this call's own)
    ws = a.new_empty((M + 127) // 128 * 128 * (K + rank))
    _launch(dev, lib().pk_adapter_gemm, ap, lda, weight.data_ptr(), ldw, M, N, K,
            out.data_ptr(), N, epi, r, ldr, b, alpha, down.data_ptr(), up.data_ptr(), rank, n, sc,
            plan.block.data_ptr(), ws.data_ptr(), _error_word(dev), _stream(dev))
    return out if flat and out.dim() == 2 else out.reshape(*a.shape[:-1], N)


__all__ = ["AdapterPlan", "adapter_gemm", "adapter_plan"]
