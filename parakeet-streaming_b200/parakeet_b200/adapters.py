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

from ._lib import check, lib
from .ops import GEMM_EPILOGUES, _gemm_error, _ptr, _rows, _stream, gemm_supported
from .tokens import _on


def _error_word(device):
    err = _gemm_error.get(device)
    if err is None:
        err = _gemm_error[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return err


class AdapterPlan:
    """The rows of a step sorted by adapter (``adapter_plan``)."""

    __slots__ = ("ids", "rows", "num_adapters", "block")

    def __init__(self, ids, rows, num_adapters, block):
        self.ids, self.rows, self.num_adapters, self.block = ids, rows, num_adapters, block


def adapter_plan(ids: torch.Tensor, num_adapters: int) -> AdapterPlan:
    """ids int32 [M] on the device: each row's adapter in [0, num_adapters), or
    -1.  An id out of range counts as -1 and sets PK_DEV_BAD_SLOT in the GEMMs'
    error word (``ops.gemm_error_word``).  The plan keeps ``ids``; they must not
    change while it is in use."""
    if ids.dtype is not torch.int32 or not ids.is_cuda or ids.dim() != 1 or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous int32 [M] CUDA tensor")
    rows = ids.shape[0]
    words = lib().pk_adapter_plan_words(rows, num_adapters)
    if words < 0:
        raise ValueError(f"{rows} rows or {num_adapters} adapters: out of range")
    block = torch.empty(words, dtype=torch.int32, device=ids.device)
    with _on(ids.device):
        check(lib().pk_adapter_plan(ids.data_ptr(), rows, num_adapters, block.data_ptr(),
                                    _error_word(ids.device).data_ptr(), _stream(ids.device)),
              "pk_adapter_plan")
    return AdapterPlan(ids, rows, num_adapters, block)


def adapter_gemm(a: torch.Tensor, weight: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                 plan: AdapterPlan, epilogue: str = "store", residual: torch.Tensor | None = None,
                 alpha: float = 1.0, bias: torch.Tensor | None = None,
                 scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """epilogue(acc) with acc[m] = a[m] weight^T + scale[i] (a[m] down[i]^T) up[i]^T
    for row m's adapter i, a[m] weight^T for rows without one; epilogues,
    ``residual``, ``alpha``, ``bias`` and ``out`` as in ``ops.gemm``.

    a [..., K], weight [N, K], down [num_adapters, rank, K], up [num_adapters, N,
    rank], bf16; K and N multiples of 64, rank a multiple of 8 up to 128; scale
    float32 [num_adapters] or None.  The plan's rows are those of ``a`` flattened."""
    if not gemm_supported(a, weight):
        raise ValueError("adapter_gemm needs bf16 CUDA operands, K and N multiples of 64, and an "
                         "aligned weight")
    dev = a.device
    N, K = weight.shape
    n, rank = plan.num_adapters, down.shape[1] if down.dim() == 3 else 0
    for t, shape, name in ((down, (n, rank, K), "down"), (up, (n, N, rank), "up")):
        if t.shape != shape or t.dtype is not torch.bfloat16 or not t.is_contiguous() or \
                t.device != dev:
            raise ValueError(f"{name} must be a contiguous bf16 {shape} tensor on {dev}, got "
                             f"{tuple(t.shape)} {t.dtype}")
    if weight.device != dev or plan.ids.device != dev:
        raise ValueError("operands on different devices")
    if scale is not None and (scale.dtype is not torch.float32 or scale.shape != (n,)
                              or not scale.is_contiguous() or scale.device != dev):
        raise ValueError(f"scale must be a contiguous float32 [{n}] tensor on {dev}")
    a2 = _rows(a, K)
    M = a2.shape[0]
    if plan.rows != M:
        raise ValueError(f"the plan is for {plan.rows} rows, a has {M}")
    if out is None:
        out = torch.empty((M, N), dtype=a.dtype, device=dev)
    elif not out.is_contiguous() or out.numel() != M * N or out.dtype is not a.dtype or \
            out.device != dev:
        raise ValueError("out must be a contiguous [M, N] tensor of a's type and device")
    if epilogue not in GEMM_EPILOGUES:
        raise ValueError(f"epilogue {epilogue!r}: one of {sorted(GEMM_EPILOGUES)}")
    r2 = None
    if epilogue in ("residual", "residual_relu"):
        if residual is None or residual.dtype is not a.dtype or residual.device != dev or \
                residual.shape[-1] != N or residual.numel() != M * N:
            raise ValueError(f"the residual epilogue needs a bf16 residual of {M} x {N}")
        r2 = _rows(residual, N)
    if epilogue == "bias" and (bias is None or not bias.is_contiguous() or bias.shape != (N,)
                               or bias.dtype is not a.dtype or bias.device != dev):
        raise ValueError(f"the bias epilogue needs a contiguous bf16 bias of {N}")
    with _on(dev):
        ws = torch.empty(max(lib().pk_adapter_workspace(M, K, rank), 0), dtype=torch.uint8, device=dev)
        check(lib().pk_adapter_gemm(
            a2.data_ptr(), a2.stride(0), weight.data_ptr(), weight.stride(0), M, N, K,
            out.data_ptr(), N, GEMM_EPILOGUES[epilogue], _ptr(r2),
            r2.stride(0) if r2 is not None else 0, _ptr(bias), float(alpha), down.data_ptr(),
            up.data_ptr(), rank, n, _ptr(scale), plan.ids.data_ptr(), plan.block.data_ptr(),
            ws.data_ptr(), _error_word(dev).data_ptr(), _stream(dev)), "pk_adapter_gemm")
    return out.reshape(*a.shape[:-1], N)


__all__ = ["AdapterPlan", "adapter_gemm", "adapter_plan"]
