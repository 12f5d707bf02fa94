"""y (op)= x . W^T + b: picks the kernel for a dtype and a shape.

float32 operands of more than a decode step's rows, with a K of 128 and more or a large
output, run on the tensor cores as exact sums of three bfloat16 values each, the others on
the CUDA cores; both keep 32-bit products.  bfloat16 operands take the tcgen05 kernel where its
tile rules hold and the row count makes it worthwhile, else the CUDA-core
kernel.  NNIS makes the same kind of choice per projection family with its
projection plans (crates/nnis-model/src/projection_plan.rs:10-90).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from ..csrc import ops

STORE, STORE_F32, ADD_F32 = ops.STORE, ops.STORE_F32, ops.ADD_F32


@dataclass
class Int8Matrix:
    """A matrix [n, k] held in 8-bit codes with a scale for each of its rows (``ops.quantize_rows``), a projection's output channels."""
    codes: torch.Tensor   # int8 [n, ops.int8_width(k)]
    scales: torch.Tensor  # float32 [n]
    shape: tuple

    @classmethod
    def of(cls, weight: torch.Tensor) -> "Int8Matrix":
        n, k = weight.shape
        if k > ops.INT8_LONGEST:
            raise ValueError(f"an 8-bit matrix has up to {ops.INT8_LONGEST} columns; got {k}")
        codes = torch.empty((n, ops.int8_width(k)), dtype=torch.int8, device=weight.device)
        scales = torch.empty(n, dtype=torch.float32, device=weight.device)
        ops.quantize_rows(weight, codes, scales)
        return cls(codes, scales, (n, k))

    def bytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()


def matrix_bytes(weight: Union[None, torch.Tensor, Int8Matrix]) -> int:
    """Bytes of a matrix or a bias as it is held; 0 for None."""
    if weight is None:
        return 0
    return weight.bytes() if isinstance(weight, Int8Matrix) else weight.numel() * weight.element_size()


def normed_codes(hidden: torch.Tensor, norm, dtype: torch.dtype, workspace):
    """(codes, scales) of a norm's rows, for products of 8-bit matrices that read the same rows."""
    n, width = hidden.shape
    codes = workspace.get("int8_normed_codes", (n, ops.int8_width(width)), torch.int8)
    scales = workspace.get("int8_normed_scales", (n,), torch.float32)
    ops.rmsnorm_int8(hidden, norm.weight, norm.eps, codes, scales, dtype)
    return codes, scales


def linear(x: torch.Tensor, weight: Union[torch.Tensor, Int8Matrix], bias: Optional[torch.Tensor], out: torch.Tensor,
           mode: int, workspace=None, decode: bool = False) -> None:
    """``workspace``: the step's buffers (``engine.workspace.Workspace``); with it the adding
    tensor-core product may cut a long K among several CTAs per tile (few rows, few tiles),
    which needs scratch for their partial sums.  ``decode``: the step brings one token per
    sequence; a bfloat16 product of few rows then runs as a decode projection kernel (weights
    by bulk copies ahead of the wait for the kernel before) where that kernel takes the shape.
    A matrix in 8-bit codes is multiplied as such, which needs the workspace."""
    if isinstance(weight, Int8Matrix):
        ops.linear_int8(x, weight.codes, weight.scales, bias, out, mode, workspace)
        return
    m, (n, k) = x.shape[0], weight.shape
    if decode and x.dtype == torch.bfloat16 and ops.gemv_pays(m, n, k, mode, x.device):
        split = ops.gemv_split(m, n, k, workspace) if mode == ADD_F32 and workspace is not None else None
        ops.gemv_bf16(weight, bias, out, mode, x=x, split=split)  # (STORE, STORE_F32, ADD_F32 are its epilogues' codes)
    elif x.dtype == torch.bfloat16 and ops.gemm_tc_takes(m, n, k):
        scratch = tickets = None
        if mode == ADD_F32 and workspace is not None and ops.GEMM_SPLIT_K:
            splits, floats, tiles = ops.gemm_tc_splits(m, n, k, x.device)
            if splits > 1:
                scratch = workspace.get("gemm_split_sums", (floats,), torch.float32)
                tickets = workspace.zeros("gemm_split_tickets", (tiles,), torch.int32)
        ops.gemm_tc(x, weight, bias, out, mode, split_scratch=scratch, split_tickets=tickets)
    elif x.dtype == torch.float32 and ops.gemm_split_f32_pays(x, weight):
        ops.gemm_split_f32(x, weight, bias, out, mode)
    else:
        ops.gemm_simt(x, weight, bias, out, mode)
