"""A matrix product with its epilogue, as the parts use it.

``y = act(x @ W^T + b) (+ residual)`` with ``W`` kept ``[out, in]``.  Which
kernel runs is decided here from the compute dtype and the number of rows:
float32 takes the CUDA-core kernel or, over a long k, the tensor-core one that
holds whole float32 operands (the true 32-bit path); bfloat16
takes the tensor-core kernels where the shape allows them and the CUDA-core
kernel otherwise.  A model with 4-bit weights (``Runtime.weight_bits``) holds
``W`` as an ``ops.Q4Weight`` and multiplies through ``ops.linear_q4``, its rows in
8 bits where the runtime says so; ``keep`` leaves a matrix as it is (output
heads, and matrices that other kernels read too).  The reference's counterpart is
``Weight`` + ``apply`` (include/ai/LocalModel.hpp:989-1126), its 4-bit blocks of
32 and 8-bit rows include/ai/Quant.hpp.
"""
from __future__ import annotations

from typing import Optional

import torch


class Linear:
    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor], runtime, keep: bool = False):
        self.quantised = getattr(runtime, "weight_bits", 16) == 4 and not keep
        # [out, in], compute dtype unless in 4 bits
        self.weight = runtime.ops.FixedQ4Weight(*runtime.ops.quantize_q4(weight)) if self.quantised else weight
        if self.quantised:
            runtime.saved_bytes += (weight.numel() * weight.element_size()
                                    - sum(t.numel() * t.element_size() for t in self.weight))
        self.bias = bias                # [out] float32 or None
        self.runtime = runtime
        self.out_features, self.in_features = weight.shape

    def __call__(self, x: torch.Tensor, act: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        ops = self.runtime.ops
        if out is None and out_dtype is None:
            out_dtype = torch.float32 if residual is not None else torch.bfloat16 if self.quantised else getattr(x, "out_dtype", None) or x.dtype
        if self.quantised:
            if self.runtime.row_bits == 8 and not isinstance(x, ops.Q8Rows):
                x = ops.quantize_q8(x.materialize() if isinstance(x, ops.NormedInput) else x)
            return ops.linear_q4(x, self.weight, self.bias, act=act, residual=residual, out=out, out_dtype=out_dtype)
        return ops.linear(x, self.weight, self.bias, act=act, residual=residual, out=out, out_dtype=out_dtype)
