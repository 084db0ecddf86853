"""What every part is given when it is bound: dtype, device, kernels."""
from __future__ import annotations

from dataclasses import dataclass

import torch

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


_ops = None            # the kernel module, imported when first asked for


@dataclass
class Runtime:
    """``dtype`` is the compute dtype: bfloat16 (the serving path: bfloat16
    weights, activations and cache, float32 accumulation, norms, softmax and
    residual stream) or float32 (everything in true 32-bit: products by float32
    multiply-adds or, over a long k, on tensor cores from operands cut into
    three bfloat16 numbers that are together exactly them, with an error no
    larger than the multiply-adds').

    ``weight_bits`` 4 (bfloat16 only): the layers' matrices are held in 4 bits
    with a power-of-two scale for every 32 (``ops.quantize_q4``, made when a part
    is bound); tables, the output head, the experts' and the per-head matrices
    stay as they are.  ``row_bits`` 8 (with 4-bit weights): the rows that meet them
    are taken in 8 bits too, by the norm that makes them where it can."""
    dtype: torch.dtype
    device: torch.device
    weight_bits: int = 16
    row_bits: int = 16
    saved_bytes: int = 0            # what the 4-bit matrices take less than they did

    @property
    def ops(self):
        global _ops
        if _ops is None:
            from ..csrc import ops
            _ops = ops
        return _ops

    @property
    def is_fp32(self) -> bool:
        return self.dtype == torch.float32

    @classmethod
    def create(cls, dtype, device="cuda:0", weight_bits: int = 16, row_bits: int = 16) -> "Runtime":
        if isinstance(dtype, str):
            if dtype not in DTYPES:
                raise ValueError(f"dtype must be one of {', '.join(DTYPES)}, got '{dtype}'")
            dtype = DTYPES[dtype]
        if dtype not in DTYPES.values():
            raise ValueError(f"dtype must be bfloat16 or float32, got {dtype}")
        if weight_bits not in (16, 4) or row_bits not in (16, 8):
            raise ValueError(f"weights take 16 or 4 bits and rows 16 or 8, got {weight_bits} and {row_bits}")
        if weight_bits == 4 and dtype != torch.bfloat16:
            raise ValueError("4-bit weights go with dtype bfloat16")
        if row_bits == 8 and weight_bits != 4:
            raise ValueError("8-bit rows go with 4-bit weights")
        return cls(dtype=dtype, device=torch.device(device), weight_bits=weight_bits, row_bits=row_bits)
