"""Rows of values in 8 bits with one float32 scale a row.

    scale = max(amax * rn(1 / most), 2^-126),   code = rn(value * rn(1 / scale)),   value read back = code * scale

``most`` is 448 for ``"e4m3"`` (codes are ``torch.float8_e4m3fn``) and 127 for ``"int8"``.  A value of an int8 row is
off by at most half a scale, one of an e4m3 row by 2^-4 of itself (or half of the smallest code's step, 2^-10 scales,
below 2^-6 scales); both in addition to a few roundings of float32.  A row that holds an infinity or a NaN reads back
as NaN throughout.  ``ash.HashMap(value_formats=...)`` keeps its rows this way, ``ash.mlp.rms_norm(quantize=True)``
writes such rows and ``ash.mlp.fused_linear`` multiplies them.
"""
from typing import NamedTuple, Optional

import torch

from .common import _get_c_extension

backend = _get_c_extension()

FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
VALUE_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class QuantizedRows(NamedTuple):
    """``codes`` (..., width), float8_e4m3fn or int8, and ``scales`` (...,), float32."""

    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def format(self) -> str:
        for name, dtype in FORMATS.items():
            if self.codes.dtype == dtype:
                return name
        raise ValueError(f"codes must be float8_e4m3fn or int8, got {self.codes.dtype}")

    def check(self, name: str = "rows") -> "QuantizedRows":
        """Raise unless codes and scales belong together."""
        if not isinstance(self.codes, torch.Tensor) or not isinstance(self.scales, torch.Tensor):
            raise ValueError(f"{name}: codes and scales must be tensors")
        self.format
        if self.codes.dim() < 1 or self.codes.shape[:-1] != self.scales.shape:
            raise ValueError(f"{name}: a scale a row is wanted, got codes {tuple(self.codes.shape)} and scales "
                             f"{tuple(self.scales.shape)}")
        if self.scales.dtype != torch.float32:
            raise ValueError(f"{name}: scales must be float32, got {self.scales.dtype}")
        if self.codes.device != self.scales.device:
            raise ValueError(f"{name}: codes on {self.codes.device}, scales on {self.scales.device}")
        return self


def check_format(format: str) -> str:
    if format not in FORMATS:
        raise ValueError(f"format must be one of {sorted(FORMATS)}, got {format!r}")
    return format


def quantize_rows(x: torch.Tensor, format: str = "e4m3") -> QuantizedRows:
    """The rows of ``x`` (..., width) -- float32, float16 or bfloat16 -- in 8 bits.  Not differentiable."""
    check_format(format)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have rows of at least one value, got {tuple(x.shape)}")
    if x.dtype not in VALUE_TYPES:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    return QuantizedRows(*backend.quantize_rows(x, FORMATS[format]))


def dequantize_rows(rows: QuantizedRows, indices: Optional[torch.Tensor] = None,
                    dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """What the rows read back as, (..., width); with ``indices`` (int64, any shape) those of 2-D ``rows``, zeros for an
    index outside 0 .. rows - 1."""
    rows.check()
    if dtype not in VALUE_TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    if indices is not None:
        if rows.codes.dim() != 2:
            raise ValueError(f"indexed rows must be 2-D, got {tuple(rows.codes.shape)}")
        if indices.dtype != torch.int64 or indices.device != rows.codes.device:
            raise ValueError(f"indices must be int64 on {rows.codes.device}, got {indices.dtype} on {indices.device}")
    return backend.read_rows(rows.codes, rows.scales, indices, dtype)
