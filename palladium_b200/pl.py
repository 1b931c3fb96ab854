"""Stand-ins for the two Pallas / JAX types a `pallas_call`-shaped signature
mentions, for environments without JAX: `BlockSpec(block_shape, index_map)` and
`ShapeDtypeStruct(shape, dtype)`.  `cuda_call` reads both by attribute
(`block_shape`, `index_map`, `shape`, `dtype`), so the real
`jax.experimental.pallas.BlockSpec` and `jax.ShapeDtypeStruct` work as well.

NumPy has no bfloat16; `bfloat16` here is a two-byte dtype that stands for it, so
that a call can name the element type and host arrays can carry its bits
(`array.view(pl.bfloat16)` of a uint16 array).  `as_dtype` reads it from what
else means the same: the name, torch's or ml_dtypes' type."""

from __future__ import annotations

import dataclasses
from collections.abc import Callable

import numpy as np

__all__ = ["BlockSpec", "ShapeDtypeStruct", "as_dtype", "bfloat16", "dtype_name"]

bfloat16 = np.dtype([("bfloat16", np.uint16)])
_NAMES: dict[np.dtype, str] = {}


def as_dtype(dtype) -> np.dtype:
    """`np.dtype(dtype)`, with every way of writing bfloat16 read as `pl.bfloat16`."""
    if isinstance(dtype, np.dtype) and dtype.kind != "V":
        return dtype        # (what every call on host arrays asks for each of them; ml_dtypes' types are of kind V)
    if str(dtype).rsplit(".", 1)[-1] == "bfloat16" or getattr(dtype, "__name__", "") == "bfloat16":
        return bfloat16
    try:
        return np.dtype(dtype)
    except TypeError:
        return np.dtype(str(dtype).rsplit(".", 1)[-1])      # a torch dtype: "torch.float32"


def dtype_name(dtype: np.dtype) -> str:
    if dtype.kind == "V" and dtype == bfloat16:
        return "bfloat16"
    name = _NAMES.get(dtype)
    if name is None:
        name = _NAMES[dtype] = dtype.name      # (NumPy spells it out anew each time, 4 us)
    return name


@dataclasses.dataclass(frozen=True)
class BlockSpec:
    block_shape: tuple[int, ...] | None = None
    index_map: Callable[..., tuple] | None = None

    def __post_init__(self):
        if self.block_shape is not None:
            object.__setattr__(self, "block_shape", tuple(int(b) for b in self.block_shape))


@dataclasses.dataclass(frozen=True)
class ShapeDtypeStruct:
    shape: tuple[int, ...]
    dtype: np.dtype

    def __post_init__(self):
        object.__setattr__(self, "shape", tuple(int(s) for s in self.shape))
        object.__setattr__(self, "dtype", as_dtype(self.dtype))
