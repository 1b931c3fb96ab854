"""How calls of the state-space families are cut into blocks, and what a call costs before its launch, without a GPU."""

import timeit

import numpy as np
import pytest

import palladium_b200 as pd
from palladium_b200 import families, pl


def explain(family, grid, math_mode="fast"):
    call = pd.cuda_call(family, grid=grid, out_shape=families.out_shapes(family, grid), math_mode=math_mode)
    operands = [pl.ShapeDtypeStruct(info.array_shape, info.dtype) for _, info, _ in families._scan_operands(family, grid)[0]]
    return call.explain(*operands)


@pytest.mark.parametrize("dtype, state, grid, length, most", [
    # more channels a warp would leave two blocks on an SM instead of three, or one instead of two
    ("float32", 16, (4, 2048), 2048, 4), ("float32", 16, (8, 1024), 1024, 4), ("float32", 16, (2, 5120), 1024, 4),
    ("float16", 32, (16, 1536), 256, 3), ("float32", 32, (4, 2048), 2048, 4), ("float32", 64, (16, 1536), 256, 3),
    # and where three fit, the rule stands
    ("bfloat16", 16, (4, 2048), 2048, 6), ("bfloat16", 8, (2, 5120), 1024, 6), ("float32", 4, (4, 2048), 2048, 6),
])
def test_channels_per_warp_of_the_gradient_fit_the_multiprocessor(dtype, state, grid, length, most):
    diag = explain(families.selective_scan_grad(length, state, gate=True, dtype=dtype), grid)
    assert 2 <= diag.items_per_thread <= most


# ------------------------------------------------------------------ what every call pays
def test_reading_an_element_type_costs_little():
    """Every call on host arrays, of any family, reads each operand's type: spelling the type out for it once cost
    6 us an operand (str of a NumPy type takes about 3), on calls of 50 us."""
    kind = np.zeros(1, np.float32).dtype
    best = lambda f: min(timeit.repeat(f, number=2000, repeat=7))  # noqa: E731
    assert best(lambda: pl.dtype_name(pl.as_dtype(kind))) < best(lambda: str(kind)) / 2
    assert pl.as_dtype(kind) is kind and pl.dtype_name(kind) == "float32"


def test_element_types_are_still_told_apart():
    ml_dtypes = pytest.importorskip("ml_dtypes")
    assert pl.as_dtype(np.dtype(ml_dtypes.bfloat16)) == pl.bfloat16
    assert pl.as_dtype(pl.bfloat16) == pl.bfloat16 and pl.dtype_name(pl.bfloat16) == "bfloat16"
    record = np.dtype([("a", np.uint16)])
    assert pl.as_dtype(record) == record and pl.dtype_name(record) != "bfloat16"
    for kind in (np.float32, np.uint32, np.int32, np.float64, np.float16, np.uint8, np.dtype(">f4")):
        assert pl.dtype_name(pl.as_dtype(kind)) == np.dtype(kind).name
