"""How calls of the state-space families are cut into blocks: what `explain` says of them, without a GPU."""

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
