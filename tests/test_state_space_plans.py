"""How calls of the state-space families are cut into blocks, and what a call costs before its launch, without a GPU."""

import timeit

import numpy as np
import pytest

import palladium_b200 as pd
from palladium_b200 import families, pl
from tests.oracle_provider import interpret
from tests.state_space import Case, check


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


@pytest.mark.parametrize("length, channels, most", [(131072, 16, 181), (32768, 64, 90), (2 ** 20, 16, 512), (8192, 2048, 16)])
def test_segments_of_a_long_prompt_over_few_channels(length, channels, most):
    """A block composes the states of all segments before its own: half the root of the length is what pays."""
    diag = explain(families.selective_scan(length, 16, dtype="bfloat16"), (1, channels))
    tiles = -(-channels // 16)
    assert diag.launches == 2 and most // 2 <= diag.cuda_grid[0] // tiles <= most


# ------------------------------------------------------------------ constants
@pytest.mark.parametrize("length", [float("nan"), float("inf"), -float("inf"), None, "eight", "8", [8], True, 8.5, 2 ** 31])
def test_lengths_that_are_no_whole_numbers_are_refused(length):
    for make in (families.causal_conv, families.selective_scan_grad):
        with pytest.raises(pd.TraceError, match="length must be a whole number"):
            make(length)
    assert families.causal_conv(np.int64(8)).constants["length"] == families.causal_conv(8.0).constants["length"] == 8


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


# ------------------------------------------------------------------ what explain says of a call's resources
SCANS = [("bfloat16", 4, 2), ("bfloat16", 8, 4), ("bfloat16", 16, 5), ("bfloat16", 32, 5), ("bfloat16", 64, 3),
         ("float32", 4, 1), ("float32", 8, 2), ("float32", 16, 4), ("float32", 32, 4), ("float32", 64, 2)]


@pytest.mark.parametrize("dtype, state, blocks", SCANS)
def test_shared_memory_of_the_prompt_kernel(dtype, state, blocks):
    """An SM's 228 KB hold that many blocks, each with 1 KB of its own, or five where it would hold more."""
    diag = explain(families.selective_scan(512, state, gate=True, dtype=dtype), (2, 96))
    fit = 228 * 1024 // (diag.dynamic_smem_bytes + 1024)
    assert min(fit, 5) == blocks and diag.dynamic_smem_bytes <= 227 * 1024


def test_shared_memory_of_the_gradients_and_steps():
    for state in (1, 4, 5, 8, 16, 17, 33, 64):
        for dtype in ("float32", "bfloat16"):
            for grid in ((1, 8), (40, 250), (120, 63)):
                diag = explain(families.selective_scan_grad(9, state, gate=True, dtype=dtype), grid)
                assert 0 < diag.dynamic_smem_bytes <= 227 * 1024
    assert explain(families.causal_conv_grad(9), (2, 8)).dynamic_smem_bytes == 4096
    assert explain(families.causal_conv_grad(9), (2, 7)).dynamic_smem_bytes == 1024
    for family in (families.causal_conv(9), families.causal_conv_step(), families.selective_scan_step(16)):
        assert explain(family, (2, 8)).dynamic_smem_bytes == 0


@pytest.mark.gpu
@pytest.mark.parametrize("math_mode", ["safe", "relaxed", "fast"])
@pytest.mark.parametrize("dtype, state, blocks", SCANS)
def test_blocks_of_the_prompt_kernel_on_a_multiprocessor(dtype, state, blocks, math_mode):
    """Its registers leave room for as many blocks as its shared memory does."""
    diag = explain(families.selective_scan(512, state, gate=True, dtype=dtype), (2, 96), math_mode)
    assert diag.blocks_per_sm == blocks and 0 < diag.regs <= 255 and diag.smem_bytes == 0
    assert f"smem=0+{diag.dynamic_smem_bytes} blocks_per_sm={blocks}" in str(diag)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_registers_and_blocks_of_every_form(packed):
    for family in (families.causal_conv(40, packed=packed), families.causal_conv_grad(40, silu=False, packed=packed),
                   families.causal_conv_step(3, dtype="float16"), families.selective_scan_step(5, dtype="bfloat16"),
                   families.selective_scan(40, 24, packed=packed, initial=True, final=True, carries=True),
                   families.selective_scan_grad(40, 24, packed=packed, initial=True, final=True, gate=True)):
        for grid in ((3, 20), (0, 20)):
            diag = explain(family, grid)
            assert 0 < diag.regs <= 255 and diag.blocks_per_sm >= 1 and diag.smem_bytes == 0, (family.name, grid)


# ------------------------------------------------------------------ interpret
@pytest.fixture
def provider():
    previous = pd.register_interpret_provider(interpret)
    yield
    pd.register_interpret_provider(previous)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind", ["conv", "scan"])
@pytest.mark.parametrize("packed", [False, True])
def test_interpret_reaches_prompts_and_gradients(provider, packed, kind, dtype):
    more = dict(state=3, groups=2, gate=True) if kind == "scan" else {}
    case = Case(kind, [70, 0, 33] if packed else [40, 40], 4, dtype=dtype, packed=packed, lead=2 * packed, spare=packed,
                initial=True, final=True, **more)
    call = case.call(pd.cuda_call, **({"carries": True} if kind == "scan" else {}))
    forward = list(call.interpret(*case.operands()))
    carries = forward.pop() if kind == "scan" else None
    check(case, case.forward_names(), forward)
    # (the gradient starts from the carries, float32, so from the initial state itself)
    check(case, case.grad_names(), case.call(pd.cuda_call_jit, "_grad").interpret(*case.operands(grad=True, carries=carries)))


@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_interpret_reaches_single_tokens(provider, kind):
    case = Case(kind, [1] * 5, 4, initial=True, final=True, **(dict(state=3, gate=True) if kind == "scan" else {}))
    if kind == "conv":
        family, order = families.causal_conv_step(), ["x", "initial", "weight", "bias"]
    else:
        family = families.selective_scan_step(3, gate=True)
        order = ["initial", "x", "delta", "A", "B", "C", "bias", "skip", "z"]
    operands = [case.typed(n) for n in order]
    operands = [a.reshape(a.shape[:1] + a.shape[2:]) if n in ("x", "delta", "B", "C", "z") else a for n, a in zip(order, operands)]
    call = pd.cuda_call(family, grid=case.grid, out_shape=families.out_shapes(family, case.grid))
    check(case, ["y", "final"], call.interpret(*operands), case.oracle(grad=False))
