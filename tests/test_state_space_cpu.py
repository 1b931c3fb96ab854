"""The state-space families without a GPU: the oracle's gradients against differences, shapes and operand
order, refusals."""

import ctypes

import numpy as np
import pytest

import palladium_b200 as pd
from oracle import state_space as S
from palladium_b200 import DispatchError, TraceError, _native, families, pl
from tests.state_space import Case, host, rounded, wide


# ------------------------------------------------------------------ the oracle itself
@pytest.mark.parametrize("kind", ["conv", "scan"])
@pytest.mark.parametrize("plain", [False, True])
def test_oracle_gradients_match_differences(kind, plain):
    more = dict(width=3, silu=not plain) if kind == "conv" else dict(state=3, groups=2, softplus=not plain, gate=not plain)
    case = Case(kind, [3, 0, 1, 5], 4, packed=True, spare=2, lead=1, initial=True, final=True, seed=3, **more)
    want = case.oracle()

    def value():
        out = case.oracle(grad=False)
        return float((out["y"].value * case.v["dy"]).sum() + (out["final"].value * case.v["dfinal"]).sum())

    names = case.grad_names()
    for name in names:
        operand = case.v[name[1:]]
        got, step = want[name].value, 1e-6
        for at in np.ndindex(operand.shape):
            keep = operand[at]
            operand[at] = keep + step
            up = value()
            operand[at] = keep - step
            down = value()
            operand[at] = keep
            # central difference: truncation step^2 times a third derivative of order 10^3 at most, rounding
            # 2^-52 * |value| / step with |value| < 10^3
            assert abs((up - down) / (2 * step) - got[at]) < 2e-6, (name, at)


def test_running_bound_covers_a_float32_evaluation():
    # the same recurrence in NumPy float32 stays inside the bound
    case = Case("scan", [200], 3, state=4, seed=5, skip=False)
    v, want = case.v, case.oracle(grad=False)
    f = {k: a.astype(np.float32) for k, a in v.items()}
    h = np.zeros((3, 4), np.float32)
    for t in range(200):
        raw = f["delta"][t] + f["bias"]
        d = np.maximum(raw, np.float32(0)) + np.log1p(np.exp(-np.abs(raw)))
        h = np.exp(d[:, None] * f["A"]) * h + (d * f["x"][t])[:, None] * f["B"][t]
        y = (h * f["C"][t]).sum(1, dtype=np.float32)
        assert (np.abs(y - want["y"].value[t]) <= S.UNIT * want["y"].error[t]).all()
    # and it is a bound worth having: below 1e-4 of the largest state
    assert (S.UNIT * want["final"].error).max() < 1e-4 * np.abs(want["final"].value).max()


def test_rounding_helpers():
    assert rounded(1 + 2.0 ** -8, "bfloat16") == 1.0 and rounded(1 + 3 * 2.0 ** -8, "bfloat16") == 1 + 2.0 ** -6
    values = rounded(np.linspace(-3, 3, 17), "bfloat16")
    assert np.array_equal(wide(host(values, "bfloat16")), values)


# ------------------------------------------------------------------ shapes and types
def test_bfloat16_names():
    import torch

    assert pl.as_dtype("bfloat16") == pl.as_dtype(torch.bfloat16) == pl.bfloat16
    assert pl.dtype_name(pl.bfloat16) == "bfloat16" and pl.as_dtype(torch.float16) == np.float16
    assert pl.ShapeDtypeStruct((2,), "bfloat16").dtype == pl.bfloat16
    for kind in ("bfloat16", pl.bfloat16, torch.bfloat16):
        assert families.causal_conv(4, dtype=kind).constants["dtype"] == "bfloat16"


def test_out_shapes_and_operands():
    fam = families.selective_scan(130, 5, groups=2, gate=True, initial=True, final=True, carries=True, dtype="float16")
    y, final, carries = families.out_shapes(fam, (3, 8))
    assert y.shape == (3, 130, 8) and y.dtype == np.float16
    assert final.shape == (3, 8, 5) and carries.shape == (3, -(-130 // families.SCAN_CHUNK), 8, 5) and carries.dtype == np.float32
    packed = families.selective_scan(130, 5, carries=True, packed=True)
    assert families.out_shapes(packed, (7, 8))[1].shape == (130 // families.SCAN_CHUNK + 7, 8, 5)
    grad = families.selective_scan_grad(130, 5, groups=2, gate=True, initial=True, final=True)
    assert [o.shape for o in families.out_shapes(grad, (3, 8))] == [
        (3, 130, 8), (3, 130, 8), (8, 5), (3, 130, 2, 5), (3, 130, 2, 5), (8,), (8,), (3, 130, 8), (3, 8, 5)]
    assert families.out_shapes(families.causal_conv(9), (2, 3)).shape == (2, 9, 3)
    step = families.out_shapes(families.causal_conv_step(3), (2, 5))
    assert [o.shape for o in step] == [(2, 5), (2, 2, 5)]
    with pytest.raises(TraceError, match="out_shapes knows"):
        families.out_shapes(families.lv_rk4(), (3,))


@pytest.mark.parametrize("kind", ["conv", "scan"])
@pytest.mark.parametrize("packed", [False, True])
def test_explain_takes_every_operand(kind, packed):
    case = Case(kind, [5, 5] if not packed else [5, 2], 6, packed=packed, initial=True, final=True, dtype="bfloat16",
                **({} if kind == "conv" else dict(gate=True, groups=3)))
    diag = case.call(pd.cuda_call).explain(*case.operands())
    assert diag.grid == (2, 6) and diag.launches >= 1 and "kernel" in diag.cuda_kernel and diag.msl_lines > 0
    carries = None
    if kind == "scan":
        carries = pl.ShapeDtypeStruct(families.out_shapes(case.family(carries=True), case.grid)[2].shape, np.float32)
    grad = case.call(pd.cuda_call, "_grad").explain(*case.operands(grad=True, carries=carries))
    assert grad.scratch_bytes > 0
    assert "pd_scan.cu" in pd.debug_msl(case.family(), grid=case.grid, out_shape=families.out_shapes(case.family(), case.grid))


def test_in_specs_are_checked():
    fam = families.selective_scan(10, 4, groups=2, bias=False, skip=False)
    specs = [pl.BlockSpec((1, 10, 1), lambda i, j: (i, 0, j))] * 2 + [pl.BlockSpec((1, 4), lambda i, j: (j, 0))] + \
            [pl.BlockSpec((1, 10, 1, 4), lambda i, j: (i, 0, j // 3, 0))] * 2
    pd.cuda_call(fam, grid=(2, 6), in_specs=specs, out_shape=families.out_shapes(fam, (2, 6)))
    specs[3] = pl.BlockSpec((1, 10, 1, 4), lambda i, j: (i, 0, 0, 0))
    with pytest.raises(TraceError, match="index_map"):
        pd.cuda_call(fam, grid=(2, 6), in_specs=specs, out_shape=families.out_shapes(fam, (2, 6)))


# ------------------------------------------------------------------ refusals
@pytest.mark.parametrize("make, words", [
    (lambda: families.causal_conv(8, 5), "width must be"),
    (lambda: families.causal_conv(8, 1), "width must be"),
    (lambda: families.causal_conv(-1), "length must be"),
    (lambda: families.causal_conv(2.5), "length must be"),
    (lambda: families.causal_conv(8, dtype="float64"), "dtype must be one of"),
    (lambda: families.selective_scan(8, 0), "state must be"),
    (lambda: families.selective_scan(8, 65), "state must be"),
    (lambda: families.selective_scan(8, 16, groups=0), "groups must be"),
    (lambda: families.selective_scan_step(True), "state must be"),
])
def test_constants_are_checked(make, words):
    with pytest.raises(TraceError, match=words):
        make()


def test_call_descriptions_are_checked():
    fam = families.selective_scan(8, 4, groups=3)
    with pytest.raises(TraceError, match="do not divide into 3 groups"):
        families.out_shapes(fam, (2, 8))
    with pytest.raises(TraceError, match=r"grid must be \(sequences, channels\)"):
        pd.cuda_call(families.causal_conv(8), grid=(4,), out_shape=pl.ShapeDtypeStruct((4, 8), np.float32))
    with pytest.raises(TraceError, match="at least one channel"):
        families.out_shapes(families.causal_conv(8), (4, 0))
    with pytest.raises(TraceError, match="the kernel family produces"):
        pd.cuda_call(families.causal_conv(8, dtype="float16"), grid=(2, 3), out_shape=pl.ShapeDtypeStruct((2, 8, 3), np.float32))


def test_argument_types_are_checked():
    case = Case("conv", [4, 4], 3, dtype="bfloat16")
    call = case.call(pd.cuda_call)
    good = case.operands()
    with pytest.raises(DispatchError, match="dtype float32 does not match the traced bfloat16"):
        call.explain(good[0].view(np.uint16).astype(np.float32), *good[1:])
    with pytest.raises(TraceError, match="takes 3 arrays, got 2"):
        call.explain(*good[:2])
    with pytest.raises(DispatchError, match="argument 1 has dtype float64"):
        call.explain(good[0], good[1].astype(np.float64), good[2])
    # the trajectory families still take float32 alone
    lv = pd.cuda_call(families.lv_rk4(), grid=(4,), out_shape=(pl.ShapeDtypeStruct((4,), np.float32),) * 2)
    with pytest.raises(DispatchError, match="float16, which palladium cannot lower"):
        lv.explain(*[np.zeros(4, np.float16)] * 6)


def _explain(family, params, grid, block=None):
    return _native.explain(family, params, 2, grid, block)


@pytest.mark.parametrize("fields, grid, words", [
    (dict(type=3), (2, 8), "type must be"),
    (dict(width=7), (2, 8), "width must lie"),
    (dict(length=-1), (2, 8), "length must lie"),
    (dict(length=2 ** 31), (2, 8), "length must lie"),
    (dict(silu=2), (2, 8), "flags must be"),
    (dict(), (2, 0), "channels"),
    (dict(), (2, 8, 2), "grid must be"),
    (dict(length=2 ** 31 - 1), (2 ** 31 - 1, 2 ** 20), "2\\^40 elements"),
])
def test_native_conv_refusals(fields, grid, words):
    base = dict(length=4, width=4, type=0, silu=1, bias=1, initial=0, final=0, packed=0)
    for family in (10, 12):
        with pytest.raises(DispatchError, match=words):
            _explain(family, _native.CausalConvParams(*{**base, **fields}.values()), grid)


@pytest.mark.parametrize("fields, grid, words", [
    (dict(state=0), (2, 8), "state must lie"),
    (dict(state=65), (2, 8), "state must lie"),
    (dict(groups=3), (2, 8), "do not divide"),
    (dict(groups=0), (2, 8), "do not divide"),
    (dict(groups=70000), (2, 70000), "65535 groups"),
    (dict(gate=-1), (2, 8), "flags must be"),
    (dict(packed=2), (2, 8), "flags must be"),
])
def test_native_scan_refusals(fields, grid, words):
    base = dict(length=4, state=16, groups=1, type=0, softplus=1, bias=1, skip=1, gate=0, initial=0, final=0, carries=0, packed=0)
    for family in (13, 14, 15):
        with pytest.raises(DispatchError, match=words):
            _explain(family, _native.SelectiveScanParams(*{**base, **fields}.values()), grid)


def test_native_params_and_threadgroup():
    conv = _native.CausalConvParams(4, 4, 0, 1, 1, 0, 0, 0)
    with pytest.raises(DispatchError, match="params block must be 96 bytes"):
        _explain(13, conv, (2, 8))
    with pytest.raises(DispatchError, match="leave it unset"):
        _explain(10, conv, (2, 8), 128)
    with pytest.raises(DispatchError, match="math_mode out of range"):
        _native.explain(10, conv, 5, (2, 8), None)


def test_native_params_layout_matches_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parent.parent / "include" / "palladium_cuda.h").read_text()
    for name, kind in (("pd_causal_conv_params", _native.CausalConvParams), ("pd_selective_scan_params", _native.SelectiveScanParams)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = [f.strip() for line in re.findall(r"int64_t ([^;]+);", body) for f in line.split(",")]
        assert fields == [f for f, _ in kind._fields_] and ctypes.sizeof(kind) == 8 * len(fields)
    assert int(re.search(r"#define PD_SCAN_CHUNK (\d+)", text).group(1)) == families.SCAN_CHUNK
