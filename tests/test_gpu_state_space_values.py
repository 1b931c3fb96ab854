"""Values of the state-space families where float32's range or a rounding decides, on a GPU against the float64
operators inside the bounds of their running error analysis."""

import numpy as np
import pytest

import palladium_b200 as pd
from tests.state_space import Case, check
from tests.test_gpu_state_space import compare, run

pytestmark = pytest.mark.gpu

MODES = ["safe", "relaxed", "fast"]


# ------------------------------------------------------------------ rates and states at the ends of float32's range
@pytest.mark.parametrize("math_mode", MODES)
@pytest.mark.parametrize("packed", [False, True])
def test_cut_sequence_whose_zero_states_grow(math_mode, packed):
    """Growing rates and no input until the last tokens: every state is zero until then, however the call is cut."""
    case = Case("scan", [512] if not packed else [40, 512, 3], 12, packed=packed, state=16, softplus=False, bias=False,
                final=True)
    case.v["A"][:] = 2.0
    case.v["delta"][:] = 1.0
    case.v["x"][:] = 0.0
    end = case.starts[1 if not packed else 2]
    case.v["x"][end - 10:end] = 1.0
    assert case.call(pd.cuda_call).explain(*case.operands()).launches == 2
    forward, _ = run(case, math_mode, grad=False)
    check(case, case.forward_names(), forward, case.oracle(grad=False))


@pytest.mark.parametrize("math_mode", MODES)
@pytest.mark.parametrize("rate, entering", [(1.5, 1e-30), (-1.5, 1e30)])
def test_cut_sequence_whose_factor_leaves_the_range(math_mode, rate, entering):
    """A segment's factor e^96 (or its inverse) is outside float32, the state behind it is not."""
    case = Case("scan", [128], 12, state=16, softplus=False, bias=False, initial=True, final=True)
    case.v["A"][:] = rate
    case.v["delta"][:] = 0.0
    case.v["delta"][:64] = 1.0
    case.v["x"][:] = 0.0
    case.v["initial"][:] = np.float32(entering)
    assert case.call(pd.cuda_call).explain(*case.operands()).launches == 2
    forward, _ = run(case, math_mode, grad=False)
    check(case, case.forward_names(), forward, case.oracle(grad=False))


@pytest.mark.parametrize("math_mode", MODES)
@pytest.mark.parametrize("state", [3, 7, 16, 24])
@pytest.mark.parametrize("rate", [1.0, 5.0, 6.0, 20.0])
def test_gradient_through_tokens_whose_decays_grow(math_mode, state, rate):
    """In every other channel tokens 10 to 39 grow by e^rate each, no state enters them and no gradient comes back to
    them: products of their factors pass float32's range from rates of 5.5 on, states and gradients do not."""
    case = Case("scan", [70, 70], 6, state=state, softplus=False, bias=False, gate=True)
    case.v["A"][::2] = rate
    for name, rows in (("delta", slice(10, 40)), ("x", slice(0, 40)), ("dy", slice(10, 70))):
        every = case.v[name].reshape(2, 70, 6)[:, :, ::2]
        if name == "delta":
            every[:] = 2.0 ** -7
        every[:, rows] = 1.0 if name == "delta" else 0.0
    compare(case, math_mode)
