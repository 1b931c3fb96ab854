"""Kernel families: what takes the place of a Pallas kernel function.

The reference traces an arbitrary Pallas function into a `KernelSpec` and emits
MSL for it (src/palladium/trace.py:117-178, src/palladium/emit/core.py:383-466).
This package has no emitter: the five integrator kernels are hand-written CUDA,
and `cuda_call(kernel, ...)` takes a *family descriptor* as its `kernel`
argument.  A descriptor names the family, carries the constants the reference
kernels close over as module globals (DT, STEPS, tolerances, ...), and checks
that the `grid` / `in_specs` / `out_specs` / `out_shape` of the call describe
the launch that family performs -- the same keywords, with the same meaning, a
user of the reference already writes for `metal_call`.

Two families are open-ended and compiled at run time, as the reference compiles
the MSL it emits: `custom_ode` (a right-hand side of the caller's inside the
library's RK4 or adaptive loop) and `source_kernel` (a complete CUDA kernel of
the caller's).

The state-space families (`causal_conv`, `selective_scan` and their `_step` and
`_grad` forms) integrate ensembles of driven linear systems over sequences of
tokens; they are not in the reference.

`trace(family, call_kwargs, *args)` produces the `KernelSpec` analogue: name,
grid, and one `BlockInfo` per operand.
"""

from __future__ import annotations

import ctypes
import dataclasses
from collections.abc import Callable, Sequence
from typing import Any

import numpy as np

from . import _native
from .errors import DispatchError, TraceError, UnsupportedPrimitiveError
from .pl import ShapeDtypeStruct, as_dtype, bfloat16, dtype_name

__all__ = [
    "BlockInfo",
    "Family",
    "KernelSpec",
    "SCAN_CHUNK",
    "STATE_SPACE",
    "causal_conv",
    "causal_conv_grad",
    "causal_conv_step",
    "custom_ode",
    "gbm_pcg",
    "gbm_threefry",
    "gray_scott",
    "kepler_rk4_df32",
    "lv_rk4",
    "lv_rk4_df32",
    "out_shapes",
    "selective_scan",
    "selective_scan_grad",
    "selective_scan_step",
    "source_kernel",
    "threefry_bits",
    "trace",
    "vdp_bs32",
    "vdp_cost_order",
]

F32 = np.dtype(np.float32)
U32 = np.dtype(np.uint32)
I32 = np.dtype(np.int32)
F64 = np.dtype(np.float64)


@dataclasses.dataclass(frozen=True)
class BlockInfo:
    """One operand of a traced call (src/palladium/trace.py:26-50)."""

    block_shape: tuple[int, ...]
    array_shape: tuple[int, ...]
    dtype: np.dtype


@dataclasses.dataclass(frozen=True)
class KernelSpec:
    """A validated call: the analogue of the reference's traced KernelSpec
    (src/palladium/trace.py:53-80) with the family in place of a jaxpr."""

    name: str
    family: "Family"
    grid: tuple[int, ...]
    inputs: tuple[BlockInfo, ...]
    outputs: tuple[BlockInfo, ...]
    params: ctypes.Structure

    @property
    def num_programs(self) -> int:
        return int(np.prod(self.grid)) if self.grid else 1


@dataclasses.dataclass(frozen=True)
class Family:
    """A hand-written kernel family plus the constants of one problem.

    `pallas_fn`, when given and JAX is installed, is the user's own Pallas
    kernel function for the same computation; `.interpret` then runs it through
    `pl.pallas_call(..., interpret=True)` exactly as the reference does."""

    name: str
    constants: dict[str, Any]
    pallas_fn: Callable | None = None

    @property
    def family_id(self) -> int:
        return _native.FAMILY_IDS[self.name]

    def __call__(self, *refs):
        raise UnsupportedPrimitiveError(
            f"{self.name} is a hand-written CUDA kernel family, not a Pallas function; "
            "pass it to palladium_b200.cuda_call instead of calling it"
        )


# ----------------------------------------------------------------------------- constructors
def lv_rk4(dt: float = 0.01, steps: int = 500, pallas_fn: Callable | None = None) -> Family:
    """Fixed-step RK4 Lotka-Volterra ensemble (examples/01_ode_ensembles.py:72-91).
    Call signature: grid=(N,), six (N,) float32 inputs x0, y0, a, b, c, d,
    two (N,) float32 outputs, or a single (N, 2) float32 output holding the
    final (x, y) pairs."""
    return Family("lv_rk4", dict(dt=float(dt), steps=int(steps)), pallas_fn)


def vdp_bs32(t1: float = 10.0, rtol: float = 1e-5, atol: float = 1e-7, dt0: float = 0.01,
             max_steps: int = 6000, pcoeff: float = 0.4, icoeff: float = 0.3, safety: float = 0.9,
             factor_min: float = 0.2, factor_max: float = 10.0, error_order: int = 3,
             pallas_fn: Callable | None = None) -> Family:
    """Adaptive Bogacki-Shampine 3(2) Van der Pol ensemble
    (examples/02_adaptive_lockstep.py:69-171; defaults from :20-32).
    grid=(N,), inputs x0, v0, mu.  The output layout follows `out_shape`:
    six float32 (N,) arrays t, x, v, steps, rejected, real; five (without
    `real`, tests/test_08_adaptive.py:33-142); or an (N, 2) float32 state plus
    int32 accepted and rejected counts."""
    return Family("vdp_bs32", dict(t1=float(t1), rtol=float(rtol), atol=float(atol), dt0=float(dt0),
                                   max_steps=int(max_steps), pcoeff=float(pcoeff), icoeff=float(icoeff),
                                   safety=float(safety), factor_min=float(factor_min),
                                   factor_max=float(factor_max), error_order=int(error_order)), pallas_fn)


_CHECKED_SOURCES: set = set()


_ODE_METHODS = {"rk4": 0, "bs32": 1, "dopri5": 2, "tsit5": 3}


def custom_ode(rhs: str, dim: int, nparam: int = 0, *, method: str = "rk4", dt: float = 0.01, steps: int = 500,
               t1: float = 10.0, rtol: float = 1e-5, atol: float = 1e-7, dt0: float = 0.01, max_steps: int = 6000,
               pcoeff: float = 0.4, icoeff: float = 0.3, safety: float = 0.9, factor_min: float = 0.2,
               factor_max: float = 10.0, error_order: int | None = None, check: bool = True,
               pallas_fn: Callable | None = None) -> Family:
    """An ensemble of independent systems y' = f(t, y, p) with a right-hand side
    of the caller's: the open end of the family set, where the reference lets a
    user write any Pallas function (and register lowering rules for what its
    emitter lacks, docs/extending.md:1-69).

    `rhs` is CUDA C: the statements of
    `void rhs(float t, const float* y, const float* p, float* dy)`, e.g.
    `"dy[0] = y[1]; dy[1] = (p[0] * (1.0f - y[0] * y[0])) * y[1] - y[0];"`.
    It is compiled at run time (NVRTC) under the flag set of the call's math
    mode and cached by source text, the way the reference compiles the MSL it
    emits on a cache miss (src/palladium/__init__.py:146-158).

    method="rk4": `steps` classic RK4 steps of `dt`; grid=(N,), inputs are the
    `dim` state arrays then the `nparam` parameter arrays, outputs the `dim`
    final states (all (N,) float32).  With the Lotka-Volterra right-hand side
    this reproduces `lv_rk4` bit for bit under MathMode.SAFE.
    method="bs32": adaptive Bogacki-Shampine 3(2) with the controller, counters
    and stall semantics of `vdp_bs32`; outputs t, the `dim` states, steps,
    rejected, real.
    method="dopri5" / "tsit5": the seven-stage 5(4) pairs of Dormand-Prince and of
    Tsitouras (what the reference's CPU comparison integrates with,
    benchmarks/bench_ensembles.py:88-118) under the same controller and with the
    same outputs.  `error_order` defaults to 3 for bs32 and 5 for these.

    With `check` (default) the source is compiled once here, without a GPU, so a
    faulty right-hand side raises EmitError where it is defined."""
    if method not in _ODE_METHODS:
        raise TraceError(f"custom_ode: method must be one of {sorted(_ODE_METHODS)}, got {method!r}")
    if error_order is None:
        error_order = 5 if method in ("dopri5", "tsit5") else 3
    if not isinstance(rhs, str) or not rhs.strip():
        raise TraceError("custom_ode: rhs must be a non-empty string of CUDA C statements")
    if not 1 <= int(dim) <= 8:
        raise TraceError(f"custom_ode: dim must lie in [1, 8], got {dim}")
    if not 0 <= int(nparam) <= 8:
        raise TraceError(f"custom_ode: nparam must lie in [0, 8], got {nparam}")
    fam = Family("custom_ode", dict(rhs=rhs, dim=int(dim), nparam=int(nparam), method=method, dt=float(dt),
                                    steps=int(steps), t1=float(t1), rtol=float(rtol), atol=float(atol),
                                    dt0=float(dt0), max_steps=int(max_steps), pcoeff=float(pcoeff),
                                    icoeff=float(icoeff), safety=float(safety), factor_min=float(factor_min),
                                    factor_max=float(factor_max), error_order=int(error_order)), pallas_fn)
    key = (rhs, int(dim), int(nparam), method)
    if check and key not in _CHECKED_SOURCES:
        _native.custom_ode_check(_custom_ode_params(fam.constants))
        _CHECKED_SOURCES.add(key)
    return fam


def _custom_ode_params(c: dict) -> "_native.CustomOdeParams":
    return _native.CustomOdeParams(c["rhs"].encode(), c["dim"], c["nparam"], _ODE_METHODS[c["method"]],
                                   c["dt"], c["steps"], c["t1"], c["rtol"], c["atol"], c["dt0"], c["pcoeff"],
                                   c["icoeff"], c["safety"], c["factor_min"], c["factor_max"], c["error_order"],
                                   c["max_steps"])


def source_kernel(source: str, function_name: str, check: bool = True) -> Family:
    """A complete kernel of your own as CUDA C source: what `metal_call` hands
    its runtime as emitted MSL plus an entry-point name
    (src/palladium/dispatch.py:286-292), written by hand here because there is
    no Pallas-to-CUDA emitter.

    The kernel is declared
    `extern "C" __global__ void name(T0* b0, ..., Tk* bk, long long gx, long long gy, long long gz)`:
    one pointer per array in call order (inputs, then the outputs of
    `out_shape`), then the extents of `grid`.  One thread runs per grid point,
    rounded up to whole blocks: return when `PD_THREAD_X >= gx` (and likewise
    `PD_THREAD_Y`, `PD_THREAD_Z`).  `pd_math.h` (Threefry, df32, `pd_powf`) is
    in scope.  Compiled at run time under the call's math mode, cached by
    source; array shapes and dtypes are whatever the call passes, unchecked
    against the kernel, as with hand-written MSL."""
    if not isinstance(source, str) or not source.strip():
        raise TraceError("source_kernel: source must be a non-empty string of CUDA C")
    if not isinstance(function_name, str) or not function_name.isidentifier() or len(function_name) > 63:
        raise TraceError(f"source_kernel: function_name must be a C identifier of at most 63 characters, "
                         f"got {function_name!r}")
    fam = Family("source", dict(source=source, function_name=function_name))
    key = ("source", source, function_name)
    if check and key not in _CHECKED_SOURCES:
        _native.source_kernel_check(_native.SourceKernelParams(source.encode(), function_name.encode()))
        _CHECKED_SOURCES.add(key)
    return fam


def vdp_cost_order(x0, v0, mu, *, pilot_rtol: float = 1e-3, pilot_atol: float = 1e-5, **constants):
    """A hand-out order for `vdp_bs32` from a pilot run at a looser tolerance.

    The adaptive kernel's run time ends with the trajectories that happen to be
    both long and late in the queue: each attempt of a lone trajectory costs its
    full dependent latency, so a 7500-attempt member started last adds
    milliseconds.  Handing out the trajectories by decreasing cost removes that
    tail -- with the true costs, 15.8 -> 13.7 ms at 2^20 trajectories (RELAXED) --
    and `vdp_bs32` takes such an order as an optional fourth operand (int32, a
    permutation of 0..N-1; results do not depend on it).  Use it when the costs
    are known, e.g. from an earlier solve of the same ensemble.

    This helper estimates them with a pilot run.  Measured, that does not pay:
    the pilot's step pattern predicts the tight-tolerance count only loosely
    (run 15.0 ms instead of 15.8, plus 0.8 ms for the pilot), so it is here for
    completeness rather than speed.  Takes and returns torch CUDA tensors."""
    import torch

    from .ffi import cuda_call_jit
    from .pl import ShapeDtypeStruct

    n = int(x0.shape[0])
    cfg = dict(constants)
    cfg.update(rtol=pilot_rtol, atol=pilot_atol)
    pilot = cuda_call_jit(vdp_bs32(**cfg), grid=(n,),
                          out_shape=(ShapeDtypeStruct((n, 2), np.float32), ShapeDtypeStruct((n,), np.int32),
                                     ShapeDtypeStruct((n,), np.int32)), math_mode="fast")
    _, accepted, rejected = pilot(x0, v0, mu)
    return torch.argsort(accepted + rejected, descending=True).to(torch.int32)


def gbm_threefry(s0: float = 100.0, strike: float = 105.0, r: float = 0.03, sigma: float = 0.2, t: float = 1.0,
                 steps: int = 256, output: str = "payoff", path_offset: int = 0,
                 pallas_fn: Callable | None = None) -> Family:
    """GBM European call paths with in-kernel Threefry (examples/03_sde_montecarlo.py:97-119;
    defaults from :30-32).  grid=(N,), one (2,) uint32 input (key data), one (N,)
    float32 output: the payoff max(S_T - K, 0) (`output="payoff"`, the reference)
    or the terminal price S_T (`output="terminal"`).  An optional second output
    of shape (2,) float64 receives (sum payoff, sum payoff^2)."""
    if output not in ("payoff", "terminal"):
        raise TraceError(f"gbm_threefry: output must be 'payoff' or 'terminal', got {output!r}")
    return Family("gbm_threefry", dict(s0=float(s0), strike=float(strike), r=float(r), sigma=float(sigma),
                                       t=float(t), steps=int(steps), output=output,
                                       path_offset=int(path_offset)), pallas_fn)


def gbm_pcg(s0: float = 100.0, strike: float = 105.0, r: float = 0.03, sigma: float = 0.2, t: float = 1.0,
            steps: int = 256, output: str = "payoff", path_offset: int = 0) -> Family:
    """The reference's hand-written GBM kernel (`GBM_MSL`, examples/03_sde_montecarlo.py:34-70):
    same model as `gbm_threefry` with the cheap `pcg_hash` counter RNG, one hash
    per uniform.  grid=(N,), no inputs, one (N,) float32 output (payoff or
    terminal price) and an optional (2,) float64 output of payoff sums."""
    if output not in ("payoff", "terminal"):
        raise TraceError(f"gbm_pcg: output must be 'payoff' or 'terminal', got {output!r}")
    return Family("gbm_pcg", dict(s0=float(s0), strike=float(strike), r=float(r), sigma=float(sigma), t=float(t),
                                  steps=int(steps), output=output, path_offset=int(path_offset)))


def gray_scott(du: float = 0.16, dv: float = 0.08, f: float = 0.035, k: float = 0.065, dt: float = 1.0,
               steps: int = 1, halo: int = 0, pallas_fn: Callable | None = None) -> Family:
    """Gray-Scott 5-point stencil (examples/04_reaction_diffusion.py:61-74; constants :35).
    grid=(rows, cols), inputs u, v and outputs u', v' of shape (rows, cols)
    float32.  `steps` > 1 runs that many steps inside one call with the fields
    resident on the device (the reference's ping-pong loop, :99-107).
    `halo` > 0 treats the arrays as a row slab of shape (rows + 2*halo, cols)
    with ghost rows that the caller fills; at most `halo` steps per call."""
    return Family("gray_scott", dict(du=float(du), dv=float(dv), f=float(f), k=float(k), dt=float(dt),
                                     steps=int(steps), halo=int(halo)), pallas_fn)


def lv_rk4_df32(dt: float = 0.01, steps: int = 500) -> Family:
    """RK4 Lotka-Volterra in df32 compensated arithmetic
    (examples/05_df32_precision.py:27-80).  Same signature as `lv_rk4`."""
    return Family("lv_rk4_df32", dict(dt=float(dt), steps=int(steps)))


def kepler_rk4_df32(dt: float = 1e-3, gm: float = 1.0, steps: int = 1000) -> Family:
    """RK4 two-body orbits in df32.  grid=(N,), eight (N,) float32 inputs
    (x, y, vx, vy as hi/lo pairs) and eight outputs of the same layout."""
    return Family("kepler_rk4_df32", dict(dt=float(dt), gm=float(gm), steps=int(steps)))


def threefry_bits(op: str = "bits", count: int = 1) -> Family:
    """The RNG primitives on their own (src/palladium/emit/rules.py:168-201):
    op "bits": (N,) uint32 = random_bits(key, (N,)); "uniform": (N,) float32;
    "fold_in": inputs key and (M,) uint32 data, output (M, 2) uint32 key data;
    "fold_uniform": (G, count) float32, row g = uniform(fold_in(key, g), (count,));
    "pcg": (N,) uint32 = pcg_hash(i), the hash of examples/03_sde_montecarlo.py:38-43
    (the key input is ignored)."""
    ops = {"bits": 0, "uniform": 1, "fold_in": 2, "fold_uniform": 3, "pcg": 4}
    if op not in ops:
        raise TraceError(f"threefry_bits: op must be one of {sorted(ops)}, got {op!r}")
    return Family("threefry_bits", dict(op=op, op_code=ops[op], count=int(count)))


# ----------------------------------------------------------------------------- state-space families
SCAN_CHUNK = 32       # tokens between two states that `selective_scan(carries=True)` keeps

_TYPE_CODES = {"float32": 0, "float16": 1, "bfloat16": 2}


def _element_type(what: str, dtype) -> str:
    try:
        name = dtype_name(as_dtype(dtype))
    except TypeError:
        name = str(dtype)
    if name not in _TYPE_CODES:
        raise TraceError(f"{what}: dtype must be one of {', '.join(_TYPE_CODES)}, got {name}")
    return name


def _whole(what: str, name: str, value, low: int, high: int) -> int:
    try:
        whole = int(value) if not isinstance(value, bool) and int(value) == value else None
    except (TypeError, ValueError, OverflowError):      # None, text, NaN, infinities
        whole = None
    if whole is None or not low <= whole <= high:
        raise TraceError(f"{what}: {name} must be a whole number in [{low}, {high}], got {value!r}")
    return whole


def _conv_family(name: str, length, width, silu, bias, initial, final, packed, dtype) -> Family:
    return Family(name, dict(length=_whole(name, "length", length, 0, 2**31 - 1), width=_whole(name, "width", width, 2, 4),
                             silu=bool(silu), bias=bool(bias), initial=bool(initial), final=bool(final),
                             packed=bool(packed), dtype=_element_type(name, dtype)))


def causal_conv(length: int, width: int = 4, *, silu: bool = True, bias: bool = True, initial: bool = False,
                final: bool = False, packed: bool = False, dtype="float32") -> Family:
    """A short causal convolution over the tokens of S sequences, channel by channel:
    `y_t = act(bias + sum_j weight[:, width - 1 - j] * x_{t-j})`, j = 0 .. width - 1,
    with act(v) = v / (1 + e^-v) or, with `silu=False`, v itself.  Not in the reference.

    grid=(S, D).  Inputs: x (S, length, D), weight (D, width) float32, bias (D,)
    float32 with `bias`, initial (S, width - 1, D) with `initial` (the inputs before
    each sequence's first token, else zeros), offsets with `packed`.  Outputs:
    y like x, and with `final` the last width - 1 inputs of each sequence, what the
    next call's `initial` or `causal_conv_step`'s state is.  `width` is 2, 3 or 4.

    `packed=True`: sequences of different lengths behind one another.  Token arrays
    are (length, D) with `length` rows in all; the last operand, offsets (S + 1,)
    int32, gives sequence s the rows offsets[s] .. offsets[s + 1] - 1.  It is read on
    the device: values are clamped to [0, length], a decreasing pair is an empty
    sequence, rows before the first and behind the last sequence come out as zeros.
    Beside a decreasing pair other sequences' results are undefined.

    `dtype`: float32, float16 or bfloat16 (`pl.bfloat16`, torch.bfloat16), the type
    of x, y, initial and final.  Sums are float32, rounded once."""
    return _conv_family("causal_conv", length, width, silu, bias, initial, final, packed, dtype)


def causal_conv_step(width: int = 4, *, silu: bool = True, bias: bool = True, dtype="float32") -> Family:
    """`causal_conv` for one token of each of S sequences.  grid=(S, D); inputs x (S, D),
    state (S, width - 1, D), weight, bias; outputs y (S, D) and the state one token on.
    On device tensors `call.on_device(..., out=(y, state))` updates a state in place."""
    return _conv_family("causal_conv_step", 1, width, silu, bias, True, True, False, dtype)


def causal_conv_grad(length: int, width: int = 4, *, silu: bool = True, bias: bool = True, initial: bool = False,
                     final: bool = False, packed: bool = False, dtype="float32") -> Family:
    """Gradients of `causal_conv` with the same constants.  Inputs: dy like y, then x,
    weight, bias, initial as there, dfinal (the gradient of final) with `final`, offsets
    with `packed`.  Outputs: dx, dweight float32, dbias float32 with `bias`, dinitial with
    `initial`.  Sums run in a fixed order: equal calls on one device give equal bits.
    (Results of `causal_conv` carry no autograd history: a `torch.autograd.Function` of the
    caller's connects the two calls.)"""
    return _conv_family("causal_conv_grad", length, width, silu, bias, initial, final, packed, dtype)


def _scan_family(name: str, length, state, groups, softplus, bias, skip, gate, initial, final, carries, packed,
                 dtype) -> Family:
    return Family(name, dict(length=_whole(name, "length", length, 0, 2**31 - 1), state=_whole(name, "state", state, 1, 64),
                             groups=_whole(name, "groups", groups, 1, 65535), softplus=bool(softplus), bias=bool(bias),
                             skip=bool(skip), gate=bool(gate), initial=bool(initial), final=bool(final),
                             carries=bool(carries), packed=bool(packed), dtype=_element_type(name, dtype)))


def selective_scan(length: int, state: int = 16, *, groups: int = 1, softplus: bool = True, bias: bool = True,
                   skip: bool = True, gate: bool = False, initial: bool = False, final: bool = False,
                   carries: bool = False, packed: bool = False, dtype="float32") -> Family:
    """An ensemble of driven linear systems h' = A h + B(t) x(t), y = C(t) h + skip x with
    `state` states each, one trajectory per (sequence, channel), integrated over steps of
    input-dependent length d with B and x held constant in each (the selective state-space
    scan).  Not in the reference, whose ensembles have parameters fixed in time.

        d = softplus(delta + bias)         (softplus=False: delta + bias)
        h_t = exp(d A) h_{t-1} + d x_t B_t
        y_t = (C_t . h_t + skip x_t) * z_t / (1 + e^-z_t)      (the last factor with `gate`)

    grid=(S, D).  Inputs: x (S, length, D), delta like x, A (D, state) float32,
    B (S, length, groups, state), C like B, bias (D,) float32 with `bias`, skip (D,) float32
    with `skip`, z like x with `gate`, initial (S, D, state) float32 with `initial` (else
    zeros), offsets with `packed` (see `causal_conv`; B and C are then (length, groups, state)).
    Channel c reads group c // (D // groups).  Outputs: y like x; final (S, D, state) float32
    with `final`; with `carries` the states a later `selective_scan_grad` recomputes from, one
    per SCAN_CHUNK tokens: (S, ceil(length / SCAN_CHUNK), D, state) float32, packed
    (length // SCAN_CHUNK + S, D, state) with entries that no token owns left unwritten.

    `state` is 1 .. 64.  `dtype` (float32, float16, bfloat16) is the type of x, delta, B, C, z
    and y; states are float32 throughout and y is rounded once.  Rates may have either sign; the
    factor exp(d A) of a single token has to be in float32's range.  In FAST the prompts of 2-byte
    tokens take an approximate power of two: states that remember hundreds of tokens are then up
    to about 3e-6 off in norm, a tenth of that for float32 tokens and in the other modes."""
    return _scan_family("selective_scan", length, state, groups, softplus, bias, skip, gate, initial, final, carries,
                        packed, dtype)


def selective_scan_step(state: int = 16, *, groups: int = 1, softplus: bool = True, bias: bool = True,
                        skip: bool = True, gate: bool = False, dtype="float32") -> Family:
    """`selective_scan` for one token of each of S sequences.  grid=(S, D); inputs
    state (S, D, state) float32, x (S, D), delta, A, B (S, groups, state), C, bias, skip, z;
    outputs y (S, D) and the state one token on.  On device tensors
    `call.on_device(..., out=(y, state))` updates a state in place."""
    return _scan_family("selective_scan_step", 1, state, groups, softplus, bias, skip, gate, True, True, False, False,
                        dtype)


def selective_scan_grad(length: int, state: int = 16, *, groups: int = 1, softplus: bool = True, bias: bool = True,
                        skip: bool = True, gate: bool = False, initial: bool = False, final: bool = False,
                        packed: bool = False, dtype="float32") -> Family:
    """Gradients of `selective_scan` with the same constants.  Inputs: dy like y, then x,
    delta, A, B, C, bias, skip, z as there, the carries of a forward call with
    `carries=True`, dfinal (the gradient of final) with `final`, offsets with `packed`.
    Outputs: dx, ddelta, dA float32, dB, dC, then dbias and dskip float32, dz and
    dinitial float32 where the constants have them.  B and C are shared by the channels of
    a group and the parameters by all tokens: their sums are float32 in a fixed order, so
    equal calls on one device give equal bits.  Scratch: about 8 bytes per token, state and
    block of up to 24 channels (`call.explain(...).scratch_bytes` says how much).
    (Results of `selective_scan` carry no autograd history: a `torch.autograd.Function` of the
    caller's connects the two calls.)"""
    return _scan_family("selective_scan_grad", length, state, groups, softplus, bias, skip, gate, initial, final, False,
                        packed, dtype)


STATE_SPACE = ("causal_conv", "causal_conv_step", "causal_conv_grad", "selective_scan", "selective_scan_step",
                  "selective_scan_grad")


def _scan_operands(family: Family, grid) -> tuple[list, list]:
    """(inputs, outputs) of a state-space call as (name, BlockInfo, index map): one program per
    (sequence, channel), whose blocks are that channel's column of the sequence's tokens."""
    c, name = family.constants, family.name
    if len(grid) != 2:
        raise TraceError(f"{name}: grid must be (sequences, channels), got {grid}")
    s, d = grid
    if s < 0 or d < 1:
        raise TraceError(f"{name}: grid must hold at least one channel, got {grid}")
    kind = bfloat16 if c["dtype"] == "bfloat16" else np.dtype(c["dtype"])
    step, n, packed = name.endswith("step"), c["length"], c["packed"]

    def tokens(label, dtype=kind):
        if step:
            return label, BlockInfo((1, 1), (s, d), dtype), lambda i, j: (i, j)
        if packed:
            return label, BlockInfo((n, 1), (n, d), dtype), lambda i, j: (0, j)
        return label, BlockInfo((1, n, 1), (s, n, d), dtype), lambda i, j: (i, 0, j)

    def parameter(label, *shape):
        return label, BlockInfo((1,) + shape, (d,) + shape, F32), lambda i, j: (j,) + (0,) * len(shape)

    offsets = [("offsets", BlockInfo((s + 1,), (s + 1,), I32), lambda i, j: (0,))] if packed else []
    if name.startswith("causal_conv"):
        w = c["width"]

        def edge(label):
            return label, BlockInfo((1, w - 1, 1), (s, w - 1, d), kind), lambda i, j: (i, 0, j)

        weights = [parameter("weight", w)] + [parameter("bias")] * c["bias"]
        if step:
            return [tokens("x"), edge("state")] + weights, [tokens("y"), edge("state")]
        before = [edge("initial")] * c["initial"]
        if name == "causal_conv":
            return [tokens("x")] + weights + before + offsets, [tokens("y")] + [edge("final")] * c["final"]
        return ([tokens("dy"), tokens("x")] + weights + before + [edge("dfinal")] * c["final"] + offsets,
                [tokens("dx"), parameter("dweight", w)] + [parameter("dbias")] * c["bias"] + [edge("dinitial")] * c["initial"])
    k, g = c["state"], c["groups"]
    if d % g:
        raise TraceError(f"{name}: {d} channels do not divide into {g} groups")
    per = d // g

    def coupling(label):
        if step:
            return label, BlockInfo((1, 1, k), (s, g, k), kind), lambda i, j: (i, j // per, 0)
        if packed:
            return label, BlockInfo((n, 1, k), (n, g, k), kind), lambda i, j: (0, j // per, 0)
        return label, BlockInfo((1, n, 1, k), (s, n, g, k), kind), lambda i, j: (i, 0, j // per, 0)

    def edge(label):
        return label, BlockInfo((1, 1, k), (s, d, k), F32), lambda i, j: (i, j, 0)

    def kept(label):
        if packed:
            chunks = n // SCAN_CHUNK + s
            return label, BlockInfo((chunks, 1, k), (chunks, d, k), F32), lambda i, j: (0, j, 0)
        chunks = -(-n // SCAN_CHUNK)
        return label, BlockInfo((1, chunks, 1, k), (s, chunks, d, k), F32), lambda i, j: (i, 0, j, 0)

    operands = ([tokens("x"), tokens("delta"), parameter("A", k), coupling("B"), coupling("C")]
                + [parameter("bias")] * c["bias"] + [parameter("skip")] * c["skip"] + [tokens("z")] * c["gate"])
    if step:
        return [edge("state")] + operands, [tokens("y"), edge("state")]
    if name == "selective_scan":
        return (operands + [edge("initial")] * c["initial"] + offsets,
                [tokens("y")] + [edge("final")] * c["final"] + [kept("carries")] * c["carries"])
    return ([tokens("dy")] + operands + [kept("carries")] + [edge("dfinal")] * c["final"] + offsets,
            [tokens("dx"), tokens("ddelta"), parameter("dA", k), coupling("dB"), coupling("dC")]
            + [parameter("dbias")] * c["bias"] + [parameter("dskip")] * c["skip"] + [tokens("dz")] * c["gate"]
            + [edge("dinitial")] * c["initial"])


def _scan_params(family: Family):
    c = dict(family.constants, type=_TYPE_CODES[family.constants["dtype"]])
    kind = _native.CausalConvParams if family.name.startswith("causal_conv") else _native.SelectiveScanParams
    return kind(*[int(c[field]) for field, _ in kind._fields_])


def out_shapes(family: Family, grid):
    """The `out_shape` of a state-space call, for families whose outputs follow from their
    constants: a ShapeDtypeStruct, or a tuple of them in output order."""
    if not isinstance(family, Family) or family.name not in STATE_SPACE:
        raise TraceError(f"out_shapes knows the state-space families ({', '.join(STATE_SPACE)}), not {family!r}")
    grid = tuple(int(g) for g in grid)
    shapes = tuple(ShapeDtypeStruct(info.array_shape, info.dtype) for _, info, _ in _scan_operands(family, grid)[1])
    return shapes[0] if len(shapes) == 1 else shapes


# ----------------------------------------------------------------------------- tracing
def _shape_dtype(x) -> tuple[tuple[int, ...], np.dtype]:
    shape = getattr(x, "shape", None)
    dtype = getattr(x, "dtype", None)
    if shape is None or dtype is None:
        arr = np.asarray(x)
        shape, dtype = arr.shape, arr.dtype
    dtype = as_dtype(dtype)
    return tuple(int(s) for s in shape), dtype


def _as_list(x) -> list:
    if x is None:
        return []
    if isinstance(x, (list, tuple)):
        return list(x)
    return [x]


def _check_specs(what: str, specs, expected_blocks: Sequence[tuple[tuple[int, ...], Callable]], grid) -> None:
    """Validate in_specs / out_specs against the block shapes and index maps the
    family implements.  A spec of None (or a missing list) is accepted: Pallas
    then defaults to whole-array blocks, which the fixed kernels do not depend on."""
    specs = _as_list(specs)
    if not specs:
        return
    if len(specs) != len(expected_blocks):
        raise TraceError(f"{what} has {len(specs)} entries, the kernel family takes {len(expected_blocks)}")
    probes = [tuple(0 for _ in grid), tuple(max(g - 1, 0) for g in grid)]
    for i, (spec, (block, index_map)) in enumerate(zip(specs, expected_blocks)):
        if spec is None:
            continue
        got_block = getattr(spec, "block_shape", None)
        if got_block is not None and tuple(int(b) for b in got_block) != tuple(block):
            raise TraceError(f"{what}[{i}]: block shape {tuple(got_block)} is not the {tuple(block)} this family uses")
        got_map = getattr(spec, "index_map", None)
        if got_map is not None:
            for probe in probes:
                try:
                    got = tuple(int(v) for v in got_map(*probe))
                except Exception as exc:  # a map of the wrong arity, most likely
                    raise TraceError(f"{what}[{i}]: index_map could not be evaluated at {probe}: {exc}") from None
                want = tuple(int(v) for v in index_map(*probe))
                if got != want:
                    raise TraceError(f"{what}[{i}]: index_map{probe} = {got}, this family needs {want}")


def _check_args(args, inputs: Sequence[BlockInfo]) -> None:
    if not args:
        return
    if len(args) != len(inputs):
        raise TraceError(f"kernel takes {len(inputs)} arrays, got {len(args)}")
    for i, (a, info) in enumerate(zip(args, inputs)):
        shape, dtype = _shape_dtype(a)
        if shape != info.array_shape:
            raise TraceError(f"argument {i}: shape {shape} does not match the {info.array_shape} implied by grid")
        if dtype != info.dtype:
            raise DispatchError(
                f"argument {i}: dtype {dtype_name(dtype)} does not match the traced {dtype_name(info.dtype)}; cast explicitly"
            )


def _out_structs(out_shape) -> list[tuple[tuple[int, ...], np.dtype]]:
    if out_shape is None:
        raise TraceError("out_shape is required")
    return [_shape_dtype(o) for o in _as_list(out_shape)]


def _per_item(n: int):
    return ((1,), lambda i: (i,))


def trace(family: Family, call_kwargs: dict[str, Any], *args) -> KernelSpec:
    """Validate a `pallas_call`-shaped call against a family; returns the spec.

    Raises TraceError when grid / specs / out_shape / argument shapes do not
    describe a launch of that family (the reference raises TraceError when a
    pallas_call cannot be traced, src/palladium/trace.py:83-99,139-166)."""
    if not isinstance(family, Family):
        raise UnsupportedPrimitiveError(
            "cuda_call needs a kernel family from palladium_b200.families (there is no "
            f"Pallas-to-CUDA emitter); got {type(family).__name__}"
        )
    unknown = set(call_kwargs) - {"grid", "in_specs", "out_specs", "out_shape", "name", "interpret", "debug",
                                  "input_output_aliases", "compiler_params", "cost_estimate", "grid_spec"}
    if unknown:
        raise TraceError(f"unsupported pallas_call keywords: {sorted(unknown)}")
    if call_kwargs.get("grid_spec") is not None:
        raise TraceError("grid_spec (scalar prefetch) is not supported; pass grid / in_specs / out_specs")
    if call_kwargs.get("input_output_aliases"):
        raise TraceError("input_output_aliases is not supported")
    grid = call_kwargs.get("grid")
    grid = (int(grid),) if isinstance(grid, (int, np.integer)) else tuple(int(g) for g in (grid or ()))
    outs = _out_structs(call_kwargs.get("out_shape"))
    c = family.constants
    name = family.name

    def vec(n, dtype=F32):
        return BlockInfo((1,), (n,), dtype)

    if name in ("lv_rk4", "lv_rk4_df32"):
        if len(grid) != 1:
            raise TraceError(f"{name}: grid must be (N,), got {grid}")
        n = grid[0]
        inputs = tuple(vec(n) for _ in range(6))
        outputs = tuple(vec(n) for _ in range(2))
        blocks_in = [_per_item(n)] * 6
        blocks_out = [_per_item(n)] * 2
        if name == "lv_rk4" and len(outs) == 1:
            # the final state as one (N, 2) array of (x, y) pairs
            outputs = (BlockInfo((1, 2), (n, 2), F32),)
            blocks_out = [((1, 2), lambda i: (i, 0))]
        if name == "lv_rk4":
            params = _native.LvRk4Params(c["dt"], c["steps"])
        else:
            params = _native.LvRk4Df32Params(c["dt"], c["steps"])
    elif name == "vdp_bs32":
        if len(grid) != 1:
            raise TraceError(f"{name}: grid must be (N,), got {grid}")
        n = grid[0]
        inputs = tuple(vec(n) for _ in range(3))
        blocks_in = [_per_item(n)] * 3
        if len(args) == 4 or len(_as_list(call_kwargs.get("in_specs"))) == 4:
            # optional fourth operand: the order in which the work queue hands out the
            # trajectories, a permutation of 0..N-1 (see `vdp_cost_order`)
            inputs = inputs + (vec(n, I32),)
            blocks_in = blocks_in + [_per_item(n)]
        if len(outs) == 6:
            layout, outputs, blocks_out = 0, tuple(vec(n) for _ in range(6)), [_per_item(n)] * 6
        elif len(outs) == 5:
            layout, outputs, blocks_out = 1, tuple(vec(n) for _ in range(5)), [_per_item(n)] * 5
        elif len(outs) == 3:
            layout = 2
            outputs = (BlockInfo((1, 2), (n, 2), F32), vec(n, I32), vec(n, I32))
            blocks_out = [((1, 2), lambda i: (i, 0)), _per_item(n), _per_item(n)]
        else:
            raise TraceError(f"{name}: out_shape must list 6, 5 or 3 outputs, got {len(outs)}")
        params = _native.VdpBs32Params(c["t1"], c["rtol"], c["atol"], c["dt0"], c["pcoeff"], c["icoeff"],
                                       c["safety"], c["factor_min"], c["factor_max"], c["error_order"],
                                       c["max_steps"], layout)
    elif name in ("gbm_threefry", "gbm_pcg"):
        if len(grid) != 1:
            raise TraceError(f"{name}: grid must be (N,), got {grid}")
        n = grid[0]
        if name == "gbm_threefry":
            inputs = (BlockInfo((2,), (2,), U32),)
            blocks_in = [((2,), lambda i: (0,))]
        else:
            inputs, blocks_in = (), []
        outputs = (vec(n),)
        blocks_out = [_per_item(n)]
        if len(outs) == 2:
            outputs = outputs + (BlockInfo((2,), (2,), F64),)
            blocks_out = blocks_out + [((2,), lambda i: (0,))]
        elif len(outs) != 1:
            raise TraceError(f"{name}: out_shape must list 1 or 2 outputs, got {len(outs)}")
        params = _native.GbmParams(c["s0"], c["strike"], c["r"], c["sigma"], c["t"], c["steps"], c["path_offset"],
                                   0 if c["output"] == "payoff" else 1)
    elif name == "gray_scott":
        if len(grid) != 2:
            raise TraceError(f"{name}: grid must be (rows, cols), got {grid}")
        rows, cols = grid
        shape = (rows + 2 * c["halo"], cols)
        inputs = tuple(BlockInfo(shape, shape, F32) for _ in range(2))
        outputs = tuple(BlockInfo(shape, shape, F32) for _ in range(2))
        blocks_in = [(shape, lambda i, j: (0, 0))] * 2
        blocks_out = [(shape, lambda i, j: (0, 0))] * 2
        params = _native.GrayScottParams(c["du"], c["dv"], c["f"], c["k"], c["dt"], c["steps"], rows, cols, c["halo"])
    elif name == "kepler_rk4_df32":
        if len(grid) != 1:
            raise TraceError(f"{name}: grid must be (N,), got {grid}")
        n = grid[0]
        inputs = tuple(vec(n) for _ in range(8))
        outputs = tuple(vec(n) for _ in range(8))
        blocks_in = [_per_item(n)] * 8
        blocks_out = [_per_item(n)] * 8
        params = _native.KeplerRk4Df32Params(c["dt"], c["gm"], c["steps"])
    elif name == "custom_ode":
        if len(grid) != 1:
            raise TraceError(f"{name}: grid must be (N,), got {grid}")
        n = grid[0]
        n_in = c["dim"] + c["nparam"]
        n_out = c["dim"] if c["method"] == "rk4" else c["dim"] + 4
        inputs = tuple(vec(n) for _ in range(n_in))
        outputs = tuple(vec(n) for _ in range(n_out))
        blocks_in = [_per_item(n)] * n_in
        blocks_out = [_per_item(n)] * n_out
        params = _custom_ode_params(c)
    elif name == "source":
        if not 1 <= len(grid) <= 3:
            raise TraceError(f"{name}: grid must have 1 to 3 dimensions, got {grid}")
        # the kernel defines its own operands: take them as the call gives them
        inputs = tuple(BlockInfo(shape, shape, dtype) for shape, dtype in (_shape_dtype(a) for a in args))
        outputs = tuple(BlockInfo(shape, shape, dtype) for shape, dtype in outs)
        blocks_in = blocks_out = None
        params = _native.SourceKernelParams(c["source"].encode(), c["function_name"].encode())
    elif name == "threefry_bits":
        if len(grid) != 1:
            raise TraceError(f"{name}: grid must be (N,), got {grid}")
        n = grid[0]
        key = BlockInfo((2,), (2,), U32)
        op = c["op"]
        if op in ("bits", "pcg"):
            inputs, outputs = (key,), (vec(n, U32),)
        elif op == "uniform":
            inputs, outputs = (key,), (vec(n),)
        elif op == "fold_in":
            inputs, outputs = (key, vec(n, U32)), (BlockInfo((1, 2), (n, 2), U32),)
        else:
            inputs, outputs = (key,), (BlockInfo((1, c["count"]), (n, c["count"]), F32),)
        blocks_in = blocks_out = None
        params = _native.ThreefryParams(c["op_code"], c["count"])
    elif name in STATE_SPACE:
        taken, given = _scan_operands(family, grid)
        inputs, outputs = tuple(info for _, info, _ in taken), tuple(info for _, info, _ in given)
        blocks_in = [(info.block_shape, index) for _, info, index in taken]
        blocks_out = [(info.block_shape, index) for _, info, index in given]
        params = _scan_params(family)
    else:
        raise UnsupportedPrimitiveError(f"no CUDA kernel family named {name!r}")

    if len(outs) != len(outputs):
        raise TraceError(f"{name}: out_shape lists {len(outs)} outputs, the kernel family produces {len(outputs)}")
    for i, ((shape, dtype), info) in enumerate(zip(outs, outputs)):
        if shape != info.array_shape or dtype != info.dtype:
            raise TraceError(
                f"{name}: out_shape[{i}] is {shape} {dtype}, the kernel family produces "
                f"{info.array_shape} {info.dtype} for grid {grid}"
            )
    if blocks_in is not None:
        _check_specs("in_specs", call_kwargs.get("in_specs"), blocks_in, grid)
        _check_specs("out_specs", call_kwargs.get("out_specs"), blocks_out, grid)
    _check_args(args, inputs)
    return KernelSpec(name=f"palladium_{name}", family=family, grid=grid, inputs=inputs, outputs=outputs, params=params)
