"""Inputs, calls and comparisons shared by the tests of the state-space families."""

import numpy as np

from oracle import state_space as S
from palladium_b200 import families, pl

TYPES = ("float32", "float16", "bfloat16")
# half a step of each element type, relative to the value, and half the smallest step near zero
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
SMALLEST = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def rounded(values, dtype):
    """float64 values after a rounding to `dtype`, ties to even."""
    if dtype == "bfloat16":
        bits = np.asarray(values, np.float32).view(np.uint32)
        return ((bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32).astype(np.float64)
    return np.asarray(values).astype(dtype).astype(np.float64)


def host(values, dtype):
    """An array a call takes, from values that `dtype` holds exactly."""
    if dtype == "bfloat16":
        return (np.asarray(values, np.float32).view(np.uint32) >> 16).astype(np.uint16).view(pl.bfloat16)
    return np.ascontiguousarray(np.asarray(values).astype(dtype))


def wide(array):
    """float64 values of an array that a call returned."""
    if array.dtype == pl.bfloat16:
        return (array.view(np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return array.astype(np.float64)


def starts_of(lengths, lead=0):
    return [lead] + [lead + int(v) for v in np.cumsum(lengths)]


class Case:
    """One problem: the operands in float64 (already rounded to their types), the sequences' rows, the
    constants of the family, and the operator's values and tolerances."""

    def __init__(self, kind, lengths, channels, *, dtype="float32", packed=False, spare=0, lead=0, seed=0, width=4,
                 state=16, groups=1, silu=True, softplus=True, bias=True, skip=True, gate=False, initial=False,
                 final=False):
        rng = np.random.default_rng(seed)
        self.kind, self.dtype, self.packed = kind, dtype, packed
        self.seqs, self.channels = len(lengths), channels
        if not packed:
            assert len(set(lengths)) <= 1
        self.starts = starts_of(lengths, lead)
        self.rows = self.starts[-1] + spare
        self.length = self.rows if packed else (lengths[0] if lengths else 0)
        tok = lambda *tail: rounded(rng.standard_normal((self.rows,) + tail), dtype)  # noqa: E731
        par = lambda v: np.asarray(v, np.float32).astype(np.float64)  # noqa: E731
        self.constants = dict(length=self.length, bias=bias, initial=initial, final=final, packed=packed, dtype=dtype)
        v = self.v = {"x": tok(channels), "dy": tok(channels)}
        if kind == "conv":
            self.constants.update(width=width, silu=silu)
            v["weight"] = par(rng.standard_normal((channels, width)) * 0.5)
            if bias:
                v["bias"] = par(rng.standard_normal(channels) * 0.1)
            edge = (self.seqs, width - 1, channels)
            if initial:
                v["initial"] = rounded(rng.standard_normal(edge), dtype)
            if final:
                v["dfinal"] = rounded(rng.standard_normal(edge), dtype)
        else:
            self.constants.update(state=state, groups=groups, softplus=softplus, skip=skip, gate=gate)
            v["delta"] = rounded(rng.standard_normal((self.rows, channels)) * 0.5, dtype)
            if not softplus:
                v["delta"] = rounded(np.abs(v["delta"]) * 0.1, dtype)
            v["A"] = par(-np.arange(1, state + 1) * np.exp(0.1 * rng.standard_normal((channels, state))))
            v["B"], v["C"] = tok(groups, state), tok(groups, state)
            if bias:
                v["bias"] = par(rng.uniform(-4.0, -1.0, channels) if softplus else np.zeros(channels))
            if skip:
                v["skip"] = par(1 + 0.1 * rng.standard_normal(channels))
            if gate:
                v["z"] = tok(channels)
            edge = (self.seqs, channels, state)
            if initial:
                v["initial"] = par(rng.standard_normal(edge))
            if final:
                v["dfinal"] = par(rng.standard_normal(edge))

    @property
    def grid(self):
        return (self.seqs, self.channels)

    # -- the operator itself ------------------------------------------------------------
    def oracle(self, grad=True):
        v = self.v
        extra = dict(dy=v["dy"] if grad else None, dfinal=v.get("dfinal") if grad else None)
        if self.kind == "conv":
            return S.causal_conv(v["x"], v["weight"], v.get("bias"), self.starts, v.get("initial"),
                                 silu=self.constants["silu"], **extra)
        return S.selective_scan(v["x"], v["delta"], v["A"], v["B"], v["C"], self.starts, v.get("bias"), v.get("skip"),
                                v.get("z"), v.get("initial"), softplus_=self.constants["softplus"], **extra)

    # -- operands in call order ----------------------------------------------------------
    def shaped(self, name):
        array = self.v[name]
        if name in ("x", "dy", "delta", "B", "C", "z") and not self.packed:
            return array.reshape((self.seqs, self.length) + array.shape[1:])
        return array

    def typed(self, name):
        short = name in ("x", "dy", "delta", "B", "C", "z") or (self.kind == "conv" and name in ("initial", "dfinal"))
        return host(self.shaped(name), self.dtype if short else "float32")

    def offsets(self):
        return [np.asarray(self.starts, np.int32)] if self.packed else []

    def operands(self, grad=False, carries=None):
        if self.kind == "conv":
            names = ["x", "weight", "bias", "initial"]
        else:
            names = ["x", "delta", "A", "B", "C", "bias", "skip", "z"] + ([] if grad else ["initial"])
        arrays = [self.typed(n) for n in (["dy"] if grad else []) + names if n in self.v]
        if grad:
            arrays += [] if carries is None else [carries]
            arrays += [self.typed("dfinal")] if "dfinal" in self.v else []
        return arrays + self.offsets()

    # -- calls ---------------------------------------------------------------------------
    def family(self, form="", **more):
        maker = getattr(families, ("causal_conv" if self.kind == "conv" else "selective_scan") + form)
        return maker(**{**self.constants, **more})

    def call(self, maker, form="", math_mode="fast", **more):
        family = self.family(form, **more)
        return maker(family, grid=self.grid, out_shape=families.out_shapes(family, self.grid), math_mode=math_mode)

    def forward_names(self):
        return ["y"] + ["final"] * self.constants["final"]

    def grad_names(self):
        c = self.constants
        if self.kind == "conv":
            return ["dx", "dweight"] + ["dbias"] * c["bias"] + ["dinitial"] * c["initial"]
        return (["dx", "ddelta", "dA", "dB", "dC"] + ["dbias"] * c["bias"] + ["dskip"] * c["skip"] + ["dz"] * c["gate"]
                + ["dinitial"] * c["initial"])

    def is_short(self, name):
        if self.kind == "conv":
            return name not in ("dweight", "dbias")
        return name in ("y", "dx", "ddelta", "dB", "dC", "dz")


def tolerance(r, dtype):
    """Twice the running bound of the float32 evaluation, then the rounding to `dtype` (for float32 it is
    part of the bound already)."""
    bound = 2.0 * S.UNIT * r.error
    if dtype != "float32":
        bound = bound + HALF_STEP[dtype] * (np.abs(r.value) + bound)
    return bound + SMALLEST[dtype] + 2.0 ** -126     # float32 results below 2^-126 may be flushed


def check(case, names, results, want=None):
    want = want if want is not None else case.oracle()
    results = results if isinstance(results, (tuple, list)) else (results,)
    assert len(names) == len(results)
    for name, got in zip(names, results):
        r = want[name]
        got = wide(np.asarray(got)).reshape(r.value.shape)
        dtype = case.dtype if case.is_short(name) else "float32"
        off, most = np.abs(got - r.value), tolerance(r, dtype)
        bad = ~(off <= most)
        assert not bad.any(), (f"{name}: {bad.sum()} of {bad.size} values outside; worst {np.nanmax(off / most):.3g} times "
                               f"the tolerance at {np.unravel_index(np.nanargmax(off / most), off.shape)}")
