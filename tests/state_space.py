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


# -- the operators as `.interpret` gives them: from a call's arrays to its results, float64 rounded once ------------
def interpret(family, grid, *args):
    """What a call of `family` on host arrays returns, from the oracle."""
    c, form = family.constants, family.name
    seqs, channels = grid
    scan, step, grad = form.startswith("selective_scan"), form.endswith("_step"), form.endswith("_grad")
    names = ["x", "delta", "A", "B", "C"] if scan else ["x", "weight"]
    names += [n for n in ("bias", "skip", "z") if c.get("gate" if n == "z" else n)]
    if step:
        names = ["initial"] + names if scan else ["x", "initial"] + names[1:]
    elif grad:
        names = ["dy"] + names + (["carries"] if scan else ["initial"] * c["initial"]) + ["dfinal"] * c["final"]
    else:
        names += ["initial"] * c["initial"]
    names += ["offsets"] * c["packed"]
    assert len(names) == len(args)
    v = {n: (np.asarray(a) if n == "offsets" else wide(np.asarray(a))) for n, a in zip(names, args)}
    length = 1 if step else c["length"]
    rows = length if c["packed"] else seqs * length
    starts = [int(o) for o in np.clip(v["offsets"], 0, rows)] if c["packed"] else [s * length for s in range(seqs + 1)]
    flat = {n: v[n].reshape((rows,) + v[n].shape[-1 if n in ("x", "dy", "delta", "z") else -2:]) for n in
            ("x", "dy", "delta", "z", "B", "C") if n in v}
    initial = v.get("initial")
    if scan and grad:
        initial = np.zeros((seqs, channels, c["state"]))
        for s in range(seqs):
            if starts[s + 1] > starts[s]:
                initial[s] = v["carries"][starts[s] // families.SCAN_CHUNK + s] if c["packed"] else v["carries"][s, 0]
    given = dict(dy=flat.get("dy"), dfinal=v.get("dfinal"))

    def run(starts, initial, **more):
        if scan:
            return S.selective_scan(flat["x"], flat["delta"], v["A"], flat["B"], flat["C"], starts, v.get("bias"),
                                    v.get("skip"), flat.get("z"), initial, softplus_=c["softplus"], **more)
        return S.causal_conv(flat["x"], v["weight"], v.get("bias"), starts, initial, silu=c["silu"], **more)

    found = {n: r.value for n, r in run(starts, initial, **given).items()}
    if c.get("carries"):
        kept = found["carries"] = np.zeros(families.out_shapes(family, grid)[-1].shape)
        for s in range(seqs):
            for k in range(-(-(starts[s + 1] - starts[s]) // families.SCAN_CHUNK)):
                before = run([starts[s], starts[s] + k * families.SCAN_CHUNK], None if initial is None else initial[s:s + 1])
                kept[(starts[s] // families.SCAN_CHUNK + s + k,) if c["packed"] else (s, k)] = before["final"].value[0]
    if not grad:
        order = ["y"] + ["final"] * (step or c["final"]) + ["carries"] * bool(c.get("carries"))
    elif scan:
        order = ["dx", "ddelta", "dA", "dB", "dC"] + [n for n, f in (("dbias", "bias"), ("dskip", "skip"), ("dz", "gate"),
                                                                     ("dinitial", "initial")) if c[f]]
    else:
        order = ["dx", "dweight"] + [n for n, f in (("dbias", "bias"), ("dinitial", "initial")) if c[f]]
    shapes = families.out_shapes(family, grid)
    shapes = shapes if isinstance(shapes, tuple) else (shapes,)
    results = tuple(host(rounded(found[n], pl.dtype_name(o.dtype)), pl.dtype_name(o.dtype)).reshape(o.shape)
                    for n, o in zip(order, shapes, strict=True))
    return results[0] if len(results) == 1 else results
