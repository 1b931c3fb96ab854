"""The state-space operators in float64 NumPy, token by token, with a running
error analysis: what a float32 evaluation of the same formulas may be off by.

`Rough` carries a value and a bound of its error in units of 2^-24 (half a float32
step relative to 1).  Every operation adds the error its own rounding can make and
passes on those of its operands, to first order, so a test's tolerance follows from
the formula and the inputs alone.  A kernel may associate a recurrence's products
and sums differently (a token's contribution still passes through no more roundings
than tokens), which the tests' factor of two on the bound covers.
"""

from __future__ import annotations

import numpy as np

UNIT = 2.0 ** -24


class Rough:
    __array_priority__ = 100

    def __init__(self, value, error=0.0):
        self.value = np.asarray(value, np.float64)
        self.error = np.broadcast_to(np.asarray(error, np.float64), self.value.shape)

    def __getitem__(self, key):
        return Rough(self.value[key], self.error[key])

    def __neg__(self):
        return Rough(-self.value, self.error)

    def __add__(self, other):
        other = rough(other)
        value = self.value + other.value
        return Rough(value, self.error + other.error + np.abs(value))

    __radd__ = __add__

    def __sub__(self, other):
        return self + (-rough(other))

    def __rsub__(self, other):
        return rough(other) + (-self)

    def __mul__(self, other):
        other = rough(other)
        value = self.value * other.value
        return Rough(value, np.abs(self.value) * other.error + np.abs(other.value) * self.error + np.abs(value))

    __rmul__ = __mul__

    def sum(self, axis):
        """n terms in any order: each passes through at most n additions."""
        n = self.value.shape[axis]
        return Rough(self.value.sum(axis), self.error.sum(axis) + n * np.abs(self.value).sum(axis))


def rough(v) -> Rough:
    return v if isinstance(v, Rough) else Rough(v)


def exp(v: Rough) -> Rough:
    """e^v as 2^(v log2 e): the argument is rounded twice (2 |v|), the approximate
    power is off by 2^-22 (4 units)."""
    value = np.exp(v.value)
    return Rough(value, value * (v.error + 2 * np.abs(v.value) + 4))


def sigmoid(v: Rough) -> Rough:
    """1 / (1 + e^-v): slope s (1 - s), an exponential (4 + 2 |v|, as above, which reaches the
    result through 1 - s), a sum and a division of two units' error."""
    s = 1.0 / (1.0 + np.exp(-v.value))
    return Rough(s, s * (1 - s) * (v.error + 4 + 2 * np.abs(v.value)) + 3 * s)


def softplus(v: Rough) -> Rough:
    """max(v, 0) + log1p(e^-|v|): slope sigmoid(v); log1p is within two units of its value and
    passes on the exponential's error times 1 / (1 + e) <= 1."""
    e = np.exp(-np.abs(v.value))
    value = np.maximum(v.value, 0.0) + np.log1p(e)
    return Rough(value, v.error / (1.0 + np.exp(-v.value)) + e * (4 + 2 * np.abs(v.value)) + 2 * np.log1p(e) + value)


def stack(parts) -> Rough:
    return Rough(np.stack([p.value for p in parts]), np.stack([p.error for p in parts]))


class Rows:
    """An output's token rows, zero (and exactly so) where no sequence has them."""

    def __init__(self, *shape):
        self.value, self.error = np.zeros(shape), np.zeros(shape)

    def put(self, row, v: Rough):
        self.value[row], self.error[row] = v.value, v.error

    def rough(self):
        return Rough(self.value, self.error)


def causal_conv(x, weight, bias, starts, initial=None, *, silu=True, dy=None, dfinal=None):
    """x (rows, D), sequences in rows starts[s] .. starts[s + 1].  Returns {"y", "final"} and, given dy,
    the gradients."""
    rows, d = x.shape
    w = weight.shape[1]
    seqs = len(starts) - 1
    weight = Rough(weight)
    bias = None if bias is None else Rough(bias)
    y, final = Rows(rows, d), np.zeros((seqs, w - 1, d))
    dx, dinitial = Rows(rows, d), Rows(seqs, w - 1, d)
    dweight, dbias = [Rough(np.zeros((1, d)))] * w, Rough(np.zeros((1, d)))
    terms = [[] for _ in range(w)], []
    for s in range(seqs):
        n = starts[s + 1] - starts[s]
        before = np.zeros((w - 1, d)) if initial is None else initial[s]
        seen = np.concatenate([before, x[starts[s]:starts[s + 1]]])
        final[s] = seen[n:]
        gs = []
        for t in range(n):
            pre = Rough(np.zeros(d))
            for k in range(w):
                pre = pre + weight[:, k] * seen[t + k]
            if bias is not None:
                pre = pre + bias
            sig = sigmoid(pre)
            y.put(starts[s] + t, pre * sig if silu else pre)
            if dy is not None:
                g = Rough(dy[starts[s] + t])
                gs.append(g * (sig * (1.0 + pre * (1.0 - sig))) if silu else g)
        if dy is None:
            continue
        for i in range(n + w - 1):       # row i of `seen` is read by tokens i - (w - 1) .. i
            total = Rough(np.zeros(d))
            for k in range(w):
                if 0 <= i - k < n:
                    total = total + weight[:, k] * gs[i - k]
            if dfinal is not None and i >= n:
                total = total + dfinal[s, i - n]
            if i >= w - 1:
                dx.put(starts[s] + i - (w - 1), total)
            else:
                dinitial.put((s, i), total)
        for t, g in enumerate(gs):
            for k in range(w):
                terms[0][k].append(g * seen[t + k])
            terms[1].append(g)
    out = {"y": y.rough(), "final": Rough(final)}
    if dy is not None:
        if terms[1]:
            dweight, dbias = [stack(t).sum(0) for t in terms[0]], stack(terms[1]).sum(0)
        else:
            dweight, dbias = [Rough(np.zeros(d))] * w, Rough(np.zeros(d))
        out.update(dx=dx.rough(), dweight=Rough(np.stack([v.value for v in dweight], 1), np.stack([v.error for v in dweight], 1)),
                   dbias=dbias, dinitial=dinitial.rough())
    return out


def selective_scan(x, delta, A, B, C, starts, bias=None, skip=None, z=None, initial=None, *, softplus_=True, dy=None,
                   dfinal=None):
    """x, delta, z (rows, D), B, C (rows, groups, N).  Returns {"y", "final"} and, given dy, the gradients."""
    rows, d = x.shape
    k, groups = A.shape[1], B.shape[1]
    per, seqs = d // groups, len(starts) - 1
    A = Rough(A)
    y, final = Rows(rows, d), Rows(seqs, d, k)
    grads = {n: Rows(rows, d) for n in ("dx", "ddelta", "dz")}
    grads.update(dB=Rows(rows, groups, k), dC=Rows(rows, groups, k), dinitial=Rows(seqs, d, k))
    sums = {"dA": [Rough(np.zeros((d, k)))], "dbias": [Rough(np.zeros(d))], "dskip": [Rough(np.zeros(d))]}
    for s in range(seqs):
        h = Rough(np.zeros((d, k)) if initial is None else initial[s])
        kept = []
        for r in range(starts[s], starts[s + 1]):
            raw = Rough(delta[r]) if bias is None else Rough(delta[r]) + bias
            step = softplus(raw) if softplus_ else raw
            decay = exp(step[:, None] * A)
            wide_b, wide_c = np.repeat(B[r], per, 0), np.repeat(C[r], per, 0)
            u = step * x[r]
            before, h = h, decay * h + u[:, None] * wide_b
            out = (h * wide_c).sum(1)
            if skip is not None:
                out = out + Rough(skip) * x[r]
            if z is not None:
                gate = Rough(z[r]) * sigmoid(Rough(z[r]))
            y.put(r, out if z is None else out * gate)
            kept.append((r, raw, step, decay, wide_b, wide_c, u, before, h, out))
        final.put(s, h)
        if dy is None:
            continue
        g = Rough(np.zeros((d, k)) if dfinal is None else dfinal[s])
        for r, raw, step, decay, wide_b, wide_c, u, before, h, out in reversed(kept):
            v = Rough(dy[r])
            if z is not None:
                sig = sigmoid(Rough(z[r]))
                grads["dz"].put(r, v * out * (sig * (1.0 + Rough(z[r]) * (1.0 - sig))))
                v = v * (Rough(z[r]) * sig)
            g = g + v[:, None] * wide_c
            group = lambda q: Rough(q.value.reshape(groups, per, k), q.error.reshape(groups, per, k)).sum(1)  # noqa: E731
            grads["dB"].put(r, group(g * u[:, None]))
            grads["dC"].put(r, group(h * v[:, None]))
            du = (g * wide_b).sum(1)
            g = g * decay
            moved = g * before
            dd = (moved * A).sum(1) + du * x[r]
            if softplus_:
                dd = dd * sigmoid(raw)
            grads["ddelta"].put(r, dd)
            grads["dx"].put(r, du * step if skip is None else du * step + v * Rough(skip))
            sums["dA"].append(moved * step[:, None])
            sums["dbias"].append(dd)
            sums["dskip"].append(v * x[r])
        grads["dinitial"].put(s, g)
    out = {"y": y.rough(), "final": final.rough()}
    if dy is not None:
        out.update({n: v.rough() for n, v in grads.items()})
        out.update({n: stack(v).sum(0) for n, v in sums.items()})
    return out
