"""The state-space operators as a user's program calls them: cases, inputs, plain forms and the values in 64 bits.

A case names an operator (`op`), its sizes and its element type.  `run` makes one pass: with `own` through
the framework's calls, without it through elementary torch operations in 32 bits.  Tokens are rows: a batch of
S sequences of L tokens has arrays (S, L, D); `packed` cases hold sequences of different lengths behind one
another in arrays (T, D) with their starts in `offsets` (S + 1), and rows behind the last sequence come out as zeros.
"""

import functools
import math

import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # one user's next token through the convolution: nothing but latency
        dict(name="conv_step_1", op="conv_step", seqs=1, length=1, channels=1536, width=4, dtype="bfloat16"),
        # the same for a full serving batch
        dict(name="conv_step_256", op="conv_step", seqs=256, length=1, channels=4096, width=4, dtype="bfloat16"),
        # prompts of different lengths packed behind one another, each continuing an earlier chunk
        dict(name="conv_packed", op="conv", seqs=13, length=8191, channels=2560, width=4, dtype="bfloat16",
             packed=True, initial=True, final=True),
        # the forward pass of a training batch
        dict(name="conv_batch", op="conv", seqs=8, length=2048, channels=4096, width=4, dtype="bfloat16",
             packed=False, initial=False, final=False),
        # gradients of a small model in 32 bits, every size odd
        dict(name="conv_grad_odd", op="conv_grad", seqs=3, length=517, channels=333, width=3, dtype="float32",
             packed=False, initial=True, final=True),
        # gradients of a training batch
        dict(name="conv_grad_batch", op="conv_grad", seqs=8, length=2048, channels=2048, width=4, dtype="bfloat16",
             packed=False, initial=False, final=False),
        # one user's next token through the recurrence
        dict(name="scan_step_1", op="scan_step", seqs=1, length=1, channels=1536, state=16, groups=1,
             dtype="bfloat16", gate=True),
        # a full serving batch: the states are read and written once
        dict(name="scan_step_256", op="scan_step", seqs=256, length=1, channels=4096, state=16, groups=1,
             dtype="bfloat16", gate=True),
        # one long prompt alone: few channels, many tokens
        dict(name="scan_long", op="scan", seqs=1, length=8192, channels=2048, state=16, groups=1, dtype="bfloat16",
             gate=True, packed=False, initial=False, final=True),
        # prompts of different lengths packed behind one another, each continuing an earlier chunk
        dict(name="scan_packed", op="scan", seqs=17, length=8200, channels=2560, state=16, groups=1,
             dtype="bfloat16", gate=True, packed=True, initial=True, final=True),
        # a training step of a small model in 32 bits, every size odd, channels in two groups
        dict(name="scan_train_odd", op="scan_train", seqs=2, length=333, channels=210, state=11, groups=2,
             dtype="float32", gate=True, packed=False, initial=True, final=True),
        # a training step: forward pass and all gradients
        dict(name="scan_train_batch", op="scan_train", seqs=4, length=2048, channels=2048, state=16, groups=1,
             dtype="bfloat16", gate=True, packed=False, initial=False, final=False),
    ]


MOST_CELLS = {"conv": 8 * 2048 * 4096, "conv_grad": 8 * 2048 * 2048, "conv_step": 256 * 4096,
              "scan": 8200 * 2560 * 16, "scan_train": 4 * 2048 * 2048 * 16, "scan_step": 256 * 4096 * 16}


def draw(rng):
    op = rng.choice(("conv_step", "conv", "conv_grad", "scan_step", "scan", "scan_train"))
    spread = lambda low, high: int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))  # noqa: E731
    case = dict(op=op, dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")), channels=spread(24, 5120))
    per_token = case["channels"]
    if op.startswith("scan"):
        case["groups"] = rng.choice((1, 1, 1, 2, 4))
        case["channels"] = per_token = -(-case["channels"] // case["groups"]) * case["groups"]
        case["state"] = rng.choice((16, 16, 16, 1, 4, 7, 8, 12, 24, 32, 64))
        case["gate"] = rng.random() < 0.7
        per_token *= case["state"]
    else:
        case["width"] = rng.choice((4, 4, 4, 2, 3))
    most = max(1, MOST_CELLS[op] // per_token)
    if op.endswith("step"):
        case.update(seqs=spread(1, min(256, most)), length=1)
        return case
    case["length"] = spread(1, min(8192, most))
    case["packed"] = rng.random() < 0.5
    if case["packed"]:
        case["seqs"] = spread(1, min(32, case["length"]))
    else:
        case["seqs"] = spread(1, max(1, min(16, most // case["length"])))
    case["initial"] = rng.random() < 0.5
    case["final"] = rng.random() < 0.5
    return case


# ----------------------------------------------------------------------------- inputs
def _starts(case, seed):
    """Where each sequence begins, and where the last one ends, as a list of seqs + 1 numbers."""
    s, n = case["seqs"], case["length"]
    if not case.get("packed"):
        return [i * n for i in range(s + 1)]
    # a few per cent of the rows stay unused, as in a buffer of fixed size
    used = n - n // 32
    g = torch.Generator().manual_seed(seed)
    cuts = torch.sort(torch.randint(0, used + 1, (s - 1,), generator=g))[0].tolist()
    return [0] + cuts + [used]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    s, n, d = case["seqs"], case["length"], case["channels"]
    rows = (s, d) if case["op"].endswith("step") else (n, d) if case.get("packed") else (s, n, d)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    state = dict(case=case, x=normal(*rows, dtype=t))
    starts = _starts(case, seed)
    if case.get("packed"):
        state["offsets"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    state["longest"] = max(b - a for a, b in zip(starts, starts[1:]))
    if case["op"].startswith("conv"):
        w = case["width"]
        state["weight"] = normal(d, w, scale=w ** -0.5)
        state["bias"] = normal(d, scale=0.1)
        if case["op"] == "conv_step" or case.get("initial"):
            state["initial"] = normal(s, w - 1, d, dtype=t)
        if case["op"] == "conv_grad":
            state["dy"] = normal(*rows, dtype=t)
            if case["final"]:
                state["dfinal"] = normal(s, w - 1, d, dtype=t)
        return state
    k, groups = case["state"], case["groups"]
    state["delta"] = normal(*rows, dtype=t, scale=0.5)
    # decay rates around 1 .. state, step sizes around 0.001 .. 0.1 after the softplus
    rates = torch.arange(1, k + 1, device="cuda", dtype=torch.float32).expand(d, k)
    state["A"] = -rates * torch.exp(normal(d, k, scale=0.1))
    size = torch.exp(torch.empty(d, device="cuda").uniform_(math.log(1e-3), math.log(1e-1), generator=g))
    state["delta_bias"] = size + torch.log(-torch.expm1(-size))
    state["skip"] = 1.0 + normal(d, scale=0.1)
    state["B"] = normal(*rows[:-1], groups, k, dtype=t)
    state["C"] = normal(*rows[:-1], groups, k, dtype=t)
    if case["gate"]:
        state["z"] = normal(*rows, dtype=t)
    if case["op"] == "scan_step" or case.get("initial"):
        state["initial"] = normal(s, d, k)
    if case["op"] == "scan_train":
        state["dy"] = normal(*rows, dtype=t)
        if case["final"]:
            state["dfinal"] = normal(s, d, k)
    return state


# ----------------------------------------------------------------------------- the framework's calls
@functools.lru_cache(maxsize=64)
def _call(kind, grid, **constants):
    """The call object a user's program builds once for its sizes and keeps."""
    import palladium_b200 as pd
    from palladium_b200 import families

    family = getattr(families, kind)(**constants)
    return pd.cuda_call_jit(family, grid=grid, out_shape=families.out_shapes(family, grid))


def _named(names, values):
    return dict(zip(names, values if isinstance(values, tuple) else (values,)))


def _own(state):
    case = state["case"]
    op, grid = case["op"], (case["seqs"], case["channels"])
    given = lambda *names: [state[n] for n in names if n in state]  # noqa: E731
    if op == "conv_step":
        call = _call("causal_conv_step", grid, width=case["width"], dtype=case["dtype"])
        return _named(("y", "final"), call(state["x"], state["initial"], state["weight"], state["bias"]))
    if op == "scan_step":
        call = _call("selective_scan_step", grid, state=case["state"], groups=case["groups"], gate=case["gate"],
                     dtype=case["dtype"])
        return _named(("y", "final"), call(state["initial"], *given("x", "delta", "A", "B", "C", "delta_bias", "skip", "z")))
    common = dict(length=case["length"], packed=case["packed"], initial=case["initial"], final=case["final"],
                  dtype=case["dtype"])
    if op == "conv":
        call = _call("causal_conv", grid, width=case["width"], **common)
        return _named(("y", "final"), call(*given("x", "weight", "bias", "initial", "offsets")))
    if op == "conv_grad":
        call = _call("causal_conv_grad", grid, width=case["width"], **common)
        grads = call(*given("dy", "x", "weight", "bias", "initial", "dfinal", "offsets"))
        return _named(("dx", "dweight", "dbias", "dinitial"), grads)
    common.update(state=case["state"], groups=case["groups"], gate=case["gate"])
    operands = given("x", "delta", "A", "B", "C", "delta_bias", "skip", "z")
    if op == "scan":
        return _named(("y", "final"), _call("selective_scan", grid, **common)(*operands, *given("initial", "offsets")))
    *results, carries = _call("selective_scan", grid, carries=True, **common)(*operands, *given("initial", "offsets"))
    grads = _call("selective_scan_grad", grid, **common)(state["dy"], *operands, carries, *given("dfinal", "offsets"))
    names = ["dx", "ddelta", "dA", "dB", "dC", "ddelta_bias", "dskip"] + ["dz"] * case["gate"] + ["dinitial"]
    return {**_named(("y", "final"), tuple(results)), **_named(names, grads)}


# ----------------------------------------------------------------------------- plain forms, 32 bits
def _places(state):
    """(row, sequence, position in the sequence, length of the sequence, whether a sequence has it) of every token row."""
    case = state["case"]
    s = case["seqs"]
    if "offsets" in state:
        starts = state["offsets"].long()
        row = torch.arange(case["length"], device="cuda")
        seq = torch.searchsorted(starts[1:], row, right=True)
        inside = seq < s
        seq = seq.clamp(max=s - 1)
        return row, seq, row - starts[seq], (starts[1:] - starts[:-1])[seq], inside, starts
    row = torch.arange(s * case["length"], device="cuda")
    seq, pos = row // case["length"], row % case["length"]
    starts = torch.arange(s + 1, device="cuda") * case["length"]
    return row, seq, pos, torch.full_like(pos, case["length"]), torch.ones_like(pos, dtype=torch.bool), starts


def _silu(v):
    return v / (1.0 + torch.exp(-v))


def _silu_slope(v):
    s = 1.0 / (1.0 + torch.exp(-v))
    return s * (1.0 + v * (1.0 - s))


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-torch.abs(v)))


def _plain_conv(state):
    case = state["case"]
    t, d, w, s = TYPES[case["dtype"]], case["channels"], case["width"], case["seqs"]
    row, seq, pos, count, inside, starts = _places(state)
    x = state["x"].reshape(-1, d).float()
    before = state["initial"].reshape(-1, d).float() if "initial" in state else x.new_zeros(s * (w - 1), d)
    values = torch.cat([x, before])
    back = torch.arange(w - 1, -1, -1, device="cuda")   # how far behind the token each tap lies
    at = torch.where(pos[:, None] >= back, row[:, None] - back, len(x) + seq[:, None] * (w - 1) + w - 1 + pos[:, None] - back)
    seen = values[at]                                    # (T, W, D)
    pre = (seen * state["weight"].float().t()).sum(1) + state["bias"].float()
    last = torch.arange(w - 1, device="cuda") + (starts[1:] - starts[:-1])[:, None] - (w - 1)
    last = torch.where(last >= 0, starts[:-1, None] + last, len(x) + torch.arange(s, device="cuda")[:, None] * (w - 1) + w - 1 + last)
    keep = inside[:, None]
    if case["op"] != "conv_grad":
        out = {"y": (_silu(pre) * keep).to(t).reshape(state["x"].shape)}
        if case["op"] == "conv_step" or case["final"]:
            out["final"] = values[last].to(t)
        return out
    g = state["dy"].reshape(-1, d).float() * _silu_slope(pre) * keep
    dvalues = torch.zeros_like(values)
    ahead = torch.arange(w, device="cuda")               # the tokens that see this one
    there = (pos[:, None] + ahead < count[:, None]) & keep
    taken = g[torch.where(there, row[:, None] + ahead, 0)] * there[:, :, None]
    dvalues[:len(x)] = (taken * state["weight"].float().flip(1).t()).sum(1)
    if "initial" in state:
        # row i of the carried-in inputs lies w - 1 - i tokens before the first one
        near = torch.arange(w - 1, device="cuda")[:, None] - (w - 1) + ahead          # position of the token that sees it
        there = (near >= 0) & (near < (starts[1:] - starts[:-1])[:, None, None])      # (S, W-1, W)
        taken = g[torch.where(there, starts[:-1, None, None] + near, 0)] * there[..., None]
        dvalues[len(x):] = (taken * state["weight"].float().flip(1).t()).sum(2).reshape(-1, d)
    if "dfinal" in state:
        dvalues.index_add_(0, last.reshape(-1), state["dfinal"].reshape(-1, d).float())
    out = {"dx": dvalues[:len(x)].to(t).reshape(state["x"].shape),
           "dweight": (seen * g[:, None]).sum(0).t().contiguous(), "dbias": g.sum(0)}
    if "initial" in state:
        out["dinitial"] = dvalues[len(x):].to(t).reshape(s, w - 1, d)
    return out


def _plain_scan(state):
    case = state["case"]
    t, d, k, s = TYPES[case["dtype"]], case["channels"], case["state"], case["seqs"]
    per = d // case["groups"]
    row, seq, pos, count, inside, starts = _places(state)
    x = state["x"].reshape(-1, d).float()
    raw = state["delta"].reshape(-1, d).float() + state["delta_bias"]
    delta = _softplus(raw)
    wide = lambda v: v.reshape(-1, case["groups"], k).float().repeat_interleave(per, 1)  # noqa: E731 (T, D, N)
    b, c = wide(state["B"]), wide(state["C"])
    decay = torch.exp(delta[:, :, None] * state["A"])
    first, keep = (pos == 0)[:, None, None], inside[:, None, None]
    entering = state["initial"][seq] if "initial" in state else 0.0
    # the recurrence h = decay * h_before + u by doubling: after each pass a row holds the sum over twice as many
    h = (delta * x)[:, :, None] * b + torch.where(first, decay * entering, 0.0)
    a = torch.where(first, 0.0, decay)
    step = 1
    while step < state["longest"]:
        h = torch.cat([h[:step], h[step:] + a[step:] * h[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    y = (h * c).sum(2) + state["skip"] * x
    gated = y * _silu(state["z"].reshape(-1, d).float()) if case["gate"] else y
    out = {"y": (gated * inside[:, None]).to(t).reshape(state["x"].shape)}
    if case["op"] == "scan_step" or case["final"]:
        lengths = starts[1:] - starts[:-1]
        ends = h[(starts[1:] - 1).clamp(min=0)]
        empty = state["initial"] if "initial" in state else torch.zeros_like(ends)
        out["final"] = torch.where((lengths > 0)[:, None, None], ends, empty)
    if case["op"] != "scan_train":
        return out
    dy = state["dy"].reshape(-1, d).float() * inside[:, None]
    if case["gate"]:
        z = state["z"].reshape(-1, d).float()
        dz = dy * y * _silu_slope(z)
        dy = dy * _silu(z)
    last = (pos == count - 1)[:, None, None] & keep
    g = dy[:, :, None] * c * keep
    if "dfinal" in state:
        g = g + torch.where(last, state["dfinal"][seq], 0.0)
    following = torch.where(last | ~keep, 0.0, torch.cat([decay[1:], torch.zeros_like(decay[:1])]))
    step = 1
    while step < state["longest"]:
        g = torch.cat([g[:-step] + following[:-step] * g[step:], g[-step:]])
        following = torch.cat([following[:-step] * following[step:], following[-step:]])
        step *= 2
    del following, a
    h = torch.cat([torch.zeros_like(h[:1]), h[:-1]])     # the state before each token
    h = torch.where(first, entering, h)
    kept = g * decay
    moved = kept * h
    group = lambda v: v.reshape(-1, case["groups"], per, k).sum(2).to(t).reshape(state["B"].shape)  # noqa: E731
    grad_u = (g * b).sum(2)
    ddelta = ((moved * state["A"]).sum(2) + grad_u * x) / (1.0 + torch.exp(-raw))
    u = (delta * x)[:, :, None]
    out["dx"] = (grad_u * delta + dy * state["skip"]).to(t).reshape(state["x"].shape)
    out["ddelta"] = ddelta.to(t).reshape(state["x"].shape)
    out["dA"] = (moved * delta[:, :, None]).sum(0)
    out["dB"] = group(g * u)
    out["dC"] = group((decay * h + u * b) * dy[:, :, None])
    out["ddelta_bias"] = ddelta.sum(0)
    out["dskip"] = (dy * x).sum(0)
    if case["gate"]:
        out["dz"] = dz.to(t).reshape(state["x"].shape)
    if case["initial"]:
        begins = kept[starts[:-1].clamp(max=len(x) - 1)]
        empty = state["dfinal"] if "dfinal" in state else torch.zeros_like(begins)
        out["dinitial"] = torch.where((starts[1:] > starts[:-1])[:, None, None], begins, empty)
    return out


def run(state):
    if own:
        return _own(state)
    return _plain_conv(state) if state["case"]["op"].startswith("conv") else _plain_scan(state)


# ----------------------------------------------------------------------------- 64 bits, token by token
def exact(case, seed):
    """The definitions token by token in 64 bits; gradients by differentiating those very steps."""
    state = prepare(case, seed)
    starts = _starts(case, seed)
    op, s, d = case["op"], case["seqs"], case["channels"]
    lengths = [b - a for a, b in zip(starts, starts[1:])]
    most = max(lengths)
    rows = state["x"].numel() // d
    training = op in ("conv_grad", "scan_train")
    wide = {k: v.double().requires_grad_(training and k not in ("dy", "dfinal")) for k, v in state.items()
            if isinstance(v, torch.Tensor) and v.is_floating_point()}
    alive = torch.tensor(lengths, device="cuda")
    at = torch.tensor(starts[:-1], device="cuda") + torch.arange(most, device="cuda")[:, None]          # (longest, S)
    live = torch.arange(most, device="cuda")[:, None] < alive
    at = torch.where(live, at, rows)
    inner = 1 if op.endswith("step") or case.get("packed") else 2
    tokens = {n: wide[n].reshape(rows, *wide[n].shape[inner:])[at.clamp(max=rows - 1)].unbind(0)
              for n in ("x", "delta", "B", "C", "z") if n in wide}
    outs = [wide["x"].new_zeros(0, s, d)]
    if op.startswith("conv"):
        w = case["width"]
        window = list((wide["initial"] if "initial" in wide else wide["x"].new_zeros(s, w - 1, d)).unbind(1))
        for p in range(most):
            window.append(tokens["x"][p])
            pre = sum(window[i] * wide["weight"][:, i] for i in range(w)) + wide["bias"]
            outs.append((pre * torch.sigmoid(pre))[None])
            window = [torch.where(live[p][:, None], window[i + 1], window[i]) for i in range(w - 1)]
        final = torch.stack(window, 1)
    else:
        h = wide["initial"] if "initial" in wide else wide["x"].new_zeros(s, d, case["state"])
        spread = lambda v: v.repeat_interleave(d // case["groups"], 1)  # noqa: E731
        for p in range(most):
            raw = tokens["delta"][p] + wide["delta_bias"]
            delta = torch.logaddexp(raw, torch.zeros_like(raw))
            new = torch.exp(delta[..., None] * wide["A"]) * h + (delta * tokens["x"][p])[..., None] * spread(tokens["B"][p])
            y = torch.einsum("sdn,sdn->sd", new, spread(tokens["C"][p])) + wide["skip"] * tokens["x"][p]
            if case["gate"]:
                y = y * tokens["z"][p] * torch.sigmoid(tokens["z"][p])
            outs.append(y[None])
            h = torch.where(live[p][:, None, None], new, h)
        final = h
    # rows of no sequence stay zero; what lies behind a sequence's end goes to a row that is dropped
    y = wide["x"].new_zeros(rows + 1, d).index_put((at.reshape(-1),), torch.cat(outs).reshape(-1, d), accumulate=True)
    y = y[:rows].reshape(state["x"].shape)
    out = {}
    if op != "conv_grad":
        out["y"] = y.detach()
        if op.endswith("step") or case["final"]:
            out["final"] = final.detach()
    if training:
        value = (y * wide["dy"]).sum() + ((final * wide["dfinal"]).sum() if "dfinal" in wide else 0.0)
        order = [n for n in ("x", "weight", "bias", "delta", "A", "B", "C", "delta_bias", "skip", "z", "initial") if n in wide]
        grads = torch.autograd.grad(value, [wide[n] for n in order], allow_unused=True)
        out.update({"d" + n: torch.zeros_like(wide[n]) if v is None else v.detach() for n, v in zip(order, grads)})
    return out


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = TYPES[case["dtype"]].itemsize
    op, s, d = case["op"], case["seqs"], case["channels"]
    tokens = s if op.endswith("step") else case["length"] if case["packed"] else s * case["length"]
    cells = tokens * d
    ends = 2 if op.endswith("step") else case["initial"] + case["final"]
    if op.startswith("conv"):
        w = case["width"]
        edge = s * (w - 1) * d * size
        if op == "conv_grad":
            read, write = 2 * cells * size, cells * size
            return {"bytes": read + write + 8 * d * (w + 1) + edge * (2 * case["initial"] + case["final"]),
                    "flops": cells * (6 * w + 10)}
        return {"bytes": 2 * cells * size + 4 * d * (w + 1) + edge * ends, "flops": cells * (2 * w + 6)}
    k, groups, gate = case["state"], case["groups"], case["gate"]
    params = 4 * d * (k + 2)
    coupling = 2 * tokens * groups * k * size
    edge = 4 * s * d * k
    forward = {"bytes": (3 + gate) * cells * size + coupling + params + edge * ends, "flops": cells * (7 * k + 12)}
    if op != "scan_train":
        return forward
    # the backward pass reads the inputs and the gradient again and writes a gradient for each input
    return {"bytes": forward["bytes"] + (3 + gate + 2 + gate) * cells * size + 2 * coupling + 2 * params + edge * ends,
            "flops": forward["flops"] + cells * (22 * k + 30)}
