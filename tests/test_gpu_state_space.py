"""The state-space families on a GPU against the float64 operators, inside the bounds that their running
error analysis gives (tests/state_space.py)."""

import numpy as np
import pytest
import torch

import palladium_b200 as pd
from palladium_b200 import DispatchError, families, pl
from tests.state_space import TYPES, Case, check, wide

pytestmark = pytest.mark.gpu


def device(array):
    """A CUDA tensor with an array's bits."""
    if array.dtype == pl.bfloat16:
        return torch.from_numpy(np.ascontiguousarray(array).view(np.uint16).copy()).cuda().view(torch.bfloat16)
    return torch.from_numpy(np.array(array)).cuda()


def back(tensor):
    if tensor.dtype == torch.bfloat16:
        return tensor.view(torch.uint16).cpu().numpy().view(pl.bfloat16)
    return tensor.cpu().numpy()


def results(value):
    return [back(t) for t in (value if isinstance(value, tuple) else (value,))]


def run(case, math_mode="fast", grad=True):
    """The forward results, and the gradients behind them."""
    operands = [device(a) for a in case.operands()]
    scan = case.kind == "scan"
    forward = results(case.call(pd.cuda_call_jit, math_mode=math_mode, **(dict(carries=True) if scan else {}))(*operands))
    carries = device(forward.pop()) if scan else None
    if not grad:
        return forward, None
    operands = [device(a) for a in case.operands(grad=True, carries=back(carries) if scan else None)]
    return forward, results(case.call(pd.cuda_call_jit, "_grad", math_mode=math_mode)(*operands))


def compare(case, math_mode="fast"):
    forward, grads = run(case, math_mode)
    want = case.oracle()
    check(case, case.forward_names(), forward, want)
    check(case, case.grad_names(), grads, want)


# ------------------------------------------------------------------ the operators
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("lengths, channels", [([1], 1), ([2, 2], 8), ([3, 3, 3], 17), ([40, 40], 64), ([131], 136)])
def test_conv_dense(dtype, width, lengths, channels):
    for flags in (dict(), dict(initial=True, final=True), dict(silu=False, bias=False, final=True)):
        compare(Case("conv", lengths, channels, dtype=dtype, width=width, seed=width, **flags))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths, lead, spare", [([5, 1, 0, 2, 70, 3], 0, 0), ([0, 0, 1], 4, 9), ([33], 0, 31), ([0], 2, 3)])
@pytest.mark.parametrize("initial, final", [(False, False), (True, True), (True, False), (False, True)])
def test_conv_packed(dtype, lengths, lead, spare, initial, final):
    compare(Case("conv", lengths, 24, dtype=dtype, packed=True, lead=lead, spare=spare, initial=initial, final=final))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("state, channels, groups", [(1, 5, 1), (4, 33, 1), (5, 12, 3), (8, 16, 2), (11, 34, 2), (16, 40, 1),
                                                     (16, 72, 4), (24, 20, 1), (32, 8, 1), (64, 6, 2)])
def test_scan_dense(dtype, state, channels, groups):
    for lengths, flags in (([1], dict(final=True)), ([65, 65], dict(gate=True, initial=True, final=True)),
                           ([37, 37], dict(softplus=False, bias=False, skip=False)), ([130], dict(gate=True))):
        compare(Case("scan", lengths, channels, dtype=dtype, state=state, groups=groups, seed=state, **flags))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths, lead, spare", [([5, 1, 0, 64, 70, 3], 0, 0), ([0, 0, 1], 4, 9), ([129], 0, 31), ([0], 2, 3)])
@pytest.mark.parametrize("initial, final", [(False, False), (True, True), (True, False), (False, True)])
def test_scan_packed(dtype, lengths, lead, spare, initial, final):
    compare(Case("scan", lengths, 20, dtype=dtype, groups=2, gate=True, packed=True, lead=lead, spare=spare,
                 initial=initial, final=final))


@pytest.mark.parametrize("math_mode", ["safe", "relaxed", "fast"])
@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_math_modes(kind, math_mode):
    compare(Case(kind, [70, 70], 48, initial=True, final=True, **({} if kind == "conv" else dict(gate=True))), math_mode)


def test_scan_many_tiles_and_long():
    # several thousand tokens through many chunks, and more channels than one block takes
    compare(Case("scan", [2500], 40, state=16, gate=True, final=True, dtype="bfloat16"))
    compare(Case("scan", [9, 9], 700, state=16, dtype="bfloat16"))


@pytest.mark.parametrize("state, groups", [(16, 1), (3, 2), (20, 1), (64, 1)])
def test_scan_cut_into_segments(state, groups):
    """Few channels and many tokens: sequences are cut, and the states between the cuts composed."""
    flags = dict(state=state, groups=groups, gate=True, initial=True, final=True)
    case = Case("scan", [700], 12, **flags)
    assert case.call(pd.cuda_call).explain(*case.operands()).launches == 2
    compare(case)
    packed = Case("scan", [300, 0, 1, 450, 64], 12, packed=True, lead=3, spare=40, dtype="bfloat16", **flags)
    assert packed.call(pd.cuda_call).explain(*packed.operands()).launches == 2
    compare(packed)


@pytest.mark.parametrize("state, dtype", [(16, "bfloat16"), (13, "float32"), (24, "float16")])
def test_scan_two_channels_per_lane(state, dtype):
    """Calls of many blocks: each lane takes two channels."""
    case = Case("scan", [37] * 60, 1024, state=state, dtype=dtype, gate=True, initial=True, final=True)
    assert case.call(pd.cuda_call).explain(*case.operands()).items_per_thread == 2
    forward, _ = run(case, grad=False)
    check(case, case.forward_names(), forward, case.oracle(grad=False))


def test_conv_many_runs():
    for flags in (dict(), dict(packed=True, lead=2, spare=3, initial=True, final=True)):
        compare(Case("conv", [900, 900] if not flags else [700, 1, 0, 1100], 72, **flags))


# ------------------------------------------------------------------ single tokens, and prompts in parts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs, channels, state, groups", [(1, 1, 1, 1), (3, 40, 16, 2), (130, 24, 16, 1), (2, 9, 5, 3), (2, 12, 64, 1),
                                                           (83, 2048, 16, 1)])
def test_steps_match_the_prompt_form(dtype, seqs, channels, state, groups):
    """One token through the step families is a prompt of one token."""
    for kind, more in (("conv", {}), ("scan", dict(state=state, groups=groups, gate=True))):
        case = Case(kind, [1] * seqs, channels, dtype=dtype, initial=True, final=True, seed=seqs, **more)
        ops = dict(zip([n for n in ("x", "weight", "delta", "A", "B", "C", "bias", "skip", "z", "initial") if n in case.v], [None] * 20))
        tensors = {n: device(case.typed(n)) for n in ops}
        for n in ("x", "delta", "B", "C", "z"):
            if n in tensors:
                tensors[n] = tensors[n].reshape(tensors[n].shape[:1] + tensors[n].shape[2:])
        c = case.constants
        if kind == "conv":
            fam = families.causal_conv_step(c["width"], dtype=dtype)
            order = ["x", "initial", "weight", "bias"]
        else:
            fam = families.selective_scan_step(state, groups=groups, gate=True, dtype=dtype)
            order = ["initial", "x", "delta", "A", "B", "C", "bias", "skip", "z"]
        call = pd.cuda_call_jit(fam, grid=case.grid, out_shape=families.out_shapes(fam, case.grid))
        got = call(*[tensors[n] for n in order])
        check(case, ["y", "final"], results(got), case.oracle(grad=False))
        # in place: the new state lands in the old one's memory
        y = torch.empty_like(got[0])
        call.on_device(*[tensors[n] for n in order], out=(y, tensors["initial"]))
        assert torch.equal(y, got[0]) and torch.equal(tensors["initial"], got[1])


def test_steps_of_more_sequences_than_a_launch_dimension_holds():
    """The last of 70 000 sequences come out as they do alone."""
    torch.manual_seed(3)
    s, d, k = 70_000, 4, 2

    def step(family, order):
        make = lambda n: pd.cuda_call_jit(family, grid=(n, d), out_shape=families.out_shapes(family, (n, d)))  # noqa: E731
        whole = make(s)(*[t for t, _ in order])
        tail = make(100)(*[t[-100:].contiguous() if per_sequence else t for t, per_sequence in order])
        assert all(torch.equal(a[-100:], b) for a, b in zip(whole, tail))

    rand = lambda *shape: torch.randn(*shape, device="cuda")  # noqa: E731
    step(families.causal_conv_step(), [(rand(s, d), 1), (rand(s, 3, d), 1), (rand(d, 4), 0), (rand(d), 0)])
    step(families.selective_scan_step(k), [(rand(s, d, k), 1), (rand(s, d), 1), (rand(s, d), 1), (-rand(d, k).abs(), 0),
                                           (rand(s, 1, k), 1), (rand(s, 1, k), 1), (rand(d), 0), (rand(d), 0)])


def test_a_repeated_call_checks_its_operands_again():
    """A call object takes the short way only for operands like the last ones."""
    case = Case("conv", [8, 8], 16)
    call = case.call(pd.cuda_call_jit)
    x, weight, bias = [device(a) for a in case.operands()]
    first = call(x, weight, bias)
    assert torch.equal(call(x, weight, bias), first)
    with pytest.raises(DispatchError, match="does not match the traced float32"):
        call(x.half(), weight, bias)
    with pytest.raises(DispatchError, match="contiguous"):
        call(torch.empty(2, 16, 8, device="cuda").transpose(1, 2), weight, bias)
    with pytest.raises(DispatchError, match="expected a CUDA tensor"):
        call(x.cpu(), weight, bias)
    with pytest.raises(pd.TraceError, match="shape"):
        call(x[:1].contiguous(), weight, bias)
    host = call(*case.operands())
    assert np.array_equal(host, first.cpu().numpy())
    assert torch.equal(call(x + 0, weight, bias), first)


def test_calls_from_several_threads():
    import threading

    case = Case("scan", [200, 200], 40, gate=True, dtype="bfloat16")
    call = case.call(pd.cuda_call_jit)
    operands = [device(a) for a in case.operands()]
    want, got = call(*operands), {}
    torch.cuda.synchronize()

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            outs = [call(*operands) for _ in range(20)]
        stream.synchronize()
        got[i] = all(torch.equal(o, want) for o in outs)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got == {i: True for i in range(4)}


@pytest.mark.parametrize("dtype", TYPES)
def test_a_layer_over_a_prompt_in_parts_and_then_token_by_token(dtype):
    """Convolution, then scan: 100 tokens at once equal 60 tokens, a packed chunk of 37, then 3 single ones."""
    torch.manual_seed(5)
    t = getattr(torch, dtype)
    s, n, d, k = 2, 100, 48, 16
    x, delta, z = (torch.randn(s, n, d, device="cuda").to(t) for _ in range(3))
    B, C = (torch.randn(s, n, 1, k, device="cuda").to(t) for _ in range(2))
    weight, cbias = torch.randn(d, 4, device="cuda") * 0.5, torch.randn(d, device="cuda") * 0.1
    A = -torch.arange(1, k + 1, device="cuda", dtype=torch.float32).expand(d, k).contiguous()
    bias, skip = torch.full((d,), -3.0, device="cuda"), torch.ones(d, device="cuda")

    def layer(x, delta, B, C, z, edge, h, offsets=()):
        packed = bool(offsets)
        length = x.shape[0] if packed else x.shape[1]
        conv = families.causal_conv(length, initial=True, final=True, packed=packed, dtype=dtype)
        scan = families.selective_scan(length, k, gate=True, initial=True, final=True, packed=packed, dtype=dtype)
        make = lambda f: pd.cuda_call_jit(f, grid=(s, d), out_shape=families.out_shapes(f, (s, d)), math_mode="safe")  # noqa: E731
        u, edge = make(conv)(x, weight, cbias, edge, *offsets)
        y, h = make(scan)(u, delta, A, B, C, bias, skip, z, h, *offsets)
        return y, edge, h

    zeros = torch.zeros(s, 3, d, device="cuda", dtype=t), torch.zeros(s, d, k, device="cuda")
    whole, edge_all, h_all = layer(x, delta, B, C, z, *zeros)
    part = lambda a, b: [v[:, a:b].contiguous() for v in (x, delta, B, C, z)]  # noqa: E731
    y1, edge, h = layer(*part(0, 60), *zeros)
    flat = [v.reshape((s * 37,) + v.shape[2:]) for v in part(60, 97)]
    y2, edge, h = layer(*flat, edge, h, [torch.tensor([0, 37, 74], dtype=torch.int32, device="cuda")])
    ys = [y1, y2.reshape(s, 37, d)]
    conv = families.causal_conv_step(dtype=dtype)
    scan = families.selective_scan_step(k, gate=True, dtype=dtype)
    conv, scan = (pd.cuda_call_jit(f, grid=(s, d), out_shape=families.out_shapes(f, (s, d)), math_mode="safe") for f in (conv, scan))
    for i in range(97, 100):
        xi, di, bi, ci, zi = (v[:, 0].contiguous() for v in part(i, i + 1))
        u, edge = conv(xi, edge, weight, cbias)
        y, h = scan(h, u, di, A, bi, ci, bias, skip, zi)
        ys.append(y[:, None])
    assert torch.equal(edge, edge_all)
    # A state is at most 100 roundings of each of its contributions off, and a contribution here is below 50:
    # 100 * 2^-24 * 50 = 3e-4 on a state, 16 states on an output of size up to 1e3; stored values differ by
    # a step of their type besides, once where the convolution's output is stored and once at the end.
    step = {"float32": 2.0 ** -23, "float16": 2.0 ** -10, "bfloat16": 2.0 ** -7}[dtype]
    got = torch.cat(ys, 1).double()
    size = whole.double().abs().max()
    assert ((got - whole.double()).abs() <= step * (whole.double().abs() + size * 2 ** -4) + 2e-3).all()
    assert ((h - h_all).abs() <= 3e-4 + step * h_all.abs().max()).all()


# ------------------------------------------------------------------ host arrays
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("maker", [pd.cuda_call, pd.cuda_call_jit])
@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_host_arrays(kind, maker, dtype):
    case = Case(kind, [33, 33], 20, dtype=dtype, initial=True, final=True)
    got = case.call(maker)(*case.operands())
    check(case, ["y", "final"], got, case.oracle(grad=False))
    if kind == "conv":
        check(case, case.grad_names(), case.call(maker, "_grad")(*case.operands(grad=True)))


def test_pending_and_pinned_calls():
    case = Case("conv", [33, 33], 20, dtype="bfloat16")
    call = case.call(pd.cuda_call)
    first = call(*case.operands())
    pending = [call.launch(*case.operands()) for _ in range(4)]
    again = call.pin(*case.operands())
    for y in [p.wait() for p in pending] + [again(), again()]:
        assert np.array_equal(y.view(np.uint16), first.view(np.uint16))


# ------------------------------------------------------------------ what is not a sequence's own
def test_values_of_other_sequences_and_free_rows_are_not_read():
    for kind, more in (("conv", {}), ("scan", dict(gate=True))):
        case = Case(kind, [7, 3, 70], 20, packed=True, lead=2, spare=5, initial=True, final=True, **more)
        want = case.oracle()
        for name in ("x", "dy", "delta", "B", "C", "z"):
            if name in case.v:
                for rows in (slice(0, 2), slice(9, 12), slice(82, 87)):   # the free rows and the second sequence
                    case.v[name][rows] = np.nan if name in ("x", "z") else np.inf
        forward, grads = run(case)
        mine = np.r_[2:9, 12:82]
        y = wide(forward[0])
        off = np.abs(y[mine] - want["y"].value[mine])
        assert (off <= 1e-4 + 1e-4 * np.abs(want["y"].value[mine])).all()
        assert not np.isfinite(y[9:12]).any() and (y[:2] == 0).all() and (y[82:] == 0).all()
        dx = wide(grads[0])
        assert np.isfinite(dx[mine]).all() and (dx[:2] == 0).all() and (dx[82:] == 0).all()
        final = wide(forward[1])
        assert np.isfinite(final[[0, 2]]).all()


def test_offsets_outside_the_rows_are_clamped():
    for kind in ("conv", "scan"):
        case = Case(kind, [10, 20], 16, packed=True, initial=True, final=True)
        want = case.oracle()
        operands = [device(a) for a in case.operands()]
        operands[-1] = torch.tensor([-7, 10, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
        check(case, case.forward_names(), results(case.call(pd.cuda_call_jit)(*operands)), want)
        operands[-1] = torch.tensor([25, 10, 10], dtype=torch.int32, device="cuda")   # decreasing: both empty
        y, final = case.call(pd.cuda_call_jit)(*operands)
        assert torch.equal(final.cpu(), device(case.typed("initial")).cpu())


def test_empty_calls():
    for kind in ("conv", "scan"):
        for lengths, packed in (([0, 0], False), ([], False), ([0, 0], True), ([], True)):
            case = Case(kind, lengths, 6, packed=packed, initial=True, final=True)
            forward, grads = run(case)
            assert forward[0].size == 0 and np.array_equal(forward[1], case.v["initial"].astype(np.float32))
            named = dict(zip(case.grad_names(), grads))
            assert np.array_equal(named["dinitial"], case.v["dfinal"].astype(np.float32))
            assert all((named[n] == 0).all() for n in ("dweight", "dA", "dbias", "dskip") if n in named)


def test_extreme_step_sizes_and_rates():
    """Decays that underflow to zero, that are exactly one, and an infinite rate: the formula's own values."""
    case = Case("scan", [70], 8, state=16, softplus=False, bias=False, skip=False, final=True)
    case.v["delta"][:, 0] = 0.0
    case.v["delta"][:, 1] = 1e4
    case.v["A"][2] = 0.0
    case.v["A"][3] = -1e30
    compare(case)
    case.v["A"][4] = -np.inf
    case.v["delta"] = np.abs(case.v["delta"]) + 2.0 ** -10
    operands = [device(a) for a in case.operands()]
    y, final = case.call(pd.cuda_call_jit)(*operands)
    assert torch.isfinite(y).all() and torch.isfinite(final).all()


# ------------------------------------------------------------------ memory, streams, graphs
@pytest.mark.parametrize("kind", ["conv", "scan"])
@pytest.mark.parametrize("dtype", TYPES)
def test_operands_off_a_16_byte_boundary(kind, dtype):
    case = Case(kind, [30, 30], 16, dtype=dtype, initial=True, final=True, **({} if kind == "conv" else dict(gate=True)))
    want = case.oracle()

    def shifted(t):
        step = 4 // t.element_size()
        room = torch.empty(t.numel() + step, dtype=t.dtype, device="cuda")
        room[step:] = t.reshape(-1)
        return room[step:].view(t.shape)

    call = case.call(pd.cuda_call_jit)
    operands = [device(a) for a in case.operands()]
    outs = call(*operands)
    for move in range(len(operands)):
        moved = [shifted(t) if i == move else t for i, t in enumerate(operands)]
        check(case, case.forward_names(), results(call(*moved)), want)
    check(case, case.forward_names(), results(tuple(call.on_device(*operands, out=[shifted(o) for o in outs]))), want)


def test_strided_and_host_tensors_are_refused():
    case = Case("conv", [8, 8], 16)
    call = case.call(pd.cuda_call_jit)
    x, weight, bias = [device(a) for a in case.operands()]
    with pytest.raises(DispatchError, match="contiguous"):
        call(torch.empty(2, 16, 8, device="cuda").transpose(1, 2), weight, bias)
    with pytest.raises(DispatchError, match="expected a CUDA tensor"):
        call(x, weight.cpu(), bias)
    with pytest.raises(DispatchError, match="does not match the traced float32"):
        call(x.half(), weight, bias)


def test_results_over_operands_are_refused():
    case = Case("conv", [8, 8], 16)
    call = case.call(pd.cuda_call_jit)
    x, weight, bias = [device(a) for a in case.operands()]
    with pytest.raises(DispatchError, match="output 0 shares memory with input 0"):
        call.on_device(x, weight, bias, out=x)
    room = torch.empty(x.numel() + 16, device="cuda")
    room[16:] = x.reshape(-1)
    with pytest.raises(DispatchError, match="output 0 shares memory with input 0"):
        call.on_device(room[16:].view(x.shape), weight, bias, out=room[:-16].view(x.shape))
    step = families.causal_conv_step()
    call = pd.cuda_call_jit(step, grid=(2, 16), out_shape=families.out_shapes(step, (2, 16)))
    token, state = torch.randn(2, 16, device="cuda"), torch.randn(2, 3, 16, device="cuda")
    with pytest.raises(DispatchError, match="output 1 shares memory with input 1"):
        moved = torch.randn(3 * 2 * 16 + 4, device="cuda")
        call.on_device(token, moved[4:].view(2, 3, 16), weight, bias, out=(torch.empty_like(token), moved[:-4].view(2, 3, 16)))
    call.on_device(token, state, weight, bias, out=(torch.empty_like(token), state))


@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_side_streams_and_equal_bits(kind):
    case = Case(kind, [300, 300], 72, dtype="bfloat16", **({} if kind == "conv" else dict(gate=True)))
    first = run(case)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        second = run(case)
    stream.synchronize()
    for a, b in zip(first[0] + first[1], second[0] + second[1]):
        assert a.tobytes() == b.tobytes()


def test_captured_training_steps_replay_on_new_inputs():
    """Two graphs of different sizes, replayed in turn, each with memory of its own."""
    made = []
    for length, channels in ((150, 24), (90, 40)):
        case = Case("scan", [length] * 2, channels, dtype="bfloat16", gate=True)
        x, *rest = [device(a) for a in case.operands()]
        dy = device(case.typed("dy"))
        forward, grad = case.call(pd.cuda_call_jit, carries=True), case.call(pd.cuda_call_jit, "_grad")

        def step(x=x, rest=rest, dy=dy, forward=forward, grad=grad):
            y, carries = forward(x, *rest)
            return (y,) + grad(dy, x, *rest, carries)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        made.append((graph, outs, step, x))
    for _ in range(2):
        for graph, outs, step, x in made:
            x.copy_(torch.randn_like(x.float()).to(x.dtype))
            graph.replay()
            for a, b in zip(outs, step()):
                assert torch.equal(a, b)


def test_capture_without_a_workspace_is_refused():
    from palladium_b200 import _native

    case = Case("conv", [40, 40], 16)
    call = case.call(pd.cuda_call_jit, "_grad")
    operands = [device(a) for a in case.operands(grad=True)]
    outs = call(*operands)
    spec, bound = next(iter(call._cache.values()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs[0].zero_()      # a capture that stays valid
        with pytest.raises(DispatchError, match="workspace of its own"):
            _native.launch(spec.family.family_id, spec.params, 2, spec.grid, None,
                           [(t.data_ptr(), t.numel() * t.element_size()) for t in operands],
                           [(t.data_ptr(), t.numel() * t.element_size()) for t in outs],
                           stream=torch.cuda.current_stream().cuda_stream)


def test_more_than_2_31_elements():
    """The last rows of an array whose element offsets pass 32 bits equal the same rows computed alone."""
    rows, d = (1 << 19) + 5, 4104
    torch.manual_seed(1)
    x = torch.empty(1, rows, d, dtype=torch.bfloat16, device="cuda")
    for i in range(0, rows, 1 << 16):
        x[:, i:i + (1 << 16)].normal_()
    weight, bias = torch.randn(d, 4, device="cuda"), torch.randn(d, device="cuda")

    def call(n, initial):
        f = families.causal_conv(n, initial=initial, dtype="bfloat16")
        return pd.cuda_call_jit(f, grid=(1, d), out_shape=families.out_shapes(f, (1, d)))

    y = call(rows, False)(x, weight, bias)
    tail = call(100, True)(x[:, -100:].contiguous(), weight, bias, x[:, -103:-100].contiguous())
    assert torch.equal(y[:, -100:], tail)
