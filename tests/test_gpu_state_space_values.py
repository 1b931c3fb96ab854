"""Values of the state-space families where float32's range or a rounding decides, on a GPU against the float64
operators inside the bounds of their running error analysis."""

import re
from pathlib import Path

import numpy as np
import pytest
import torch

import palladium_b200 as pd
from palladium_b200 import families
from palladium_b200.pl import ShapeDtypeStruct
from tests.state_space import TYPES, Case, check, wide
from tests.test_gpu_state_space import back, compare, device, run

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


# ------------------------------------------------------------------ states that remember for long
def test_fast_decays_near_one_are_as_exact_as_safe_ones():
    """4096 tokens of float32 with decays around 1 - 1e-2: FAST's series is off by half a rounding of a value below one
    (2^-25) and a hundredth of what its argument is, SAFE's exponential by up to two, so the errors of what thousands of
    them make, against float64, may not be larger.  (Factor 1.5: both are sums of signed errors.)"""
    torch.manual_seed(2)
    s, n, d, k = 2, 4096, 32, 16
    step = 0.02 * torch.rand(s, n, d, device="cuda")
    A = -(0.5 + torch.rand(d, k, device="cuda"))
    x = torch.randn(s, n, d, device="cuda").abs()
    B, C = (torch.randn(s, n, 1, k, device="cuda").abs() for _ in range(2))
    h = torch.randn(s, d, k, device="cuda")
    plain = dict(softplus=False, bias=False, skip=False)
    want, ys = h.double(), []
    for t in range(n):
        at = step[:, t].double()
        want = torch.exp(at[..., None] * A.double()) * want + (at * x[:, t].double())[..., None] * B[:, t].double()
        ys.append((want * C[:, t].double()).sum(-1))
    want = {"y": torch.stack(ys, 1), "final": want, "stepped": want}

    def errors(math_mode):
        make = lambda f: pd.cuda_call_jit(f, grid=(s, d), out_shape=families.out_shapes(f, (s, d)), math_mode=math_mode)  # noqa: E731
        y, final = make(families.selective_scan(n, k, initial=True, final=True, **plain))(x, step, A, B, C, h)
        one, state = make(families.selective_scan_step(k, **plain)), h
        for t in range(n):
            _, state = one(state, *[v[:, t].contiguous() for v in (x, step)], A, *[v[:, t].contiguous() for v in (B, C)])
        got = {"y": y, "final": final, "stepped": state}
        return {name: float((got[name].double() - want[name]).norm() / want[name].norm()) for name in want}

    fast, safe = errors("fast"), errors("safe")
    for name in want:
        assert fast[name] <= 1.5 * safe[name], (name, fast, safe)


# ------------------------------------------------------------------ gradients of several channels per warp
# (sequences, channels) that are given one to six channels a warp; 128 staging threads divide into neither three, five nor six
SIZES = [(30, 63, 2), (50, 66, 3), (80, 63, 4), (50, 130, 5), (120, 63, 6)]


def _reached(case, items):
    carries = ShapeDtypeStruct(families.out_shapes(case.family(carries=True), case.grid)[-1].shape, np.float32)
    return case.call(pd.cuda_call, "_grad").explain(*case.operands(grad=True, carries=carries)).items_per_thread == items


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("state", [3, 8, 16])
@pytest.mark.parametrize("seqs, channels, items", SIZES)
@pytest.mark.parametrize("packed", [False, True])
def test_gradient_with_several_channels_per_warp(packed, seqs, channels, items, state, dtype):
    if packed:
        lengths = [(s * 7) % 13 for s in range(seqs)]       # empty ones and single tokens among them
        lengths[1], lengths[seqs // 2] = 33, 70             # and some of more than one chunk
    else:
        lengths = [9] * seqs
    case = Case("scan", lengths, channels, dtype=dtype, state=state, packed=packed, lead=2 * packed, spare=3 * packed,
                gate=packed, initial=packed, final=packed, seed=items)
    if not (dtype == "float32" and state == 16 and items > 4):      # (there shared memory has room for fewer)
        assert _reached(case, items)
    compare(case)


@pytest.mark.parametrize("dtype, state, seqs, channels, items", [
    ("bfloat16", 24, 50, 66, 3), ("float32", 24, 50, 66, 4), ("bfloat16", 64, 50, 66, 4), ("float32", 64, 30, 63, 2)])
def test_gradient_with_several_channels_per_warp_and_slices_of_states(dtype, state, seqs, channels, items):
    for more in (dict(), dict(gate=True, initial=True, final=True)):
        case = Case("scan", [5 if more else 34] * seqs, channels, dtype=dtype, state=state, **more)
        assert _reached(case, items)
        compare(case)


def test_gradient_with_several_channels_per_warp_and_groups():
    case = Case("scan", [40] * 30, 120, dtype="float32", state=11, groups=3, gate=True, initial=True, final=True)
    assert _reached(case, 3)
    compare(case)


# ------------------------------------------------------------------ packed buffers that are mostly free
@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("channels", [5, 24, 37, 160])
@pytest.mark.parametrize("lead, spare", [(0, 3000), (1, 777), (900, 1), (2500, 600)])
def test_rows_of_no_sequence_come_out_as_zeros(lead, spare, channels, dtype):
    for kind, more in (("conv", {}), ("scan", dict(state=4, gate=True))):
        case = Case(kind, [20, 0, 41], channels, dtype=dtype, packed=True, lead=lead, spare=spare, initial=True, final=True,
                    **more)
        compare(case)


def test_a_packed_call_takes_no_longer_for_rows_of_no_sequence_than_writing_them_does():
    """200 tokens in a buffer of 8192 rows against the same in one of 256: the zeros are 32 times as many, a fraction of
    the kernel's time (cleared row by row it was fifty times the small buffer's time)."""
    def best(rows):
        x, delta, dy = (torch.randn(rows, 2048, device="cuda").bfloat16() for _ in range(3))
        B, C = (torch.randn(rows, 1, 16, device="cuda").bfloat16() for _ in range(2))
        A, bias, skip = -torch.rand(2048, 16, device="cuda"), torch.randn(2048, device="cuda"), torch.randn(2048, device="cuda")
        offsets = torch.tensor([0, 50, 100, 150, 200], dtype=torch.int32, device="cuda")
        make = lambda f: pd.cuda_call_jit(f, grid=(4, 2048), out_shape=families.out_shapes(f, (4, 2048)))  # noqa: E731
        forward = make(families.selective_scan(rows, packed=True, carries=True, dtype="bfloat16"))
        grad = make(families.selective_scan_grad(rows, packed=True, dtype="bfloat16"))
        operands = (x, delta, A, B, C, bias, skip)
        carries = forward(*operands, offsets)[1]
        times = []
        for call in (lambda: forward(*operands, offsets), lambda: grad(dy, *operands, carries, offsets)):
            took = []
            for _ in range(8):
                start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                start.record()
                call()
                end.record()
                torch.cuda.synchronize()
                took.append(start.elapsed_time(end))
            times.append(min(took))
        return times

    small, large = best(256), best(8192)
    assert large[0] < 12 * small[0] and large[1] < 8 * small[1], (small, large)


# ------------------------------------------------------------------ calls at once
def test_gradients_of_different_block_sizes_from_several_threads():
    """One kernel with two to six channels a warp, so with different amounts of shared memory, launched by six threads at
    once: no call takes another one's leave for shared memory away, and each gives its own result."""
    import threading

    made = []
    for seqs, channels in ((30, 63), (50, 66), (80, 63), (50, 130), (120, 63), (2, 8)):
        case = Case("scan", [40] * seqs, channels, dtype="bfloat16", state=16, gate=True)
        *_, carries = case.call(pd.cuda_call_jit, carries=True)(*[device(a) for a in case.operands()])
        operands = [device(a) for a in case.operands(grad=True, carries=back(carries))]
        call = case.call(pd.cuda_call_jit, "_grad")
        made.append((call, operands, call(*operands)))
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(made))

    def work(i):
        call, operands, want = made[i]
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(200):
                    got = call(*operands)
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append((i, "other bits"))
        except Exception as e:
            wrong.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(made))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------ memory of gradients and steps
def shifted(tensor):
    """The same values four bytes off a 16-byte boundary."""
    step = 4 // tensor.element_size()
    room = torch.empty(tensor.numel() + step, dtype=tensor.dtype, device="cuda")
    room[step:] = tensor.reshape(-1)
    return room[step:].view(tensor.shape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_gradients_off_a_16_byte_boundary(kind, dtype):
    more = {} if kind == "conv" else dict(state=16, gate=True)
    case = Case(kind, [9] * 50, 68, dtype=dtype, initial=True, final=True, **more)
    carries = None
    if kind == "scan":
        carries = back(case.call(pd.cuda_call_jit, carries=True)(*[device(a) for a in case.operands()])[-1])
        assert _reached(case, 3)
    operands = [device(a) for a in case.operands(grad=True, carries=carries)]
    call, want = case.call(pd.cuda_call_jit, "_grad"), case.oracle()
    outs = call(*operands)
    for move in range(len(operands)):
        moved = [shifted(t) if i == move else t for i, t in enumerate(operands)]
        check(case, case.grad_names(), [back(t) for t in call(*moved)], want)
    got = call.on_device(*operands, out=[shifted(o) for o in outs])
    check(case, case.grad_names(), [back(t) for t in got], want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_steps_off_a_16_byte_boundary(kind, dtype):
    if kind == "conv":
        family, order = families.causal_conv_step(dtype=dtype), ["x", "initial", "weight", "bias"]
        case = Case("conv", [1] * 20, 16, dtype=dtype, initial=True, final=True)
    else:
        family = families.selective_scan_step(16, groups=2, gate=True, dtype=dtype)
        order = ["initial", "x", "delta", "A", "B", "C", "bias", "skip", "z"]
        case = Case("scan", [1] * 20, 16, dtype=dtype, state=16, groups=2, gate=True, initial=True, final=True)
    call = pd.cuda_call_jit(family, grid=case.grid, out_shape=families.out_shapes(family, case.grid))
    operands = [device(case.typed(n)) for n in order]
    operands = [t.reshape(t.shape[:1] + t.shape[2:]) if n in ("x", "delta", "B", "C", "z") else t for n, t in zip(order, operands)]
    want = case.oracle(grad=False)
    outs = call(*operands)
    for move in range(len(operands)):
        moved = [shifted(t) if i == move else t for i, t in enumerate(operands)]
        check(case, ["y", "final"], [back(t) for t in call(*moved)], want)
    check(case, ["y", "final"], [back(t) for t in call.on_device(*operands, out=[shifted(o) for o in outs])], want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("maker", [pd.cuda_call, pd.cuda_call_jit])
@pytest.mark.parametrize("packed", [False, True])
def test_scan_gradients_on_host_arrays(maker, dtype, packed):
    lengths = [40, 40] if not packed else [40, 0, 33]
    case = Case("scan", lengths, 20, dtype=dtype, packed=packed, gate=True, initial=True, final=True)
    *forward, carries = case.call(maker, carries=True)(*case.operands())
    want = case.oracle()
    check(case, case.forward_names(), forward, want)
    check(case, case.grad_names(), case.call(maker, "_grad")(*case.operands(grad=True, carries=carries)), want)


# ------------------------------------------------------------------ through torch.autograd
def test_the_readme_connects_the_scan_to_autograd():
    """The README's lines as they stand, in bfloat16: gradients of every operand against differentiating the formula in
    float64, a layer's input used once more beside the scan; and a backward pass whose incoming gradient is expanded."""
    text = (Path(__file__).resolve().parent.parent / "README.md").read_text()
    code = next(b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "class SelectiveScan" in b)
    case = Case("scan", [50, 50], 24, dtype="bfloat16", state=16, gate=True, seed=4)
    names = ["u", "delta", "A", "B", "C", "delta_bias", "skip", "z"]
    operands = [device(a).requires_grad_() for a in case.operands()]
    space = dict(torch=torch, pd=pd, families=families, batch=2, channels=24, length=50, **dict(zip(names, operands)))
    exec(code, space)
    y = space["y"]
    check(case, ["y"], [back(y.detach())])
    dy = device(case.typed("dy"))
    grads = torch.autograd.grad(y, operands, dy, retain_graph=True)
    check(case, case.grad_names(), [back(g) for g in grads])
    both = torch.autograd.grad(y + operands[0], operands[0], dy, retain_graph=True)[0]       # the sum of two paths, rounded once more
    assert torch.equal(both, (grads[0].float() + dy.float()).bfloat16())
    ones = torch.autograd.grad(y.sum(), operands)
    case.v["dy"][:] = 1.0
    check(case, case.grad_names(), [back(g) for g in ones])
    with torch.no_grad():
        assert not space["SelectiveScan"].apply(*operands).requires_grad
    assert not space["forward"](*operands)[0].requires_grad


# ------------------------------------------------------------------ results' memory
def test_results_of_another_type_are_refused():
    """float16 and bfloat16 are of one size: bits of one in a tensor of the other would be other numbers."""
    case = Case("scan", [9, 9], 16, dtype="bfloat16", final=True)
    call = case.call(pd.cuda_call_jit)
    operands = [device(a) for a in case.operands()]
    y, final = call(*operands)
    for wrong in ((y.view(torch.float16), final), (y.view(torch.int16), final), (y, final.view(torch.int32))):
        with pytest.raises(pd.DispatchError, match="does not match the .* that the call writes"):
            call.on_device(*operands, out=wrong)
    got = call.on_device(*operands, out=(torch.empty_like(y), torch.empty_like(final)))
    assert torch.equal(got[0], y) and torch.equal(got[1], final)


@pytest.mark.parametrize("kind", ["conv", "scan"])
def test_packed_calls_without_any_sequence(kind):
    """A buffer of free rows alone: zeros, and sums of nothing."""
    for lead, spare in ((0, 300), (7, 0), (100, 50)):
        case = Case(kind, [], 20, dtype="float16", packed=True, lead=lead, spare=spare, initial=True, final=True)
        forward, grads = run(case)
        assert (wide(forward[0]) == 0).all() and forward[0].shape == (lead + spare, 20) and forward[1].size == 0
        assert all((wide(g) == 0).all() for g in grads)


# ------------------------------------------------------------------ many segments
@pytest.mark.parametrize("lengths", [[9000], [8000, 3, 0, 200, 1]])
def test_sequences_of_many_segments(lengths):
    """Some forty segments, or a sequence that has nearly all the rows of a packed call: every state between them right."""
    packed = len(lengths) > 1
    case = Case("scan", lengths, 5, packed=packed, state=4, gate=True, initial=True, final=True)
    diag = case.call(pd.cuda_call).explain(*case.operands())
    assert diag.launches == 2 and diag.cuda_grid[0] > 40
    compare(case)
