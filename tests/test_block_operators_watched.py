"""The 4-bit Linear, the norms over the residual and the rotary positions under tracers, transforms, modes and derivatives, which a launch on raw pointers
would pass by: each sees an operator or gets an error, and nobody another result."""

import pytest
import torch
from torch.autograd import forward_ad


def _inputs(device, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *shape: torch.randn(shape, generator=g).to(device, dtype)
    codes = torch.randint(0, 256, (40, 48), generator=g, dtype=torch.uint8).to(device)
    zeros = torch.randint(0, 16, (3, 40), generator=g, dtype=torch.uint8).to(device)
    return {
        "linear_i4": (r(6, 96), codes, r(3, 40).abs(), zeros, r(40).float()),
        "norm_residual": (r(6, 40), r(6, 40), r(2, 40), r(40), r(40), r(40)),
        "rotary": (r(2, 3, 5, 32), r(2, 1, 5, 32), torch.arange(5).to(device), (0.5 ** torch.arange(8, dtype=torch.float64)).to(device)),
    }


def _calls():
    from samfast_amd import ops
    return {
        "linear_i4": lambda x, codes, scales, zeros, bias: ops.linear_i4(x, codes, scales, zeros, bias, group_size=32),
        "norm_residual": lambda x, residual, gate, a, b, c: ops.norm_residual(x, residual, gate=gate, post=(a, b, 1e-6), pre=(c, None, 1e-6), branch_scale=0.5),
        "rotary": lambda q, k, positions, frequencies: ops.rotary(q, k, positions, frequencies, interleaved=True, scale=1.25),
    }


NAMES = ("linear_i4", "norm_residual", "rotary")


def _equal(a, b):
    a, b = ([t] if isinstance(t, torch.Tensor) else list(t) for t in (a, b))
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("name", NAMES)
def test_tensors_without_memory_have_shapes(name):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode() as mode:
        args = [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device="cuda") for t in _inputs("cpu")[name]]
    with mode:
        got = _calls()[name](*args)
    shapes = {"linear_i4": [(6, 40)], "norm_residual": [(6, 40)] * 2, "rotary": [(2, 3, 5, 32), (2, 1, 5, 32)]}[name]
    got = [got] if name == "linear_i4" else got
    assert [tuple(t.shape) for t in got] == shapes and all(t.dtype == torch.bfloat16 and t.is_cuda for t in got)
    if name == "rotary":
        assert [t.stride() for t in got] == [(480, 32, 96, 1), (160, 32, 32, 1)]
    graph = make_fx(_calls()[name], tracing_mode="fake")
    with mode:
        assert f"samfast.{name}" in graph(*args).code


@pytest.mark.parametrize("name", NAMES)
def test_tangents_and_transforms_that_differentiate_are_refused(name, monkeypatch):
    from samfast_amd import ops
    monkeypatch.setattr(ops, "_require_gpu", lambda *args: None)  # (nothing is launched)
    call, args = _calls()[name], _inputs("cpu")[name]
    for at, t in enumerate(args):
        if t.dtype != torch.bfloat16:
            continue
        with forward_ad.dual_level():
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == at else a for i, a in enumerate(args)]
            with pytest.raises(RuntimeError, match="derivatives"):
                call(*dual)
        one = lambda a: call(*args[:at], a, *args[at + 1:])
        with pytest.raises(RuntimeError, match="derivatives"):
            torch.func.jvp(one, (t,), (torch.ones_like(t),))
        with pytest.raises(RuntimeError, match="derivatives"):
            torch.func.vjp(one, t)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_trace_replays_new_inputs(name):
    call, args, other = _calls()[name], _inputs("cuda")[name], _inputs("cuda", seed=1)[name]
    want, want_other = call(*args), call(*other)
    with torch.no_grad():
        traced = torch.jit.trace(call, args, check_trace=False)
    assert f"samfast::{name}" in str(traced.graph)
    assert _equal(traced(*args), want) and _equal(traced(*other), want_other)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_modes_see_the_operator(name):
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode
    call, args = _calls()[name], _inputs("cuda")[name]
    want = call(*args)
    seen = []

    class Dispatched(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    class Called(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for mode in (Dispatched, Called):
        seen.clear()
        with mode():
            got = call(*args)
        assert _equal(got, want) and any(f"samfast.{name}" in s for s in seen)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_tensors_that_are_more_than_their_memory(name):
    call, args = _calls()[name], _inputs("cuda")[name]
    want = call(*args)

    class Named(torch.Tensor):
        pass

    assert _equal(call(args[0].as_subclass(Named), *args[1:]), want)
    negative = call(torch._neg_view(args[0]), *args[1:])
    assert _equal(negative, call((-args[0]).contiguous(), *args[1:])) and not _equal(negative, want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_tangents_and_gradients_are_refused_on_the_gpu(name):
    call, args = _calls()[name], _inputs("cuda")[name]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="derivatives"):
            call(forward_ad.make_dual(args[0], torch.ones_like(args[0])), *args[1:])
        call(*args)  # nothing of it carries a tangent
    leaf = args[0].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="samfast"):
        call(leaf, *args[1:])
    with pytest.raises(RuntimeError, match="samfast"):
        torch.jit.trace(call, (leaf, *args[1:]), check_trace=False)
    with pytest.raises(RuntimeError, match="samfast"):
        getattr(torch.ops.samfast, name)(*_flat(name, leaf, args))
    with torch.no_grad():
        call(leaf, *args[1:])


def _flat(name, first, args):
    if name == "linear_i4":
        return (first, *args[1:], 32)
    if name == "rotary":
        return (first, *args[1:], True, 1.25)
    return (first, args[1], args[2], args[3], args[4], 1e-6, args[5], None, 1e-6, False, 0.5, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_compiled_calls(name):
    call, args, other = _calls()[name], _inputs("cuda")[name], _inputs("cuda", seed=1)[name]
    compiled = torch.compile(call, backend="eager")
    for a in (args, other):
        assert _equal(compiled(*a), call(*a))


@pytest.mark.gpu
def test_batches_by_a_transform():
    call = _calls()["linear_i4"]
    sets = [_inputs("cuda", seed=s)["linear_i4"] for s in range(2)]
    both = torch.vmap(call)(*(torch.stack(pair) for pair in zip(*sets)))
    assert all(torch.equal(both[i], call(*sets[i])) for i in range(2))


@pytest.mark.gpu
def test_outs_of_watched_calls():
    """Memory for the results is written as unwatched calls do, the inputs' own included."""
    from samfast_amd import ops
    from torch.utils._python_dispatch import TorchDispatchMode

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, residual, gate, a, b, c = _inputs("cuda")["norm_residual"]
    norm = lambda residual, out: ops.norm_residual(x, residual, gate=gate, post=(a, b, 1e-6), pre=(c, None, 1e-6), out=out)
    want = norm(residual, None)
    stream = residual.clone()
    with Mode():
        got = norm(stream, stream)
        with pytest.raises(RuntimeError, match="samfast"):
            norm(residual, stream[:3])
        with pytest.raises(RuntimeError, match="samfast"):
            norm(residual, stream.float())
    assert got[0] is stream and _equal(got, want)

    q, k, positions, frequencies = _inputs("cuda")["rotary"]
    want = ops.rotary(q, k, positions, frequencies)
    into = q.clone(), k.clone()
    with Mode():
        got = ops.rotary(*into, positions, frequencies, out=into)
        for bad in ((torch.empty_like(q),), (torch.empty_like(q), None), (torch.empty_like(k), torch.empty_like(k))):
            with pytest.raises(RuntimeError, match="samfast"):
                ops.rotary(q, k, positions, frequencies, out=bad)
        alone = ops.rotary(q, None, positions, frequencies)
    assert got[0] is into[0] and got[1] is into[1] and _equal(got, want)
    assert torch.equal(alone[0], want[0]) and alone[1] is None


@pytest.mark.gpu
def test_a_traced_module_with_a_4_bit_linear():
    """(Without a bias: torch.jit cannot trace the view of its bits as floats, and says so.)"""
    from samfast_amd import Int4Linear
    torch.manual_seed(0)
    module = Int4Linear.from_float(torch.nn.Linear(96, 40, bias=False).requires_grad_(False), 32, True).to("cuda", torch.bfloat16)
    x, other = (torch.randn((2, m, 96), device="cuda").bfloat16() for m in (5, 7))
    with torch.no_grad():
        traced = torch.jit.trace(module, (x,), check_trace=False)
    assert torch.equal(traced(x), module(x)) and torch.equal(traced(other), module(other))
