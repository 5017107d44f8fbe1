"""The 4-bit weight quantiser, the module that holds it, and rotary frequencies, on the CPU."""

import math

import pytest
import torch


@pytest.mark.parametrize("N,K,group", [(3, 8, 32), (5, 96, 32), (4, 200, 64), (7, 256, 256), (2, 1000, 128)])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_codes_are_the_nearest_to_the_weights(N, K, group, zero_points, dtype):
    from samfast_amd import quant4
    g = torch.Generator().manual_seed(N + K)
    w = (torch.randn((N, K), generator=g) * 0.02 + 0.005).to(dtype)
    w[0, : min(group, K)] = 0
    codes, scales, zeros = quant4.quantize_weight_int4(w, group, zero_points)
    groups = -(-K // group)
    assert codes.shape == (N, K // 2) and codes.dtype == torch.uint8 and scales.shape == (groups, N)
    assert scales.dtype == (torch.bfloat16 if dtype == torch.float32 else dtype)
    assert (zeros is None) == (not zero_points)
    back = quant4.dequantize_weight_int4(codes, scales, zeros, group)
    step = scales.float().t()[:, torch.arange(K) // group]
    # half a step; a scale rounded down leaves the extreme value up to 7.5 (15 with zero points) roundings of it, 2^-8 each at most, outside, and
    # a zero point is off by half a step, which the clamp at an end then adds
    slack = (0.5 + 15 * 2.0 ** -8 + (0.5 if zero_points else 0.0)) * step
    assert ((back - w.float()).abs() <= slack + 1e-7).all()
    assert (back[0, : min(group, K)] == 0).all()
    # each even input in the lower half of its byte
    c = ((w.float()[-1, :2] / step[-1, :2]).round() + (8 if zeros is None else zeros[0, -1].float())).clamp(0, 15)
    assert int(codes[-1, 0]) == int(c[0]) + 16 * int(c[1])


def test_the_quantiser_refuses():
    from samfast_amd import quant4
    for weight, group in [(torch.zeros(4, 12), 32), (torch.zeros(4, 16), 48), (torch.zeros(4, 16), 0), (torch.zeros(16), 32), (torch.zeros(4, 16, dtype=torch.int8), 32), (torch.zeros(0, 16), 32)]:
        with pytest.raises(ValueError):
            quant4.quantize_weight_int4(weight, group)


def test_module_state_and_swap():
    from samfast_amd import Int4Linear, apply_int4_weights
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(64, 40), torch.nn.Sequential(torch.nn.ReLU(), torch.nn.Linear(40, 24, bias=False)), torch.nn.Linear(24, 8))
    bias, weight = model[0].bias.detach().clone(), model[0].weight.detach().clone()
    apply_int4_weights(model, filter_fn=lambda m, fqn: fqn != "2", group_size=32, zero_points=True)
    assert isinstance(model[0], Int4Linear) and isinstance(model[1][1], Int4Linear) and type(model[2]) is torch.nn.Linear
    assert model[1][1].bias is None and "groups of 32" in repr(model[0])
    model.to(torch.float16)
    assert torch.equal(model[0].bias, bias) and model[0].scales.dtype == torch.float16 and model[0].codes.dtype == torch.uint8
    assert (model[0].weight - weight).abs().max() < 0.05 * weight.abs().max() + 0.02
    other = torch.nn.Sequential(torch.nn.Linear(64, 40), torch.nn.Sequential(torch.nn.ReLU(), torch.nn.Linear(40, 24, bias=False)), torch.nn.Linear(24, 8))
    apply_int4_weights(other, filter_fn=lambda m, fqn: fqn != "2", group_size=32, zero_points=True)
    other.to(torch.float16).load_state_dict(model.state_dict())
    assert torch.equal(other[0].weight, model[0].weight) and torch.equal(other[0].bias, bias)
    state = {k: v for k, v in model[0].state_dict().items() if k != "bias_bits"}
    other[0].load_state_dict({**state, "bias": bias + 1})
    assert torch.equal(other[0].bias, bias + 1)
    with pytest.raises(RuntimeError, match="samfast"):
        model[0](torch.zeros(2, 64, dtype=torch.float16))  # no CPU route


def test_frequencies_and_grid():
    from samfast_amd import grid_positions, rotary_frequencies
    f = rotary_frequencies(64)
    assert f.dtype == torch.float64 and f[0] == 1 and abs(float(f[32]) - 0.01) < 1e-15
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=8.0), f / 8)
    b = rotary_frequencies(64, scaling="bands", factor=8.0, trained_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(b[turns >= 32], f[turns >= 32]) and torch.allclose(b[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (b[between] < f[between]).all() and (b[between] > f[between] / 8).all() and (b[1:] < b[:-1]).all()
    for bad in (dict(pairs=0), dict(pairs=4, scaling="ntk"), dict(pairs=4, factor=0.0), dict(pairs=4, slow_turns=32.0), dict(pairs=4, base=-1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)
    assert grid_positions(2, 3).tolist() == [[0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]


def test_a_model_is_swapped_whole_or_not_at_all():
    from samfast_amd import Int4Linear, apply_int4_weights
    model = torch.nn.Sequential(torch.nn.Linear(64, 12), torch.nn.ReLU(), torch.nn.Linear(12, 8))
    with pytest.raises(ValueError, match="2: "):
        apply_int4_weights(model)
    with pytest.raises(ValueError):
        apply_int4_weights(model, lambda mod, fqn: fqn == "0", group_size=48)
    assert [type(m) for m in model] == [torch.nn.Linear, torch.nn.ReLU, torch.nn.Linear]
    apply_int4_weights(model, lambda mod, fqn: fqn == "0")
    assert isinstance(model[0], Int4Linear) and isinstance(model[2], torch.nn.Linear)


def test_a_bias_that_the_module_does_not_have_is_not_dropped_silently():
    from samfast_amd import Int4Linear
    linear = torch.nn.Linear(64, 40).requires_grad_(False)
    without = Int4Linear.from_float(torch.nn.Linear(64, 40, bias=False).requires_grad_(False), 32)
    model = torch.nn.Sequential(without)
    state = {**model.state_dict(), "0.bias": linear.bias}
    with pytest.raises(RuntimeError, match="0.bias"):
        model.load_state_dict(state)
    assert model.load_state_dict(state, strict=False).unexpected_keys == ["0.bias"] and without.bias is None and "0.bias" in state
    # one that it has is folded, and not counted as one too many
    model = torch.nn.Sequential(Int4Linear.from_float(linear, 32))
    state = {k: v for k, v in model.state_dict().items() if k != "0.bias_bits"}
    result = model.load_state_dict({**state, "0.bias": linear.bias + 2})
    assert not result.unexpected_keys and not result.missing_keys and torch.equal(model[0].bias, linear.bias + 2)


@pytest.mark.parametrize("kind", ["Int4Linear", "Int8DynamicLinear"])
def test_modules_of_one_linear_have_biases_of_their_own(kind):
    """What is loaded into one of them reaches neither the other nor the Linear."""
    import samfast_amd
    make = getattr(samfast_amd, kind).from_float
    linear = torch.nn.Linear(64, 40).requires_grad_(False)
    kept = linear.bias.clone()
    one, other = make(linear), make(linear)
    one.load_state_dict({**one.state_dict(), "bias_bits": (kept + 1).view(torch.int32)})
    assert torch.equal(one.bias, kept + 1) and torch.equal(other.bias, kept) and torch.equal(linear.bias, kept)
    linear.bias += 3
    assert torch.equal(one.bias, kept + 1) and torch.equal(other.bias, kept)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_casts_to_wider_types_keep_the_scales(dtype):
    """The kernels have half types only; a model in fp32 (or fp64) goes on calling them."""
    from samfast_amd import Int4Linear
    torch.manual_seed(1)
    module = Int4Linear.from_float(torch.nn.Linear(64, 40).to(dtype).requires_grad_(False), 32, True)
    scales, bias, weight = module.scales.clone(), module.bias.clone(), module.weight.clone()
    model = torch.nn.Sequential(module, torch.nn.Linear(40, 8))
    for cast in (model.float, model.double, lambda: model.to(torch.float32)):
        cast()
        assert model[1].weight.dtype != dtype
        assert module.scales.dtype == dtype and torch.equal(module.scales, scales) and torch.equal(module.bias, bias) and torch.equal(module.weight, weight)
        assert dict(module.named_buffers())["scales"] is module.scales


def test_a_cast_that_loses_scales_warns(recwarn):
    from samfast_amd import Int4Linear
    linear = torch.nn.Linear(64, 4).to(torch.bfloat16).requires_grad_(False)
    Int4Linear.from_float(linear, 32).half()
    assert not recwarn.list
    for size in (1e-9, 1e7):
        linear.weight[1] = size
        with pytest.warns(UserWarning, match="2 scales"):
            Int4Linear.from_float(linear, 32).half()


def test_a_linear_of_two_names_is_looked_at_under_each():
    from samfast_amd import apply_int4_weights
    shared = torch.nn.Linear(12, 64)
    model = torch.nn.ModuleDict({"a": shared, "b": torch.nn.Linear(64, 12), "c": shared, "d": torch.nn.Linear(8, 8)})
    with pytest.raises(ValueError, match="c: "):
        apply_int4_weights(model, lambda mod, fqn: fqn in "bc")
    assert all(type(m) is torch.nn.Linear for m in model.values())
    model["d"].weight = torch.nn.Parameter(torch.zeros(8, 8, dtype=torch.complex64))
    with pytest.raises(ValueError, match="d: "):
        apply_int4_weights(model, lambda mod, fqn: fqn in "bd")
    assert all(type(m) is torch.nn.Linear for m in model.values())
