"""Rotary positions, against the formula in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _turned(t, positions, frequencies, interleaved, scale):
    """(B, H, T, D) turned by the formula, in 64 bits, as products of complex numbers."""
    out = t.double().clone()
    freq = frequencies.view(1, -1) if frequencies.dim() == 1 else frequencies
    axes, pairs = freq.shape
    pos = positions.double().reshape(*positions.shape[:positions.dim() - (frequencies.dim() - 1)], axes)
    pos = pos.expand(t.shape[0], *pos.shape) if pos.dim() == 2 else pos
    for axis in range(axes):
        angle = pos[..., axis, None] * freq[axis]                       # (B, T, pairs)
        turn = torch.polar(torch.full_like(angle, scale), angle)[:, None]
        part = out[..., 2 * axis * pairs:2 * (axis + 1) * pairs]
        a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.split(pairs, -1)
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        a.copy_(z.real)
        b.copy_(z.imag)
    return out


def _check(got, t, positions, frequencies, interleaved, scale):
    ref = _turned(t, positions, frequencies, interleaved, scale)
    # one rounding to the type; the angle's turns are a product of 53 bits below 2^27 and 24 bits of a fraction, its sine and cosine fp32 values
    # to 4 units: 2^-21 of the pair's length
    length = scale * t.double().abs().amax(-1, keepdim=True) * 2 ** 0.5
    half = torch.finfo(t.dtype).eps / 2
    assert got.shape == t.shape and got.dtype == t.dtype
    assert ((got.double() - ref).abs() <= half * ref.abs() + (2.0 ** -21 + 2.0 ** -23) * length + 2.0 ** -25).all()


def _qk(B, H, KV, T, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + B + 7 * T + 3 * D)
    fused = torch.randn((B, T, H + 2 * KV, D), generator=g, device="cuda").to(dtype)
    return fused[:, :, :H].permute(0, 2, 1, 3), fused[:, :, H:H + KV].permute(0, 2, 1, 3), fused


def _frequencies(pairs, axes, base=10000.0):
    f = base ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
    return f if axes == 1 else torch.stack([f * (1 + 0.1 * a) for a in range(axes)])


@pytest.mark.parametrize("B,H,KV,T,D,pairs,axes", [
    (1, 1, 1, 1, 2, 1, 1), (1, 1, 1, 5, 3, 1, 1), (2, 3, 1, 7, 8, 4, 1), (8, 32, 8, 1, 128, 64, 1), (1, 4, 2, 33, 80, 20, 2), (3, 2, 2, 50, 96, 32, 1),
    (2, 5, 1, 17, 34, 17, 1), (2, 5, 3, 19, 66, 15, 2), (1, 16, 16, 300, 64, 32, 1), (1, 2, 1, 9, 1024, 512, 1), (5, 1, 1, 3, 50, 4, 3),
    (70, 2, 1, 1, 64, 16, 1), (1, 300, 7, 2, 72, 31, 1), (2, 24, 4, 3001, 96, 32, 1), (1, 3, 2, 11, 256, 128, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rotary(B, H, KV, T, D, pairs, axes, interleaved, dtype):
    from samfast_amd import ops
    print(f"case rotary B={B} H={H},{KV} T={T} D={D} pairs={pairs} axes={axes} interleaved={interleaved} {dtype}", flush=True)
    q, k, fused = _qk(B, H, KV, T, D, dtype)
    kept = fused.clone()
    g = torch.Generator(device="cuda").manual_seed(T)
    freq = _frequencies(pairs, axes)
    for far, scale, shared in ((100, 1.0, True), (1 << 20, 1.2079, False)):
        shape = ((T,) if shared else (B, T)) + ((axes,) if axes > 1 else ())
        positions = torch.randint(-far, far, shape, generator=g, device="cuda")
        got = ops.rotary(q, k, positions, freq, interleaved=interleaved, scale=scale)
        assert torch.equal(fused, kept)
        for o, t in zip(got, (q, k)):
            _check(o, t, positions, freq, interleaved, scale)
            assert torch.equal(o[..., 2 * axes * pairs:], t[..., 2 * axes * pairs:])
    if axes == 1:  # one axis written as such
        again = ops.rotary(q, k, positions.unsqueeze(-1), freq.view(1, -1), interleaved=interleaved, scale=scale)
        assert all(torch.equal(a, b) for a, b in zip(again, got))


def test_in_place_and_layouts():
    from samfast_amd import ops
    q, k, fused = _qk(2, 6, 2, 21, 80, torch.bfloat16)
    positions, freq = torch.arange(21, device="cuda") + 1000, _frequencies(30, 1)
    want = ops.rotary(q, k, positions, freq)
    assert want[0].permute(0, 2, 1, 3).is_contiguous()
    alone, none = ops.rotary(q, None, positions, freq)
    assert none is None and torch.equal(alone, want[0])
    heads_first = ops.rotary(q.contiguous(), k.contiguous(), positions, freq)
    assert all(torch.equal(a, b) for a, b in zip(heads_first, want))
    odd = torch.full((2, 6, 21, 83), float("nan"), dtype=q.dtype, device="cuda")
    odd[..., 1:81] = q
    assert torch.equal(ops.rotary(odd[..., 1:81], k, positions, freq)[0], want[0])
    values = fused[:, :, 8:].clone()
    got = ops.rotary(q, k, positions, freq, out=(q, k))
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, :, 8:], values)
    for empty in (q[:0], q[:, :0], q[:, :, :0]):
        p = positions[:empty.shape[2]]
        assert ops.rotary(empty, None, p, freq)[0].shape == empty.shape


@pytest.mark.parametrize("D,pairs,axes", [(6, 3, 1), (18, 9, 1), (66, 17, 1), (70, 11, 2), (84, 41, 1), (250, 102, 1), (45, 9, 2), (96, 13, 3), (30, 4, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_at_odd_widths(D, pairs, axes, interleaved):
    """Threads that share channels of a head read them before one of them writes."""
    from samfast_amd import ops
    q, k, _ = _qk(3, 7, 2, 211, D, torch.bfloat16)
    q, k = q.contiguous(), k.contiguous()
    positions = torch.arange(211 * axes, device="cuda").view(211, axes) * 3
    freq = _frequencies(pairs, axes).view(axes, pairs)
    want = ops.rotary(q, k, positions, freq, interleaved=interleaved)
    for t, w in zip((q, k), want):
        _check(w, t, positions, freq, interleaved, 1.0)
    ops.rotary(q, k, positions, freq, interleaved=interleaved, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_position_zero_and_whole_turns_change_nothing():
    from samfast_amd import ops
    q, k, _ = _qk(1, 2, 1, 4, 64, torch.float16)
    zero = ops.rotary(q, k, torch.zeros(4, dtype=torch.int64, device="cuda"), _frequencies(32, 1))
    assert torch.equal(zero[0], q) and torch.equal(zero[1], k)


def test_far_positions_keep_their_angle():
    """Relative positions alone count: q at p + d against k at p gives the product of q at d against k at 0, however far p is."""
    from samfast_amd import ops
    q, k, _ = _qk(1, 1, 1, 1, 128, torch.float16)
    freq = _frequencies(64, 1)
    at = lambda t, p: ops.rotary(t, None, torch.tensor([p], device="cuda"), freq)[0].double()
    want = (at(q, 5) * at(k, 0)).sum()
    for p in (10 ** 3, 10 ** 6, 10 ** 8):
        got = (at(q, p + 5) * at(k, p)).sum()
        # each factor is rounded to fp16 (2^-11 of it), and its angle to 2^-21: of at most sum |q'| |k'| <= |q| |k|
        assert abs(float(got - want)) <= (4 * 2.0 ** -11 + 2.0 ** -18) * float(q.double().norm() * k.double().norm())


def test_refusals():
    from samfast_amd import ops
    q, k, _ = _qk(2, 4, 2, 6, 64, torch.bfloat16)
    positions, freq = torch.arange(6, device="cuda"), _frequencies(32, 1)
    cases = [
        dict(q=q.float(), k=k.float()), dict(k=k.half()), dict(k=k[:, :, :5]), dict(k=k[:1]), dict(k=k[..., :32]), dict(q=q[0]), dict(positions=positions.int()),
        dict(positions=positions[:5]), dict(positions=positions.expand(3, 6)), dict(frequencies=freq.float()), dict(frequencies=_frequencies(33, 1)),
        dict(frequencies=freq[:0]), dict(frequencies=freq[::2]), dict(frequencies=_frequencies(16, 2)), dict(frequencies=_frequencies(17, 2), positions=positions.view(6, 1).expand(6, 2)),
        dict(q=q.transpose(2, 3), k=None), dict(out=(q[:, :3], k)), dict(out=(q, None)), dict(out=(q.half(), k)),
        dict(q=q.cpu()), dict(positions=positions.cpu()), dict(q=q.clone().requires_grad_()),
    ]
    for case in cases:
        args = dict(dict(q=q, k=k, positions=positions, frequencies=freq), **case)
        with pytest.raises(RuntimeError, match="samfast"):
            ops.rotary(**args)
    big = torch.zeros((1, 1, 1, 1026), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="samfast"):
        ops.rotary(big, None, positions[:1], freq)
    assert math.isfinite(float(q.float().sum()))


@pytest.mark.parametrize("D,pairs,axes", [(1024, 8, 64), (128, 1, 64), (1024, 1, 64), (1000, 7, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_many_axes(D, pairs, axes, interleaved):
    from samfast_amd import ops
    q, k, _ = _qk(2, 3, 1, 5, D, torch.bfloat16)
    positions = torch.arange(5 * axes, device="cuda").view(5, axes)
    freq = _frequencies(pairs, axes)
    for o, t in zip(ops.rotary(q, k, positions, freq, interleaved=interleaved), (q, k)):
        _check(o, t, positions, freq, interleaved, 1.0)
        assert torch.equal(o[..., 2 * axes * pairs:], t[..., 2 * axes * pairs:])
