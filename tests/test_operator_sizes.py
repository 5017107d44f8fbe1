"""Sizes on their way from Python integers to the 32-bit arguments of the C ABI: with a stand-in for the library and tensors without memory, on the CPU."""

import pytest
import torch

HALF = torch.bfloat16


class _Library:
    """Takes every call and keeps its arguments."""

    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        return lambda *args: self.calls.__setitem__(name, args) or 0


@pytest.fixture
def library(monkeypatch):
    from samfast_amd import _lib, ops
    _lib.host()
    stand_in = _Library()
    monkeypatch.setattr(_lib, "load", lambda: stand_in)
    monkeypatch.setattr(ops, "_require_here", lambda *args: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    return stand_in


def _empty(*shape, dtype=HALF):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("group", [96, 128, 1024, (1 << 31) - 32, 1 << 31, (1 << 32) + 32])
def test_a_group_longer_than_the_rows_is_one_group(library, group):
    from samfast_amd import ops
    y = ops.linear_i4(_empty(2, 72), _empty(5, 36, dtype=torch.uint8), _empty(1, 5), group_size=group)
    *_, M, N, K, passed, dtype, stream = library.calls["samfast_linear_i4"]
    assert y.shape == (2, 5) and (M, N, K) == (2, 5, 72)
    assert passed % 32 == 0 and 72 <= passed < 1 << 31


def test_outputs_beyond_32_bits_are_refused(library):
    from samfast_amd import ops
    N = (1 << 32) + 16
    with pytest.raises(RuntimeError, match="samfast"):
        ops.linear_i4(_empty(1, 8), _empty(N, 4, dtype=torch.uint8), _empty(1, N), group_size=32)
    assert not library.calls


def test_widths_beyond_32_bits_are_refused(library):
    from samfast_amd import ops
    for K in (32769, (1 << 32) + 8):
        with pytest.raises(RuntimeError, match="samfast"):
            ops.norm_residual(_empty(1, K), _empty(1, K))
    assert not library.calls


@pytest.mark.parametrize("heads,kv,dim", [((1 << 32) + 1, 1, 2), (1, (1 << 32) + 1, 2), (1, 1, (1 << 32) + 2)])
def test_heads_beyond_32_bits_are_refused(library, heads, kv, dim):
    from samfast_amd import ops
    with pytest.raises(RuntimeError, match="samfast"):
        ops.rotary(_empty(1, heads, 1, dim), _empty(1, kv, 1, dim), _empty(1, dtype=torch.int64), _empty(1, dtype=torch.float64))
    assert not library.calls
