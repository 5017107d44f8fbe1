"""Which memory an operator's `out` may have: the helpers that decide, on the CPU."""

import itertools

import pytest
import torch


def _cells(t):
    return {t.storage_offset() + sum(i * s for i, s in zip(at, t.stride())) for at in itertools.product(*map(range, t.shape))}


def _views():
    m = torch.zeros(4096, dtype=torch.bfloat16)
    tokens = m[:2 * 5 * 6 * 8].view(2, 5, 6, 8)             # image, token, head, channel
    heads = tokens.permute(0, 2, 1, 3)
    yield from (heads[:, :3], heads[:, 3:], heads[:, 2:4], heads[:, 0::2], heads[:, 1::2], heads[:1], heads[1:], heads[:, :, 1:3], heads[:, :, :0])
    yield from (heads[..., :4], heads[..., 4:], heads[..., 2:6], tokens, tokens[:, ::2], tokens[:, 1::2], m[480:960].view(2, 5, 6, 8))
    yield from (m[4:484].view(2, 6, 5, 8), m[:8].expand(2, 6, 5, 8), m[:80].view(2, 1, 5, 8).expand(2, 6, 5, 8), m.as_strided((2, 3, 5, 8), (120, 8, 24, 1)))
    yield from (m.as_strided((2, 2, 5, 8), (40, 4, 8, 1)), m.as_strided((2, 3, 5, 8), (130, 40, 8, 1)), m[3:4].view(1, 1, 1, 1), m.as_strided((2, 2, 2, 2), (1, 1, 1, 1)))


def test_views_that_are_called_apart_share_nothing():
    from samfast_amd import ops
    views = list(_views())
    for t in views:
        if not ops._overlaps_itself(t):
            assert len(_cells(t)) == t.numel()
    for a, b in itertools.product(views, views):
        if ops._apart(a, b):
            assert not _cells(a) & _cells(b)


def test_common_layouts_are_taken():
    from samfast_amd import ops
    fused = torch.zeros((2, 5, 10, 8), dtype=torch.bfloat16)
    q, k, v = fused[:, :, :6].permute(0, 2, 1, 3), fused[:, :, 6:8].permute(0, 2, 1, 3), fused[:, :, 8:].permute(0, 2, 1, 3)
    for a, b in ((q, k), (k, q), (q, v), (k, v)):
        assert ops._apart(a, b)
    halves = torch.zeros((3, 2, 4, 5, 8))
    assert ops._apart(halves[:, 0], halves[:, 1]) and not ops._apart(halves[:, 0], halves[:, :, 1])
    for t in (q, k, q.contiguous(), q[..., 1:], halves[:, 1], halves[0, 0, 0]):
        assert not ops._overlaps_itself(t)
    for t in (torch.zeros(3).expand(2, 3), torch.zeros(9).as_strided((4, 4), (1, 1)), torch.zeros(9).as_strided((2, 3), (2, 1))):
        assert ops._overlaps_itself(t)


@pytest.mark.gpu
def test_rotary_in_place_needs_memory_of_its_own():
    from samfast_amd import ops, rotary_frequencies
    q = torch.randn((2, 4, 10, 64), device="cuda").bfloat16()
    positions, freq = torch.arange(10, device="cuda"), rotary_frequencies(32, device="cuda")
    shared = q[:, :1].expand(2, 4, 10, 64)
    half = q[:, 1:3]
    for args, out in [((q, q), (q, q)), ((shared, None), (shared, None)), ((q, half), (q, half)), ((q, half), (torch.empty_like(q), q[:, 2:])),
                      ((q, half), (torch.empty_like(q),))]:
        kept = q.clone()
        with pytest.raises(RuntimeError, match="samfast"):
            ops.rotary(*args, positions, freq, out=out)
        assert torch.equal(q, kept)
    # both heads of a buffer in place, and each into the other's gap
    fused = torch.randn((2, 10, 6, 64), device="cuda").bfloat16()
    a, b = fused[:, :, 0::2].permute(0, 2, 1, 3), fused[:, :, 1::2].permute(0, 2, 1, 3)
    want = ops.rotary(a, b, positions, freq)
    ops.rotary(a, None, positions, freq, out=(b, None))
    assert torch.equal(b, want[0])
    want = ops.rotary(a, b, positions, freq)
    ops.rotary(a, b, positions, freq, out=(a, b))
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
