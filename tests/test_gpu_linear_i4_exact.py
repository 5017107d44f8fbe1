"""Linears with 4-bit weights against what they are said to compute, rounding by rounding: exact weights over few rows, weights rounded to the type once over
more; and inputs that one lost piece of K would change altogether."""

import pytest
import torch

from test_gpu_linear_i4 import _operands, _weight

pytestmark = pytest.mark.gpu


def _few(M, N):
    return M <= 32 and N >= 16


def _check_exactly(got, x, codes, scales, zeros, bias, group):
    M, K, N = x.shape[0], x.shape[1], codes.shape[0]
    half, xd = torch.finfo(x.dtype).eps / 2, x.double()
    w = _weight(codes, scales, zeros, group)
    b = 0.0 if bias is None else bias.double()
    if _few(M, N):
        # Codes and zero points are multiplied apart, so the sums are of code * scale * x and zero * scale * x.  A product chain is 128 inputs long at
        # most, at most 4 of them with their zeros' part are scaled and added for 128 inputs of a wavefront's eighth of K (of 256 at a time), and eight wavefronts' sums,
        # the bias and the scaling of a zero come on top.
        of = torch.arange(K, device=x.device) // group
        z = torch.full_like(scales, 8.0).double() if zeros is None else zeros.double()
        size = xd.abs() @ (w.abs() + 2 * (z * scales.double()).t()[:, of]).t()  # code <= |code - zero| + zero
        roundings = 128 + 16 * -(-K // 2048) + 24
    else:
        # (code - zero) * scale is exact in fp32 and rounded to the type once; its products with x are added one after the other at worst
        w = w.float().to(x.dtype).double()
        size = xd.abs() @ w.abs().t()
        roundings = K + 8
    ref = xd @ w.t() + b
    bound = roundings * 2.0 ** -24 * (size + (0.0 if bias is None else bias.double().abs()))
    bound = bound + half * (ref.abs() + bound) + 2.0 ** -25  # (the result is rounded; fp16 has nothing between multiples of 2^-24)
    error = (got.double() - ref).abs()
    assert (error <= bound).all(), float((error / bound).max())


SHAPES = [(256, 40, 64, True), (1000, 131, 64, True), (1096, 67, 32, False), (2048, 16, 128, True), (4104, 33, 256, False), (672, 50, 96, True),
          (640, 257, 640, False), (4096, 8200, 32, True)]


@pytest.mark.parametrize("M", [1, 7, 16, 17, 32, 33, 65, 130])
@pytest.mark.parametrize("K,N,group,zeros", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_roundings(M, K, N, group, zeros, dtype):
    from samfast_amd import ops
    print(f"case roundings M={M} K={K} N={N} group={group} zeros={zeros} {dtype}", flush=True)
    x, codes, scales, z, b = _operands(M, K, N, group, zeros, dtype, bias=M % 2 == 1)
    _check_exactly(ops.linear_i4(x, codes, scales, z, b, group_size=group), x, codes, scales, z, b, group)


@pytest.mark.parametrize("M,K,N,group,zeros", [(4096, 1280, 1280, 128, False), (2049, 712, 1031, 256, True), (5000, 1288, 3001, 64, True), (64, 8192, 300, 32, True),
                                               (300, 4096, 1024, 64, True), (3, 256, 7, 32, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_roundings_of_rounded_weights(M, K, N, group, zeros, dtype):
    test_roundings(M, K, N, group, zeros, dtype)


@pytest.mark.parametrize("M", [1, 7, 17, 40, 300, 5000])
@pytest.mark.parametrize("K,N,group", [(4104, 33, 256), (1000, 600, 64), (1096, 67, 32), (136, 20, 128), (2312, 300, 1024), (8, 40, 32), (264, 9, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_last_inputs_alone(M, K, N, group, dtype):
    """All weights but those of the last eight inputs are 0, and all x but theirs as large as ever: a result is a sum of eight products."""
    from samfast_amd import ops
    x, codes, scales, z, _ = _operands(M, K, N, group, True, dtype)
    of = torch.arange(K, device="cuda") // group
    middle = z.t()[:, of]
    codes[:, :-4] = (middle[:, 0::2] | middle[:, 1::2] << 4)[:, :-4]
    assert (_weight(codes, scales, z, group)[:, :-8] == 0).all()
    got = ops.linear_i4(x, codes, scales, z, None, group_size=group)
    _check_exactly(got, x, codes, scales, z, None, group)
    # and without the rest of x
    x[:, :-8] = 0
    _check_exactly(ops.linear_i4(x, codes, scales, z, None, group_size=group), x, codes, scales, z, None, group)


@pytest.mark.parametrize("M", [1, 16, 17, 32, 33, 300])
@pytest.mark.parametrize("K,N,group,zeros", [(256, 40, 64, True), (1000, 131, 32, False), (4104, 33, 256, True), (2048, 8200, 128, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_input_a_row(M, K, N, group, zeros, dtype):
    """A single value in each row: nothing is summed, and a weight that was rounded where it should not be shows in the result's last place."""
    from samfast_amd import ops
    x, codes, scales, z, _ = _operands(M, K, N, group, zeros, dtype)
    at = torch.arange(M, device="cuda") * 37 % K
    x = torch.zeros_like(x).scatter_(1, at[:, None], x.gather(1, at[:, None]))
    got = ops.linear_i4(x, codes, scales, z, None, group_size=group).double()
    w = _weight(codes, scales, z, group)
    half = torch.finfo(dtype).eps / 2
    of = torch.arange(K, device="cuda") // group
    middle = (torch.full_like(scales, 8.0) if z is None else z).double()
    size = x.double().abs() @ (w.abs() + 2 * (middle * scales.double()).t()[:, of]).t()
    if not _few(M, N):
        w = w.float().to(dtype).double()
    ref = x.double() @ w.t()
    # at most four fp32 steps: a group's sum scaled and added, the zeros' part scaled and added
    slack = 4 * 2.0 ** -24 * size
    assert ((got - ref).abs() <= slack + half * (ref.abs() + slack) + 2.0 ** -25).all()


@pytest.mark.parametrize("M,K,group", [(1, 1000, 32), (16, 512, 128), (24, 2312, 64)])
@pytest.mark.parametrize("N", [4095, 4096, 4097, 5000, 8191, 8192])
def test_outputs_around_a_round_of_workgroups(M, K, group, N):
    """16 or 32 columns to a workgroup, the last columns over the ones before them."""
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(M, K, N, group, True, torch.bfloat16)
    _check_exactly(ops.linear_i4(x, codes, scales, z, b, group_size=group), x, codes, scales, z, b, group)
