"""Linears with 4-bit weights and group scales, against the formula in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _operands(M, K, N, group, zeros, dtype, bias=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + M + 7 * K + 13 * N)
    groups = -(-K // group)
    x = torch.randn((M, K), generator=g, device="cuda").to(dtype)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.01 * (0.5 + torch.rand((groups, N), generator=g, device="cuda"))).to(dtype)
    z = torch.randint(0, 16, (groups, N), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    b = torch.randn((N,), generator=g, device="cuda") if bias else None
    return x, codes, scales, z, b


def _weight(codes, scales, zeros, group):
    N, K = codes.shape[0], 2 * codes.shape[1]
    c = torch.stack((codes % 16, codes // 16), -1).view(N, K).double()
    of = torch.arange(K, device=codes.device) // group
    z = torch.full_like(scales, 8.0).double() if zeros is None else zeros.double()
    return (c - z.t()[:, of]) * scales.double().t()[:, of]


def _check(got, x, codes, scales, zeros, bias, group):
    assert got.dtype == x.dtype and got.shape == (*x.shape[:-1], codes.shape[0])
    xd, w = x.double().reshape(-1, x.shape[-1]), _weight(codes, scales, zeros, group)
    b = 0.0 if bias is None else bias.double()
    ref, size = xd @ w.t() + b, xd.abs() @ w.abs().t() + (0.0 if bias is None else bias.double().abs())
    half = torch.finfo(x.dtype).eps / 2
    # every weight may be rounded to the type (and the type's subnormals) once, and the output is; fp32 sums of K products: at most K roundings
    # of partial sums below `size`, and one each of a product
    bound = half * size + 2.0 ** -25 * xd.abs().sum(-1, keepdim=True) + (x.shape[-1] + 8) * 2.0 ** -24 * size
    bound = bound + half * (ref.abs() + bound) + 2.0 ** -25
    assert ((got.double().reshape(ref.shape) - ref).abs() <= bound).all()


@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("K,N,group,zeros", [(8, 1, 32, False), (256, 40, 64, True), (1000, 131, 64, True), (1096, 67, 32, False),
                                             (2048, 16, 128, True), (4104, 33, 256, False), (672, 50, 96, True), (640, 257, 640, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_i4(M, K, N, group, zeros, dtype):
    from samfast_amd import ops
    print(f"case linear_i4 M={M} K={K} N={N} group={group} zeros={zeros} {dtype}", flush=True)
    x, codes, scales, z, b = _operands(M, K, N, group, zeros, dtype, bias=M % 2 == 1)
    outs = [ops.linear_i4(x, codes, scales, z, b, group_size=group) for _ in range(2)]
    assert torch.equal(outs[0], outs[1])
    _check(outs[0], x, codes, scales, z, b, group)


@pytest.mark.parametrize("M,K,N,group,zeros", [
    (1000, 320, 520, 32, True), (4096, 1280, 1280, 128, False), (333, 1000, 1003, 64, True), (2049, 712, 1031, 256, True),
    (5000, 1280, 3840, 128, True), (8200, 640, 648, 64, False), (300, 8192, 96, 128, True), (9001, 328, 2050, 32, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_i4_over_many_rows(M, K, N, group, zeros, dtype):
    test_linear_i4(M, K, N, group, zeros, dtype)


def test_rows_of_any_shape_and_stride():
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(24, 512, 96, 64, True, torch.bfloat16)
    want = ops.linear_i4(x, codes, scales, z, b, group_size=64)
    wide = torch.full((24, 1000), float("nan"), dtype=x.dtype, device="cuda")
    for at in (0, 8, 3):  # strided rows, the last at an odd address
        view = wide[:, at:at + 512]
        view.copy_(x)
        assert torch.equal(ops.linear_i4(view, codes, scales, z, b, group_size=64), want)
    assert torch.equal(ops.linear_i4(x.view(2, 3, 4, 512), codes, scales, z, b, group_size=64), want.view(2, 3, 4, 96))
    assert torch.equal(ops.linear_i4(x[0], codes, scales, z, b, group_size=64), ops.linear_i4(x[:1], codes, scales, z, b, group_size=64)[0])
    assert torch.equal(ops.linear_i4(x.t().contiguous().t(), codes, scales, z, b, group_size=64), want)
    assert ops.linear_i4(x[:0], codes, scales, z, b, group_size=64).shape == (0, 96)


@pytest.mark.parametrize("M", [3, 40, 300, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_row_that_is_not_finite_stays_alone(M, dtype):
    """A NaN makes its row NaN; an infinity gives what the formula gives, infinities by the sign of the weight it meets."""
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(M, 1000, 131, 64, True, dtype)
    clean = ops.linear_i4(x, codes, scales, z, b, group_size=64)
    x[0, 5], x[M - 1, 999] = float("nan"), float("inf")
    got = ops.linear_i4(x, codes, scales, z, b, group_size=64)
    assert got[0].isnan().all() and torch.equal(got[1:M - 1], clean[1:M - 1])
    want = (_weight(codes, scales, z, 64)[:, 999] * float("inf")).to(dtype)
    assert torch.equal(got[M - 1].isnan(), want.isnan()) and torch.equal(got[M - 1][~want.isnan()], want[~want.isnan()])


def test_neighbouring_memory_is_left_alone():
    """An output in a larger buffer through the C ABI: rows end at column N, and nothing lies behind the last."""
    from samfast_amd import _lib, ops
    lib = _lib.load()
    for M, K, N in [(5, 256, 37), (70, 264, 131), (400, 328, 203), (600, 640, 520)]:
        x, codes, scales, z, b = _operands(M, K, N, 32, True, torch.bfloat16)
        buf = torch.full((M + 2, N + 5), 7.0, dtype=torch.bfloat16, device="cuda")
        need = lib.samfast_linear_i4_workspace(M, N, K)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        y = buf[1:]
        _lib.check(lib.samfast_linear_i4(x.data_ptr(), K, codes.data_ptr(), scales.data_ptr(), z.data_ptr(), b.data_ptr(), y.data_ptr(), N + 5,
                                         work.data_ptr(), M, N, K, 32, 0, torch.cuda.current_stream().cuda_stream), "linear_i4")
        want = ops.linear_i4(x, codes, scales, z, b, group_size=32)
        assert torch.equal(y[:M, :N], want)
        assert (buf[0] == 7).all() and (buf[M + 1] == 7).all() and (buf[:, N:] == 7).all()


def test_refusals():
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(4, 256, 40, 64, True, torch.bfloat16)
    bad = [
        (x.float(), codes, scales, z, b, 64), (x[:, :128], codes, scales, z, b, 64), (x, codes.char(), scales, z, b, 64),
        (x, codes, scales.float(), z, b, 64), (x, codes, scales[:3], z, b, 64), (x, codes, scales, z.char(), b, 64),
        (x, codes, scales, z[:, :39], b, 64), (x, codes, scales, z, b.bfloat16(), 64), (x, codes, scales, z, b[:39], 64),
        (x, codes, scales, z, b, 48), (x, codes, scales, z, b, 0), (x, codes[:, :126], scales, z, b, 64), (x, codes.t(), scales, z, b, 64),
        (x.cpu(), codes, scales, z, b, 64), (x, codes.cpu(), scales, z, b, 64), (x, codes[:0], scales, z, b, 64),
        (x.clone().requires_grad_(), codes, scales, z, b, 64),
    ]
    for *args, group in bad:
        with pytest.raises(RuntimeError, match="samfast"):
            ops.linear_i4(*args, group_size=group)
    with torch.no_grad():
        ops.linear_i4(x.clone().requires_grad_(), codes, scales, z, b, group_size=64)


@pytest.mark.parametrize("M", [1, 3, 40])
def test_rows_far_apart(M):
    """The last tokens of long prompts: rows that lie megabytes apart."""
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(M, 512, 96, 64, True, torch.bfloat16)
    prompts = torch.zeros((M, 8200, 512), dtype=x.dtype, device="cuda")
    prompts[:, -1] = x
    want = ops.linear_i4(x, codes, scales, z, b, group_size=64)
    assert torch.equal(ops.linear_i4(prompts[:, -1], codes, scales, z, b, group_size=64), want)
    with ops.record_launches():
        assert torch.equal(ops.linear_i4(prompts[:, -1:], codes, scales, z, b, group_size=64), want.view(M, 1, 96))


# rows that end inside 64 values are copied beside the weights, and any number of columns, the last tile over the one before it
@pytest.mark.parametrize("M,K,N,group,zeros", [(5000, 1288, 3001, 64, True), (3001, 1336, 5121, 32, False), (2500, 2048, 4003, 128, True), (6000, 4000, 1990, 256, True),
                                               (20000, 400, 2046, 32, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_written_weights_of_any_shape(M, K, N, group, zeros, dtype):
    from samfast_amd import _lib, ops
    padded = -(-K // 64) * 64
    assert _lib.load().samfast_linear_i4_workspace(M, N, K) == 2 * padded * (N + (M if padded != K else 0))  # this way, not another
    x, codes, scales, z, b = _operands(M, K, N, group, zeros, dtype)
    wide = torch.full((M, K + 24), float("nan"), dtype=dtype, device="cuda")
    wide[:, :K] = x
    got = ops.linear_i4(wide[:, :K], codes, scales, z, b, group_size=group)
    _check(got, x, codes, scales, z, b, group)
    assert torch.equal(ops.linear_i4(x, codes, scales, z, b, group_size=group), got)
    x[5, K - 1], x[M - 1, 0] = float("inf"), float("nan")
    odd = ops.linear_i4(x, codes, scales, z, b, group_size=group)
    rows = torch.ones(M, dtype=torch.bool, device="cuda")
    rows[5] = rows[M - 1] = False
    assert torch.equal(odd[rows], got[rows]) and odd[M - 1].isnan().all() and not odd[5].isfinite().any()


def test_written_weights_leave_neighbouring_memory_alone():
    from samfast_amd import _lib, ops
    lib = _lib.load()
    for M, K, N in [(5000, 1288, 3001), (2500, 2048, 4003), (3001, 1336, 5121)]:
        x, codes, scales, z, b = _operands(M, K, N, 32, True, torch.bfloat16)
        buf = torch.full((M + 2, N + 5), 7.0, dtype=torch.bfloat16, device="cuda")
        work = torch.empty(lib.samfast_linear_i4_workspace(M, N, K) + 64, dtype=torch.uint8, device="cuda")
        work[-64:] = 9
        _lib.check(lib.samfast_linear_i4(x.data_ptr(), K, codes.data_ptr(), scales.data_ptr(), z.data_ptr(), b.data_ptr(), buf[1:].data_ptr(), N + 5,
                                         work.data_ptr(), M, N, K, 32, 0, torch.cuda.current_stream().cuda_stream), "linear_i4")
        assert torch.equal(buf[1:M + 1, :N], ops.linear_i4(x, codes, scales, z, b, group_size=32))
        assert (buf[0] == 7).all() and (buf[M + 1] == 7).all() and (buf[:, N:] == 7).all() and (work[-64:] == 9).all()


@pytest.mark.parametrize("M", [3, 40, 3000])
def test_a_group_longer_than_the_rows(M):
    """One group, however long it is said to be."""
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(M, 1000, 520, 1024, True, torch.bfloat16)
    want = ops.linear_i4(x, codes, scales, z, b, group_size=1024)
    for group in (1 << 16, (1 << 31) - 32, 1 << 31, (1 << 32) + 32):
        assert torch.equal(ops.linear_i4(x, codes, scales, z, b, group_size=group), want)
    with pytest.raises(RuntimeError, match="samfast"):
        ops.linear_i4(x, codes, scales, z, b, group_size=(1 << 32) + 16)


@pytest.mark.parametrize("K", [1000, 1096, 328])  # the last 128 inputs are not all there
@pytest.mark.parametrize("M,N", [(3, 131), (40, 131), (300, 200), (5000, 600), (7, 5)])
@pytest.mark.parametrize("zero", [None, 15, 255])
def test_scales_that_a_zero_point_carries_beyond_fp16(M, N, K, zero):
    """Every weight is finite; a scale times its zero point is not."""
    from samfast_amd import ops
    g = torch.Generator(device="cuda").manual_seed(M + K)
    centre = 8 if zero is None else min(zero, 15)
    low = torch.randint(centre - 2, min(centre + 1, 15) + 1, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    codes = low[:, 0::2] | low[:, 1::2] << 4
    groups = -(-K // 64)
    scales = ((258.0 if zero == 255 else 12000.0) * (1.0 + 0.03 * torch.rand((groups, N), generator=g, device="cuda"))).half()
    z = None if zero is None else torch.full((groups, N), zero, dtype=torch.uint8, device="cuda")
    assert scales.double().max() * (8 if zero is None else zero) > 65504 and _weight(codes, scales, z, 64).abs().max() < 65504
    x = (torch.randn((M, K), generator=g, device="cuda") * 2.0 ** -12).half()
    _check(ops.linear_i4(x, codes, scales, z, None, group_size=64), x, codes, scales, z, None, 64)


@pytest.mark.parametrize("M,K,N", [(3, 1000, 131), (40, 1000, 131), (64, 4096, 200), (300, 1024, 200), (5000, 640, 600), (7, 512, 5)])
@pytest.mark.parametrize("group", [32, 128])
def test_scales_that_a_zero_point_carries_beyond_bf16(M, K, N, group):
    """Weights of at most 7e37 around zero points of 15: fifteen times a scale is more than the type, and fp32, can hold."""
    from samfast_amd import ops
    g = torch.Generator(device="cuda").manual_seed(M + K)
    low = torch.randint(13, 16, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    codes = low[:, 0::2] | low[:, 1::2] << 4
    groups = -(-K // group)
    scales = (2.5e37 * (1.0 + 0.3 * torch.rand((groups, N), generator=g, device="cuda"))).bfloat16()
    z = torch.full((groups, N), 15, dtype=torch.uint8, device="cuda")
    x = (torch.randn((M, K), generator=g, device="cuda") * 2.0 ** -20).bfloat16()
    _check(ops.linear_i4(x, codes, scales, z, None, group_size=group), x, codes, scales, z, None, group)
