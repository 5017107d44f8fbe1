"""Norms joined over a gated residual, against the formula in 64 bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _norm(v, norm, rms):
    gamma, beta, eps = norm
    if not rms:
        v = v - v.mean(-1, keepdim=True)
    v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()
    return v if beta is None else v + beta.double()


def _inputs(M, K, dtype, stream, groups, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M + 3 * K)
    r = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    x, residual = (2 * r(M, K) + 0.3).to(dtype), (6 * r(M, K) + 0.5).to(stream)
    gate = None if groups == 0 else r(K).to(dtype) if groups == 1 else r(groups, K).to(dtype)
    norms = [((1 + 0.1 * r(K)).to(dtype), beta, 1e-6) for beta in (r(K).to(dtype), None)]
    return x, residual, gate, norms


def _reference(x, residual, gate, post, pre, rms, bs, rs):
    f = x.double()
    if post is not None:
        f = _norm(f, post, rms)
    if gate is not None:
        f = f * (gate if gate.dim() == 1 else gate.repeat_interleave(x.shape[0] // gate.shape[0], 0)).double()
    total = rs * residual.double() + bs * f
    return total, None if pre is None else _norm(total, pre, rms)


def _close(got, ref, slack):
    """One rounding to the type, and `slack` of the row's size for the fp32 steps before it."""
    half = torch.finfo(got.dtype).eps / 2
    size = ref.abs().amax(-1, keepdim=True)
    assert ((got.double() - ref).abs() <= half * ref.abs() + slack * size + 2.0 ** -25).all()


@pytest.mark.parametrize("M,K", [(1, 1), (2, 3), (1, 8), (6, 64), (4, 250), (3, 257), (6, 511), (4, 768), (2, 1003), (8, 1280), (6, 2047), (4, 4099),
                                 (2, 8192), (2, 10007), (300, 1280), (1030, 333), (1200, 1000), (2050, 2048), (130, 32768)])
@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("rms", [False, True])
def test_norm_residual(M, K, dtype, stream, rms):
    from samfast_amd import ops
    print(f"case norm_residual M={M} K={K} {dtype} {stream} rms={rms}", flush=True)
    groups = 2 if M % 2 == 0 else M % 3
    x, residual, gate, (with_beta, without) = _inputs(M, K, dtype, stream, groups)
    kept = residual.clone()
    for post, pre, bs, rs in [(with_beta, without, 0.5, 0.9), (None, with_beta, 1.0, 1.0), (without, None, -1.5, 0.0), (None, None, 1.0, 1.0)]:
        total, normed = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre, rms=rms, branch_scale=bs, residual_scale=rs)
        assert total.dtype == stream and (normed is None) == (pre is None) and torch.equal(residual, kept)
        ref_total, ref_normed = _reference(x, residual, gate, post, pre, rms, bs, rs)
        # statistics are fp32 sums in a tree of at most 32 + 10 levels: relative 64 * 2^-24; a row of one value has variance 0, and the
        # norm then multiplies the difference of the value and its mean, at most its last bit, by 1 / sqrt(eps) = 1000
        slack = 256 * 2.0 ** -24
        if K == 1 and not rms:
            slack = slack * 1000 * float(max(x.double().abs().max(), ref_total.abs().max()))
        _close(total, ref_total, slack)
        if pre is not None:
            # its input is off by `slack` of the row's size, which the norm divides by the row's deviation
            spread = (ref_total.abs().amax(-1) / (ref_total.square().mean(-1) if rms else ref_total.var(-1, correction=0)).add(pre[2]).sqrt()).max()
            _close(normed, ref_normed, slack * max(1.0, float(spread)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_large_mean_does_not_drown_the_deviation(dtype):
    """Values around 1000 that differ in their last bits: squares minus the mean's square would lose them."""
    from samfast_amd import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    step = 4.0 if dtype is torch.bfloat16 else 0.5
    x = (1000.0 // step + torch.randint(0, 4, (8, 1280), generator=g, device="cuda")) * step
    x = x.to(dtype)
    one = torch.ones(1280, dtype=dtype, device="cuda")
    total, normed = ops.norm_residual(x, torch.zeros_like(x), post=(one, None, 0.0), pre=(one, None, 0.0))
    ref = _norm(x.double(), (one, None, 0.0), False)
    # the mean of 1280 values near 1000 in fp32: off by 2^-24 * 1000 * 16 against a deviation above `step`
    for got in (total, normed):
        assert ((got.double() - ref).abs() <= torch.finfo(dtype).eps * ref.abs() + 2.0 ** -24 * 16000 / step * 2).all()


def test_in_place_strides_shapes_and_no_rows():
    from samfast_amd import ops
    x, residual, gate, (post, pre) = _inputs(24, 200, torch.bfloat16, torch.float32, 2)
    want = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre)
    wide_x, wide_r = torch.full((24, 333), float("nan"), device="cuda", dtype=x.dtype), torch.full((24, 211), float("nan"), device="cuda")
    wide_x[:, 7:207], wide_r[:, 11:211] = x, residual
    got = ops.norm_residual(wide_x[:, 7:207], wide_r[:, 11:211], gate=gate, post=post, pre=pre)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = ops.norm_residual(x.view(2, 3, 4, 200), residual.view(2, 3, 4, 200), gate=gate, post=post, pre=pre)
    assert got[0].shape == got[1].shape == (2, 3, 4, 200) and torch.equal(got[0].view(24, 200), want[0]) and torch.equal(got[1].view(24, 200), want[1])
    row = ops.norm_residual(x[0], residual[0], post=post, pre=pre)
    assert row[0].shape == (200,)
    stream = residual.clone()
    total, normed = ops.norm_residual(x, stream, gate=gate, post=post, pre=pre, out=stream)
    assert total is stream and torch.equal(stream, want[0]) and torch.equal(normed, want[1])
    none = ops.norm_residual(x[:0], residual[:0], post=post, pre=pre)
    assert none[0].shape == none[1].shape == (0, 200)


@pytest.mark.parametrize("M,K", [(700, 5), (3000, 9), (2000, 333), (900, 1003), (500, 1999), (300, 5001), (100, 20001)])
@pytest.mark.parametrize("norms", [0, 1, 2])
def test_in_place_at_odd_widths(M, K, norms):
    """Threads that share values of a row read them before one of them writes."""
    from samfast_amd import ops
    x, residual, gate, (post, pre) = _inputs(M, K, torch.bfloat16, torch.bfloat16, 1)
    post, pre = post if norms > 0 else None, pre if norms > 1 else None
    want = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre, residual_scale=0.5)
    for held in (residual, x):
        mine = held.clone()
        args = (mine, residual) if held is x else (x, mine)
        total, normed = ops.norm_residual(*args, gate=gate, post=post, pre=pre, residual_scale=0.5, out=mine)
        assert total is mine and torch.equal(mine, want[0]) and (pre is None or torch.equal(normed, want[1]))


def test_a_row_that_is_not_finite_stays_alone():
    from samfast_amd import ops
    x, residual, gate, (post, pre) = _inputs(9, 1280, torch.bfloat16, torch.bfloat16, 1)
    clean = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre)
    x[3, 4], residual[7, 1279] = float("nan"), float("inf")
    total, normed = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre)
    others = [0, 1, 2, 4, 5, 6, 8]
    assert torch.equal(total[others], clean[0][others]) and torch.equal(normed[others], clean[1][others])
    assert total[3].isnan().all() and normed[3].isnan().all() and normed[7].isnan().all() and total[7, 1279] == float("inf")


def test_refusals():
    from samfast_amd import ops
    x, residual, gate, (post, pre) = _inputs(6, 64, torch.bfloat16, torch.float32, 2)
    wide = torch.zeros((1, 32769), dtype=torch.bfloat16, device="cuda")
    half = x.half()
    cases = [
        dict(x=x.float()), dict(residual=residual[:5]), dict(residual=residual.double()), dict(residual=half), dict(gate=gate.float()),
        dict(gate=gate[:, :63]), dict(gate=torch.cat((gate, gate))), dict(gate=gate[:0]), dict(gate=gate.view(1, 2, 64)), dict(post=(post[0].float(), None, 1e-6)),
        dict(post=(post[0][:63], None, 1e-6)), dict(pre=(pre[0], post[1].half(), 1e-6)), dict(pre=(None, None, 1e-6)), dict(post=(post[0], None, -1.0)),
        dict(out=residual[:5]), dict(out=x), dict(x=x.cpu()), dict(residual=residual.cpu()), dict(x=x.clone().requires_grad_()),
        dict(x=wide, residual=wide, gate=None, post=None, pre=None),
    ]
    for case in cases:
        args = dict(dict(x=x, residual=residual, gate=gate, post=post, pre=pre), **case)
        with pytest.raises(RuntimeError, match="samfast"):
            ops.norm_residual(**args)


@pytest.mark.parametrize("K", [4104, 4360, 7935, 7936, 8200])  # 17, 18, 31, 31 halves of wavefronts to a row; 17 with two pieces a thread
@pytest.mark.parametrize("rms", [False, True])
def test_rows_of_odd_halves_of_wavefronts(K, rms):
    """An odd number of halves above 15 leaves half a wavefront without a row; all four sums are taken."""
    from samfast_amd import ops
    x, residual, gate, (post, pre) = _inputs(4, K, torch.float16, torch.float32, 2)
    total, normed = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre, rms=rms)
    ref_total, ref_normed = _reference(x, residual, gate, post, pre, rms, 1.0, 1.0)
    _close(total, ref_total, 256 * 2.0 ** -24)
    spread = (ref_total.abs().amax(-1) / (ref_total.square().mean(-1) if rms else ref_total.var(-1, correction=0)).add(pre[2]).sqrt()).max()
    _close(normed, ref_normed, 256 * 2.0 ** -24 * max(1.0, float(spread)))
    again = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre, rms=rms)
    assert torch.equal(again[0], total) and torch.equal(again[1], normed)
