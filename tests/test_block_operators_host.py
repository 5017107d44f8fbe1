"""What the C entries of the 4-bit Linear, the norms over the residual and the rotary positions refuse before any launch: no GPU needed."""

import ctypes

import pytest


def _lib():
    from samfast_amd import _lib
    return _lib.load()


def _refused(code, text):
    lib = _lib()
    assert code < 0 and text in lib.samfast_last_error().decode(), (code, lib.samfast_last_error())


P, Q = 0x1000, 0x2000  # aligned addresses that are never read


def _linear(x=P, ldx=64, codes=P, scales=P, zeros=None, bias=None, y=P, ldy=40, work=P, M=2, N=40, K=64, group=32, dtype=0):
    return _lib().samfast_linear_i4(x, ldx, codes, scales, zeros, bias, y, ldy, work, M, N, K, group, dtype, None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "element type"), (dict(M=-1), "bad shape"), (dict(N=0, ldy=1), "bad shape"), (dict(K=0), "bad shape"), (dict(K=60), "bad shape"),
    (dict(group=0), "groups"), (dict(group=48), "groups"), (dict(group=-32), "groups"), (dict(x=None), "null"), (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(y=None), "null"),
    (dict(ldx=56), "row strides"), (dict(ldx=68), "row strides"), (dict(ldy=39), "row strides"), (dict(x=P + 8), "aligned"), (dict(codes=P + 2), "aligned"),
    (dict(bias=P + 2), "aligned"), (dict(M=1 << 31), "too large"), (dict(ldx=1 << 22), "too large")])
def test_linear_i4_refuses(change, text):
    _refused(_linear(**change), text)


def test_no_rows_are_accepted_without_memory():
    lib = _lib()
    assert _linear(M=0, x=None, y=None) == 0
    assert lib.samfast_linear_i4_workspace(0, 8, 64) >= 0 and lib.samfast_linear_i4_workspace(-1, 8, 64) < 0 and lib.samfast_linear_i4_workspace(1, 0, 64) < 0
    assert _norm(M=0, x=None, residual=None, total=None) == 0
    assert _rotary(B=0, q=None) == 0 and _rotary(T=0, q=None) == 0 and _rotary(heads_q=0, heads_k=0) == 0


def _norm(x=P, ldx=64, residual=P, ld_res=64, gate=None, gate_rows=1, post=None, post_beta=None, post_eps=0.0, pre=P, pre_beta=None, pre_eps=0.0,
          total=P, normed=P, M=6, K=64, dtype=0, f32=0):
    return _lib().samfast_norm_residual(x, ldx, residual, ld_res, gate, gate_rows, post, post_beta, post_eps, pre, pre_beta, pre_eps, 0, 1.0, 1.0,
                                        total, normed, M, K, dtype, f32, None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "element type"), (dict(M=-1), "bad shape"), (dict(K=0), "bad shape"), (dict(K=32769, ldx=32769, ld_res=32769), "bad shape"), (dict(M=1 << 31), "too large"),
    (dict(normed=None), "go together"), (dict(pre=None), "go together"), (dict(post_beta=P), "without its weight"),
    (dict(gate=P, gate_rows=4), "evenly"), (dict(gate=P, gate_rows=0), "evenly"), (dict(pre_eps=-1e-6), "negative"), (dict(post_eps=-1.0), "negative"),
    (dict(x=None), "null"), (dict(residual=None), "null"), (dict(total=None), "null"), (dict(ldx=63), "row strides"), (dict(ld_res=63), "row strides")])
def test_norm_residual_refuses(change, text):
    _refused(_norm(**change), text)


def _rotary(q=P, k=P, q_out=P, k_out=P, positions=P, pos_sb=0, frequencies=P, B=1, T=2, heads_q=2, heads_k=1, D=64, pairs=16, axes=2, strides=True, dtype=0):
    s = (ctypes.c_int64 * 12)(*range(12)) if strides else None
    return _lib().samfast_rotary(q, k, q_out, k_out, positions, pos_sb, frequencies, B, T, heads_q, heads_k, D, pairs, axes, 0, 1.0, s, dtype, None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=-1), "element type"), (dict(B=-1), "bad shape"), (dict(T=-1), "bad shape"), (dict(heads_k=-1), "bad shape"), (dict(T=1 << 31), "bad shape"),
    (dict(pairs=17), "do not fit"), (dict(axes=0), "do not fit"), (dict(pairs=0), "do not fit"), (dict(D=1026), "do not fit"), (dict(pairs=1 << 30), "do not fit"),
    (dict(strides=False), "null"), (dict(q=None), "null"), (dict(k_out=None), "null"), (dict(positions=None), "null"), (dict(frequencies=None), "null"),
    (dict(B=1 << 20, T=1 << 12), "too many tokens")])
def test_rotary_refuses(change, text):
    _refused(_rotary(**change), text)


def test_rotary_refuses_more_pieces_than_a_workgroup_holds():
    _refused(_rotary(axes=65, pairs=1, D=256), "at most 64")
    _refused(_rotary(axes=300, pairs=1, D=640), "at most 64")


@pytest.mark.parametrize("change", [dict(M=1 << 30, N=1, K=8, ldx=8, ldy=1), dict(M=1, N=1 << 29, K=4096, ldx=4096, ldy=1 << 29)])
def test_linear_i4_refuses_what_no_launch_holds(change):
    _refused(_linear(**change), "too many for a launch")


def test_norm_residual_and_rotary_refuse_what_no_launch_holds():
    _refused(_norm(M=(1 << 31) - 1), "too many for a launch")
    _refused(_rotary(B=1, T=(1 << 31) - 2, D=1024, pairs=512, axes=1), "too many tokens")


@pytest.mark.parametrize("change", [dict(ld_res=72), dict(total=Q, x=Q, ldx=72), dict(total=Q, x=Q, f32=1)])
def test_norm_residual_refuses_a_total_over_rows_of_another_layout(change):
    _refused(_norm(**change), "another layout")


def test_rotary_refuses_in_place_in_another_layout():
    _refused(_rotary(), "another layout")


def test_norm_residual_refuses_an_fp32_total_over_a_single_half_type_row():
    _refused(_norm(M=1, total=Q, x=Q, f32=1), "another layout")
    _refused(_norm(M=1, total=Q, x=Q, residual=Q, f32=1), "another layout")
