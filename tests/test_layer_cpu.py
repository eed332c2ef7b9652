"""The transformer-layer entries refuse what they cannot do before any CUDA call."""

import ctypes as C

import pytest

from tensorforge_b200 import _lib

P = 1 << 20  # fake, aligned "device" addresses, far apart


def linear(**kw):
    a = _lib.LinearArgs(activation=1, trans_b=1, a_dtype=_lib.BF16, b_dtype=_lib.BF16, out_dtype=_lib.BF16,
                        residual_dtype=_lib.BF16, A=P, B=2 * P, bias=3 * P, residual=4 * P, out=5 * P, pre=6 * P, M=8, N=16, K=24)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().tforge_linear(C.byref(a), None)


def backward(**kw):
    a = _lib.LinearBackwardArgs(activation=1, trans_b=1, a_dtype=_lib.BF16, b_dtype=_lib.BF16, dtype=_lib.BF16,
                                grad_dtype=_lib.BF16, dout=P, pre=2 * P, A=3 * P, B=4 * P, dA=5 * P, dB=6 * P, dbias=7 * P,
                                M=8, N=16, K=24)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().tforge_linear_backward(C.byref(a), None)


def norm(**kw):
    a = _lib.RmsNormArgs(dtype=_lib.BF16, weight_dtype=_lib.F32, out_dtype=_lib.E4M3, eps=1e-5, x=P, residual=2 * P,
                         weight=3 * P, sum_out=4 * P, out=5 * P, scale=6 * P, rstd=7 * P, M=8, N=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().tforge_rms_norm(C.byref(a), None)


def norm_backward(**kw):
    a = _lib.RmsNormBackwardArgs(dtype=_lib.BF16, weight_dtype=_lib.F32, dy=P, s=2 * P, weight=3 * P, rstd=4 * P, ds=5 * P,
                                 dx=6 * P, dweight=7 * P, M=8, N=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return _lib.lib().tforge_rms_norm_backward(C.byref(a), None)


E8 = dict(a_dtype=_lib.E4M3, b_dtype=_lib.E4M3, a_scale=8 * P, b_scale=9 * P)
BIG = 1 << 31


@pytest.mark.parametrize("call,kw,code", [
    (linear, dict(activation=5), _lib.ERR_MODE),
    (linear, dict(activation=-1), _lib.ERR_MODE),
    (linear, dict(trans_b=2), _lib.ERR_MODE),
    (linear, dict(a_dtype=7), _lib.ERR_MODE),
    (linear, dict(a_dtype=_lib.E4M3), _lib.ERR_MODE),  # one 8-bit operand only
    (linear, dict(out_dtype=_lib.E4M3), _lib.ERR_MODE),
    (linear, dict(residual_dtype=_lib.E4M3), _lib.ERR_MODE),
    (linear, dict(a_scale=8 * P), _lib.ERR_MODE),  # scales belong to 8-bit operands
    (linear, dict(E8, trans_b=0), _lib.ERR_UNSUPPORTED),
    (linear, dict(E8, a_scale=None), _lib.ERR_NULL),
    (linear, dict(E8, b_scale=None), _lib.ERR_NULL),
    (linear, dict(M=-1), _lib.ERR_SHAPE),
    (linear, dict(K=BIG), _lib.ERR_SHAPE),
    (linear, dict(lda=23), _lib.ERR_SHAPE),
    (linear, dict(ldb=23), _lib.ERR_SHAPE),
    (linear, dict(trans_b=0, ldb=15), _lib.ERR_SHAPE),
    (linear, dict(ldr=15), _lib.ERR_SHAPE),
    (linear, dict(ldo=-16), _lib.ERR_SHAPE),
    (linear, dict(ldp=15), _lib.ERR_SHAPE),
    (linear, dict(lda=1 << 62), _lib.ERR_SHAPE),
    (linear, dict(A=None), _lib.ERR_NULL),
    (linear, dict(out=None), _lib.ERR_NULL),
    (linear, dict(A=P + 1), _lib.ERR_ALIGN),
    (linear, dict(bias=3 * P + 2), _lib.ERR_ALIGN),
    (linear, dict(out=P), _lib.ERR_ALIAS),
    (linear, dict(pre=5 * P + 16), _lib.ERR_ALIAS),
    (linear, dict(out=4 * P, residual_dtype=_lib.F32), _lib.ERR_ALIAS),  # in place needs one type
    (linear, dict(out=4 * P, ldo=20), _lib.ERR_ALIAS),  # and one pitch
    (linear, dict(pre=4 * P), _lib.ERR_ALIAS),
    (linear, dict(M=0), _lib.OK),
    (linear, dict(N=0, ldb=0), _lib.OK),
    (backward, dict(activation=9), _lib.ERR_MODE),
    (backward, dict(a_dtype=_lib.E4M3), _lib.ERR_MODE),
    (backward, dict(grad_dtype=_lib.E4M3), _lib.ERR_MODE),
    (backward, dict(dtype=5), _lib.ERR_MODE),
    (backward, dict(pre=None), _lib.ERR_NULL),
    (backward, dict(dout=None), _lib.ERR_NULL),
    (backward, dict(A=None), _lib.ERR_NULL),
    (backward, dict(B=None), _lib.ERR_NULL),
    (backward, dict(lddo=15), _lib.ERR_SHAPE),
    (backward, dict(N=-2), _lib.ERR_SHAPE),
    (backward, dict(dA=5 * P + 1), _lib.ERR_ALIGN),
    (backward, dict(dA=3 * P), _lib.ERR_ALIAS),
    (backward, dict(dB=5 * P), _lib.ERR_ALIAS),
    (backward, dict(dbias=P), _lib.ERR_ALIAS),
    (backward, dict(dA=None, dB=None, dbias=None), _lib.OK),
    (norm, dict(dtype=_lib.E4M3), _lib.ERR_MODE),
    (norm, dict(weight_dtype=_lib.E4M3), _lib.ERR_MODE),
    (norm, dict(out_dtype=3), _lib.ERR_MODE),
    (norm, dict(eps=-1.0), _lib.ERR_SHAPE),
    (norm, dict(eps=float("nan")), _lib.ERR_SHAPE),
    (norm, dict(eps=float("inf")), _lib.ERR_SHAPE),
    (norm, dict(scale=None), _lib.ERR_NULL),
    (norm, dict(x=None), _lib.ERR_NULL),
    (norm, dict(ldx=15), _lib.ERR_SHAPE),
    (norm, dict(x=P + 1), _lib.ERR_ALIGN),
    (norm, dict(rstd=7 * P + 2), _lib.ERR_ALIGN),
    (norm, dict(out=P), _lib.ERR_ALIAS),
    (norm, dict(out_dtype=_lib.BF16, out=4 * P), _lib.ERR_ALIAS),
    (norm, dict(sum_out=2 * P, lds=20), _lib.ERR_ALIAS),  # in place needs one pitch
    (norm, dict(sum_out=3 * P), _lib.ERR_ALIAS),
    (norm, dict(N=0), _lib.OK),
    (norm_backward, dict(dtype=2), _lib.ERR_MODE),
    (norm_backward, dict(rstd=None), _lib.ERR_NULL),
    (norm_backward, dict(dx=2 * P), _lib.ERR_ALIAS),
    (norm_backward, dict(dx=P), _lib.ERR_ALIAS),
    (norm_backward, dict(dx=5 * P, lddx=32), _lib.ERR_ALIAS),
    (norm_backward, dict(dweight=3 * P), _lib.ERR_ALIAS),
    (norm_backward, dict(lds=8), _lib.ERR_SHAPE),
    (norm_backward, dict(N=0), _lib.OK),
])
def test_refusals(call, kw, code):
    assert call(**kw) == code


def test_null_arguments():
    L = _lib.lib()
    assert L.tforge_linear(None, None) == _lib.ERR_NULL
    assert L.tforge_linear_backward(None, None) == _lib.ERR_NULL
    assert L.tforge_rms_norm(None, None) == _lib.ERR_NULL
    assert L.tforge_rms_norm_backward(None, None) == _lib.ERR_NULL


def test_quantizer_refusals():
    q = _lib.lib().tforge_quantize_e4m3
    assert q(P, _lib.E4M3, 2 * P, 3 * P, 8, 16, 0, 0, None) == _lib.ERR_MODE
    assert q(P, _lib.BF16, 2 * P, None, 8, 16, 0, 0, None) == _lib.ERR_NULL
    assert q(P, _lib.BF16, 2 * P, 3 * P, 8, 16, 8, 0, None) == _lib.ERR_SHAPE
    assert q(P, _lib.BF16, 2 * P, 3 * P, 8, 16, 0, 15, None) == _lib.ERR_SHAPE
    assert q(P + 1, _lib.BF16, 2 * P, 3 * P, 8, 16, 0, 0, None) == _lib.ERR_ALIGN
    assert q(P, _lib.BF16, P, 3 * P, 8, 16, 0, 0, None) == _lib.ERR_ALIAS
    assert q(None, _lib.BF16, None, None, 0, 16, 0, 0, None) == _lib.OK


def test_python_entries_raise():
    with pytest.raises(_lib.TforgeError) as e:
        _lib.linear(P, 2 * P, P, 8, 16, 24, trans_b=True)
    assert e.value.code == _lib.ERR_ALIAS
    with pytest.raises(KeyError):
        _lib.linear(P, 2 * P, 3 * P, 8, 16, 24, activation="tanh")
    with pytest.raises(_lib.TforgeError):
        _lib.rms_norm(P, P, 8, 16, 1e-5)


def test_forced_kernel_values():
    f = _lib.lib().tforge_debug_linear_kernel
    assert f(1, 48, 1) == _lib.ERR_MODE
    assert f(1, 64, 3) == _lib.ERR_MODE
    assert f(9, 0, 0) == _lib.ERR_MODE
    assert f(0, 0, 0) == _lib.OK


def test_mlp_command_refuses_what_the_block_lacks(capsys):
    from tensorforge_b200 import mlp

    for argv in (["--mode", "fp8"], ["--block", "--mode", "fp32"], ["--block", "--mode", "tf32"], ["--train", "--mode", "bf16"],
                 ["--block", "--mode", "fp8", "--train"]):
        with pytest.raises(SystemExit):
            mlp.main(argv)


@pytest.mark.parametrize("call,dims", [(linear, "MNK"), (backward, "MNK"), (norm, "MN"), (norm_backward, "MN")])
def test_sizes_end_at_two_to_the_thirtieth(call, dims):
    for d in dims:
        assert call(**{d: (1 << 30) + 1}) == _lib.ERR_SHAPE


@pytest.mark.parametrize("call,kw", [
    (linear, dict(ldo=34, ldp=34, pre=5 * P + 2 * 15)),  # pre begins in out's last column
    (linear, dict(ldo=31, ldp=31, pre=5 * P + 2 * 16)),  # pre's last column is out's first of the next row
    (linear, dict(ldo=32, ldp=33, pre=5 * P + 2 * 16)),  # the pitches differ
    (linear, dict(lda=64, ldo=64, out=P + 2 * 23)),
    (linear, dict(lda=64, ldo=64, out=P - 2 * 15)),
    (norm, dict(out_dtype=_lib.BF16, lds=32, ldo=32, out=4 * P + 2 * 17)),
])
def test_slices_of_one_buffer_that_overlap(call, kw):
    assert call(**kw) == _lib.ERR_ALIAS


def test_block_takes_no_weights_outside_a_gpu():
    torch = pytest.importorskip("torch")
    from tensorforge_b200.mlp import FeedForward

    for mode in ("bf16", "fp8"):
        with pytest.raises(ValueError):
            FeedForward(torch.ones(8, 16), torch.ones(16), torch.ones(16, 8), torch.ones(8), torch.ones(8), "silu", mode)
