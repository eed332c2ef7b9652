"""The pitch of an array that a call does not have, or does not use, says nothing."""

import pytest

from tensorforge_b200 import _lib
from tests.test_layer_cpu import backward, linear, norm, norm_backward

BAD = (3, -1, 1 << 62)


# M = 0 (N = 0, nothing wanted) ends each call after its checks of sizes and pitches.
@pytest.mark.parametrize("ld", BAD)
@pytest.mark.parametrize("call,kw,ldname", [
    (linear, dict(M=0, residual=None), "ldr"),
    (linear, dict(M=0, pre=None), "ldp"),
    (backward, dict(dA=None, dB=None, dbias=None), "lda"),
    (backward, dict(dA=None, dB=None, dbias=None), "ldb"),
    (backward, dict(dA=None, dB=None, dbias=None), "ldda"),
    (backward, dict(dA=None, dB=None, dbias=None), "lddb"),
    (backward, dict(dA=None, dB=None, dbias=None, activation=0), "ldp"),
    (norm, dict(M=0, residual=None), "ldr"),
    (norm, dict(M=0, sum_out=None), "lds"),
    (norm_backward, dict(N=0, ds=None), "ldds"),
])
def test_pitches_of_absent_arrays(call, kw, ldname, ld):
    assert call(**kw, **{ldname: ld}) == _lib.OK


@pytest.mark.parametrize("ld", BAD)
@pytest.mark.parametrize("call,kw,ldname", [
    (linear, dict(M=0), "ldr"), (linear, dict(M=0), "ldp"), (backward, {}, "lda"), (backward, {}, "ldb"), (backward, {}, "ldda"),
    (backward, {}, "lddb"), (backward, {}, "ldp"), (norm, dict(M=0), "ldr"), (norm, dict(M=0), "lds"), (norm_backward, {}, "ldds"),
])
def test_pitches_of_those_that_are_there(call, kw, ldname, ld):
    assert call(**kw, **{ldname: ld}) == _lib.ERR_SHAPE
