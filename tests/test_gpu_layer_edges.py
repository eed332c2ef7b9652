"""The transformer-layer operators where their approximations, roundings and limits end.

Tolerances are worked out from the roundings on the way, in units of u = 2^-23.
"""

import pytest

torch = pytest.importorskip("torch")

from tensorforge_b200 import _lib  # noqa: E402
from tests.test_gpu_layer import CODE, assert_within, device, half_step, ptr, rand  # noqa: E402, F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- one call after the other ------------------------------------------------------------------------


@pytest.mark.parametrize("m,n,k", [(40, 263, 135), (300, 519, 1001), (130, 264, 136), (1025, 1031, 517)])
@pytest.mark.parametrize("operands", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bias", [True, False])
def test_gradients_in_a_chain(m, n, k, operands, bias):
    """The first layer's dA is the second's dout, so its passes and operand copies follow products that
    have just begun to end; the inputs change from round to round by powers of two, which go through
    without a rounding."""
    st = stream()
    first, pre = rand(m, n, dtype=torch.bfloat16), rand(m, n, dtype=torch.bfloat16, seed=1)
    pre2 = rand(m, k, dtype=torch.bfloat16, seed=2)
    w1, w2 = rand(n, k, dtype=operands, seed=3, scale=1 / 16), rand(k, n, dtype=operands, seed=4, scale=1 / 16)
    a1, a2 = rand(m, k, dtype=operands, seed=5), rand(m, n, dtype=operands, seed=6)
    dout, x1, x2 = torch.empty_like(first), torch.empty_like(a1), torch.empty_like(a2)
    d1, d2, g1, g2 = (torch.empty_like(t, dtype=torch.bfloat16) for t in (a1, a2, w1, w2))
    s1, s2 = torch.empty(n, device="cuda"), torch.empty(k, device="cuda")
    outs = []
    for i in range(12):
        f = 2.0 ** (i % 5)
        torch.mul(first, f, out=dout)
        torch.mul(a1, f, out=x1)
        torch.mul(a2, f, out=x2)
        for t in (d1, d2, g1, g2, s1, s2):
            t.zero_()
        _lib.linear_backward(ptr(dout), ptr(x1), ptr(w1), m, n, k, "relu", ptr(pre), dA=ptr(d1), dB=ptr(g1),
                             dbias=ptr(s1) if bias else None, a_dtype=CODE[operands], b_dtype=CODE[operands], trans_b=True, stream=st)
        _lib.linear_backward(ptr(d1), ptr(x2), ptr(w2), m, k, n, "relu", ptr(pre2), dA=ptr(d2), dB=ptr(g2),
                             dbias=ptr(s2) if bias else None, a_dtype=CODE[operands], b_dtype=CODE[operands], trans_b=True, stream=st)
        outs.append([d1 / f, d2 / f, g1 / f ** 2, g2 / f ** 2, s1 / f, s2 / f])
    for o in outs[1:]:
        for got, want in zip(o, outs[0]):
            assert torch.equal(got, want)
    dz = torch.where(pre > 0, first, torch.zeros_like(first)).double()
    w = w1.bfloat16().double()
    want, mag = dz @ w, dz.abs() @ w.abs()
    assert_within(outs[0][0], want, half_step(torch.bfloat16) * want.abs() + 1.01 * (n + 4) * U * mag)
    dz2 = torch.where(pre2 > 0, outs[0][0], torch.zeros_like(outs[0][0])).double()
    w = w2.bfloat16().double()
    want, mag = dz2 @ w, dz2.abs() @ w.abs()
    assert_within(outs[0][1], want, half_step(torch.bfloat16) * want.abs() + 1.01 * (k + 4) * U * mag)


def test_gradients_and_norms_repeat_themselves():
    """The same inputs give the same bits."""
    m, n, k = 300, 519, 1001
    dout, a, b = rand(m, n, dtype=torch.bfloat16), rand(m, k, dtype=torch.bfloat16, seed=1), rand(n, k, dtype=torch.bfloat16, seed=2)
    da, db, dbias = torch.empty_like(a), torch.empty_like(b), torch.empty(n, device="cuda")
    q, sc, rstd = torch.empty(m, k, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    dx, dw = torch.empty_like(a), torch.empty(k, device="cuda")
    first = None
    for _ in range(6):
        _lib.linear_backward(ptr(dout), ptr(a), ptr(b), m, n, k, "silu", ptr(dout), ptr(da), ptr(db), ptr(dbias), trans_b=True, stream=stream())
        _lib.rms_norm(ptr(a), ptr(q), m, k, 1e-5, rstd=ptr(rstd), scale=ptr(sc), out_dtype=_lib.E4M3, stream=stream())
        _lib.rms_norm_backward(ptr(da), ptr(a), ptr(rstd), ptr(dx), m, k, dweight=ptr(dw), stream=stream())
        got = [t.clone() for t in (da, db, dbias, q.view(torch.uint8), sc, rstd, dx, dw)]
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(got, first))
