"""The transformer-layer operators where their approximations, roundings and limits end.

Tolerances are worked out from the roundings on the way, in units of u = 2^-23.
"""

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from tensorforge_b200 import _lib  # noqa: E402
from tests.test_gpu_layer import CODE, TINY, assert_within, block, device, half_step, ptr, rand  # noqa: E402, F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- gelu ---------------------------------------------------------------------------------------------


def phi64(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2))


# Phi(-|z|) = t q(t) exp(-z^2 / 2): the fit 0.7 u, t (a rounding and an approximate reciprocal) 1.5 u, q's
# steps 2.5 u, two products 1 u, ex2.approx 2 u, and the product with z 0.5 u: under 9 u.  The exponent
# z^2 / 2 log2 e has three roundings of half a u, each 2^-24 z^2 / 2 of the value: 0.75 z^2 u.  Phi above 0
# is 1 less a tail, nearer still.
def phi_bound(z):
    return (9 + 0.75 * z * z) * U


@pytest.mark.parametrize("force", [(0, 0, 0), (1, 16, 1), (2, 0, 0)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_gelu_keeps_its_relative_accuracy(force, out):
    """Far below 0 gelu is small, not lost: products of zeros, so that z is the bias."""
    n = 8192
    z = torch.linspace(-12.5, 8, n, device="cuda")
    a, b = torch.zeros(3, 64, device="cuda").bfloat16(), torch.zeros(n, 64, device="cuda").bfloat16()
    y = torch.empty(3, n, device="cuda", dtype=out)
    _lib.check(_lib.lib().tforge_debug_linear_kernel(*force))
    _lib.linear(ptr(a), ptr(b), ptr(y), 3, n, 64, "gelu", ptr(z), out_dtype=CODE[out], trans_b=True, stream=stream())
    z = z.double()
    want = z * phi64(z)
    hs = half_step(out)
    assert_within(y, want.expand(3, n), (phi_bound(z) * (1 + hs) + hs) * want.abs())


def test_gelu_slope_keeps_its_relative_accuracy():
    n = 8192
    z, dout, slope = torch.linspace(-12.5, 8, n, device="cuda"), torch.ones(n, device="cuda"), torch.empty(n, device="cuda")
    _lib.linear_backward(ptr(dout), None, None, 1, n, 8, "gelu", ptr(z), dbias=ptr(slope), dtype=_lib.F32, stream=stream())
    z = z.double()
    p, d = phi64(z), z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    assert_within(slope, p + d, phi_bound(z) * (p + d.abs()))


# ---- rows in 8 bits ----------------------------------------------------------------------------------


def scales(x):
    """The scales of rows of f32 values, and their reciprocals: quotients rounded once, for which 53 bits
    on the way are enough.  (torch divides by a number by multiplying by its reciprocal.)"""
    scale = (x.abs().amax(1).double() / 448).float().clamp_min(TINY)
    return scale, (1 / scale.double()).float()[:, None]


@pytest.mark.parametrize("m,n", [(3001, 1000), (500, 4096), (40, 1111), (3, 20001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantizer_to_the_bit(m, n, dtype):
    """q = e4m3(x (1 / scale)) as documented, the reciprocal and the product rounded to f32."""
    x = rand(m, n, dtype=dtype)
    q, sc = torch.empty(m, n, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(m, device="cuda")
    _lib.quantize_e4m3(ptr(x), ptr(q), ptr(sc), m, n, CODE[dtype], stream=stream())
    scale, inverse = scales(x.float())
    assert torch.equal(sc, scale)
    assert torch.equal(q.float(), (x.float() * inverse).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("m,n", [(3001, 1000), (500, 4096), (40, 1111), (3, 20001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_in_8_bits_to_the_bit(m, n, dtype):
    """The norm's 8-bit rows are those of its f32 rows."""
    x, w = rand(m, n, dtype=dtype), 1 + rand(n, seed=1, scale=0.2)
    q, sc, y = torch.empty(m, n, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(m, device="cuda"), torch.empty(m, n, device="cuda")
    _lib.rms_norm(ptr(x), ptr(q), m, n, 1e-5, ptr(w), scale=ptr(sc), dtype=CODE[dtype], out_dtype=_lib.E4M3, stream=stream())
    _lib.rms_norm(ptr(x), ptr(y), m, n, 1e-5, ptr(w), dtype=CODE[dtype], out_dtype=_lib.F32, stream=stream())
    scale, inverse = scales(y)
    assert torch.equal(sc, scale)
    assert torch.equal(q.float(), (y * inverse).to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("n", [8, 200, 1111, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantizer_poisoned_rows(n, dtype):
    """A NaN or an infinity of either sign makes its own row's scale and values NaN, and no other's."""
    x = rand(7, n, dtype=dtype)
    q, sc = torch.empty(7, n, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(7, device="cuda")
    _lib.quantize_e4m3(ptr(x), ptr(q), ptr(sc), 7, n, CODE[dtype], stream=stream())
    clean, clean_sc = q.float().clone(), sc.clone()
    x[1, n // 2], x[3, n - 1], x[5, 0] = float("nan"), float("inf"), -float("inf")
    _lib.quantize_e4m3(ptr(x), ptr(q), ptr(sc), 7, n, CODE[dtype], stream=stream())
    for i in range(7):
        if i in (1, 3, 5):
            assert bool(sc[i].isnan()) and bool(q[i].float().isnan().all()), i
        else:
            assert torch.equal(q[i].float(), clean[i]) and sc[i] == clean_sc[i]


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


# ---- limits ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("force,k", [((0, 0, 0), 1 << 27), ((1, 16, 1), 1 << 24), ((2, 0, 0), 1 << 24)])
def test_a_sum_may_take_longer_than_the_wait_limit(force, k):
    """The limit is for a step of the work: whoever waits for a whole sum over k gets one for each 2^14
    stages of it (here 131072 a CTA and 262144, over 20 ms)."""
    a, b, out = (torch.ones(r, c, device="cuda", dtype=torch.bfloat16) for r, c in ((1, k), (1, k), (1, 1)))
    L = _lib.lib()
    _lib.check(L.tforge_debug_linear_kernel(*force))
    L.tforge_set_wait_limit_ns(20_000_000)
    try:
        _lib.linear(ptr(a), ptr(b), ptr(out), 1, 1, k, trans_b=True, stream=stream())
        assert _lib.device_status(stream()) == _lib.OK
    finally:
        L.tforge_set_wait_limit_ns(0)
    assert float(out) == k  # a power of two, and so is every partial sum's unit


def test_a_failed_call_leaves_no_error_behind():
    """Scratch that no GPU has (a copy of 2^30 x 512 operands in 1 TB) fails the call before any launch;
    the error is the status and the text, and is not found again by whoever asks CUDA next."""
    args = _lib.LinearArgs(trans_b=1, a_dtype=_lib.F32, b_dtype=_lib.BF16, out_dtype=_lib.BF16, A=1 << 45, B=1 << 20, out=1 << 30,
                           M=1 << 30, N=1, K=512)
    assert _lib.lib().tforge_linear(C.byref(args), stream()) == _lib.ERR_CUDA
    assert b"memory" in _lib.lib().tforge_last_error()
    x = torch.ones(8, device="cuda")
    y = torch.empty_like(x)
    _lib.check(_lib.lib().tforge_add(ptr(x), ptr(x), ptr(y), 1, 8, stream()))
    assert bool((x + y == 3).all())


# ---- the block -----------------------------------------------------------------------------------------


def test_block_refuses_inputs_that_need_a_gradient():
    """autograd does not see the block: an input that needs a gradient would silently get none."""
    m = block(64, 128, "silu", "bf16")
    x, r = rand(4, 64, dtype=torch.bfloat16), rand(4, 64, dtype=torch.bfloat16, seed=1)
    for bad in (lambda: m(x.clone().requires_grad_()), lambda: m(x, r.clone().requires_grad_())):
        with pytest.raises(ValueError):
            bad()
        with torch.no_grad():
            out, _ = bad()
        assert not out.requires_grad
    assert torch.equal(m(x.clone().requires_grad_().detach())[0], m(x)[0])


def test_block_sees_weights_as_documented():
    """bf16 weights and f32 vectors are the caller's own, others copies of what they were."""
    from tensorforge_b200.mlp import FeedForward

    w1, w2 = (torch.nn.Parameter(rand(*s, dtype=torch.bfloat16, scale=0.1)) for s in ((64, 128), (128, 64)))
    b1, b2, g = torch.zeros(128, device="cuda"), torch.zeros(64, device="cuda"), torch.ones(64, device="cuda")
    x = rand(4, 64, dtype=torch.bfloat16)
    own, copied = FeedForward(w1, b1, w2, b2, g, "silu"), FeedForward(w1.float(), b1, w2.float(), b2, g, "silu")
    before = own(x)[0].clone()
    assert torch.equal(copied(x)[0], before) and not before.requires_grad
    with torch.no_grad():
        w1.mul_(2)
    assert not torch.equal(own(x)[0], before) and torch.equal(copied(x)[0], before)


def test_block_gradient_is_captured_with_its_call():
    """What an eager call kept is given back once its gradient is done: a graph of the gradient alone would
    read it after that, and an eager gradient what a capture has not yet made."""
    m = block(64, 128, "silu", "bf16")
    x, dout = rand(4, 64, dtype=torch.bfloat16), rand(4, 64, dtype=torch.bfloat16, seed=1)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        m(x, keep=True)
        want = {k: v.clone() for k, v in m.backward(dout).items()}
        m(x, keep=True)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with pytest.raises(ValueError):
            with torch.cuda.graph(g, stream=st):
                m.backward(dout)
        got = m.backward(dout)  # what was kept is still there
        assert all(torch.equal(got[k], want[k]) for k in want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            m(x, keep=True)
        with pytest.raises(ValueError):
            m.backward(dout)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=st):
            m(x, keep=True)
            m.backward(dout)
        st.synchronize()


@pytest.mark.parametrize("argv", [["--mode", "bf16", "--train"], ["--mode", "bf16"], ["--mode", "fp8"]])
@pytest.mark.parametrize("shape", ["300x256x512", "5x136x264"])
def test_block_command_checks_what_it_times(argv, shape, capsys):
    import json

    from tensorforge_b200 import mlp

    assert mlp.main(["--block", "--shape", shape, "--steps", "2", "--warmup", "1", *argv]) == 0
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["pass"] and line["rel_err"] <= line["rel_err_bound"]
    checked = {"dx", "dw1", "db1", "dw2", "db2", "dnorm_weight"} if "--train" in argv else set()
    assert set(line.get("gradient_rel_err", {})) == checked
