"""The transformer-layer operators on the GPU against their definitions in 64 bits.

Tolerances are worked out, not fitted.  Products of bf16 or e4m3 values are exact in f32, so a sum of
K of them is off by at most about K 2^-23 times the sum of their absolute values (2^-23: a tensor core
may cut instead of rounding).  exp, erf and the fast divide are within a few units of 2^-23, which
leaves an activation off by at most 2^-20 |z|.  Each output adds half a step of its type
(torch.finfo(t).eps / 2).
"""

import math

import pytest

torch = pytest.importorskip("torch")

from tensorforge_b200 import _lib  # noqa: E402

pytestmark = pytest.mark.gpu

CODE = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float8_e4m3fn: _lib.E4M3}
TINY = 2.0 ** -126
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(autouse=True)
def device(gpu):
    yield
    _lib.check(_lib.lib().tforge_debug_linear_kernel(0, 0, 0))
    assert _lib.device_status(torch.cuda.current_stream().cuda_stream) == 0


def half_step(t):
    return torch.finfo(t).eps / 2


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0, pad=0, shift=0):
    """Normal values as a matrix with `pad` more columns a row in memory and `shift` elements off the
    allocation's start; what lies between the rows is NaN."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 1000 * len(shape) + sum(shape))
    v = (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)
    if not pad and not shift:
        return v
    rows, cols = shape
    whole = torch.full((rows * (cols + pad) + shift,), float("nan"), device="cuda").to(dtype)
    out = whole[shift:].view(rows, cols + pad)[:, :cols]
    out.copy_(v)
    return out


def out_like(rows, cols, dtype, pad=0, shift=0):
    """An output matrix whose gaps hold a sentinel, and the check that nothing wrote there."""
    whole = torch.full((rows * (cols + pad) + shift + 64,), 7.0, device="cuda").to(dtype)
    out = whole[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]

    def untouched():
        probe = whole.float().clone()
        probe[shift:shift + rows * (cols + pad)].view(rows, cols + pad)[:, :cols] = 7.0
        assert bool((probe == 7.0).all()), "wrote outside the output"

    return out, untouched


def ptr(t):
    return None if t is None else t.data_ptr()


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        p = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z ** 2)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, torch.ones_like(z)


def quantize64(x):
    scale = (x.abs().amax(1) / 448).clamp(min=TINY)
    return (x / scale[:, None]), scale


class Linear:
    """One call of tforge_linear with its expected outputs and their bounds."""

    def __init__(self, m, n, k, dtype=torch.bfloat16, act="none", bias=True, residual=None, out=torch.bfloat16, pre=False,
                 trans_b=True, pad=0, shift=0, seed=0):
        self.dims, self.act, self.trans_b, self.out_dtype = (m, n, k), act, trans_b, out
        self.a_scale = self.b_scale = None
        if dtype == torch.float8_e4m3fn:
            self.a = rand(m, k, seed=seed, scale=60, pad=pad, shift=shift).to(dtype)
            b = rand(n, k, seed=seed + 1, scale=60).to(dtype)
            if pad or shift:  # 8-bit copies keep their gaps by hand
                whole = torch.zeros(m * (k + pad) + shift, device="cuda").to(dtype)
                v = whole[shift:].view(m, k + pad)[:, :k]
                v.copy_(self.a)
                self.a = v
            self.b = b
            self.a_scale = rand(m, seed=3).abs() * 0.01 + 1e-3
            self.b_scale = rand(n, seed=4).abs() * 0.01 / math.sqrt(max(k, 1)) + 1e-5
        else:
            self.a = rand(m, k, dtype=dtype, seed=seed, pad=pad, shift=shift)
            shape = (n, k) if trans_b else (k, n)
            self.b = rand(*shape, dtype=dtype, seed=seed + 1, scale=1 / math.sqrt(max(k, 1)), pad=pad, shift=shift)
        self.bias = rand(n, seed=5) if bias else None
        self.residual = rand(m, n, dtype=residual, seed=6, pad=pad, shift=shift) if residual is not None else None
        self.out, self.out_ok = out_like(m, n, out, pad, shift)
        self.pre, self.pre_ok = out_like(m, n, out, pad, shift) if pre else (None, lambda: None)

    def call(self, stream=None):
        m, n, k = self.dims
        ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
        _lib.linear(ptr(self.a), ptr(self.b), ptr(self.out), m, n, k, self.act, ptr(self.bias), ptr(self.residual),
                    ptr(self.pre), ptr(self.a_scale), ptr(self.b_scale), CODE[self.a.dtype], CODE[self.b.dtype],
                    CODE[self.out_dtype], CODE[self.residual.dtype] if self.residual is not None else _lib.BF16,
                    self.trans_b, ld(self.a), ld(self.b), ld(self.residual), ld(self.out), ld(self.pre),
                    stream if stream is not None else torch.cuda.current_stream().cuda_stream)
        return self

    def check(self):
        m, n, k = self.dims
        a, b = self.a, self.b
        if a.dtype == torch.float32:
            a, b = a.bfloat16(), b.bfloat16()
        a, b = a.double(), (b.double().T if self.trans_b else b.double())
        z, mag = a @ b, a.abs() @ b.abs()
        if self.a_scale is not None:
            f = self.a_scale.double()[:, None] * self.b_scale.double()
            z, mag = z * f, mag * f
        bias = self.bias.double() if self.bias is not None else torch.zeros(n, device="cuda", dtype=torch.float64)
        z = z + bias
        ez = (k + 4) * 2.0 ** -23 * mag + 2.0 ** -23 * (z.abs() + bias.abs())
        y = act64(z, self.act)[0]
        ey = 1.13 * ez + 2.0 ** -20 * z.abs()  # 1.13: the largest slope of any of the activations
        if self.residual is not None:
            y = y + self.residual.double()
            ey = ey + 2.0 ** -23 * (y.abs() + self.residual.double().abs())
        hs = half_step(self.out_dtype)
        assert_within(self.out, y, ey * (1 + hs) + hs * y.abs())
        self.out_ok()
        if self.pre is not None:
            assert_within(self.pre, z, ez * (1 + hs) + hs * z.abs())
            self.pre_ok()


def assert_within(got, want, bound):
    over = (got.double() - want).abs() - bound - 1e-300
    assert bool(torch.isfinite(got.float()).all())
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, f"off by {worst} more than the bound at {int(over.argmax())}"


# ---- the linear layer ---------------------------------------------------------------------------


@pytest.mark.parametrize("m,n,k", [(1, 128, 64), (1, 4096, 512), (3, 7, 5), (16, 200, 129), (17, 128, 256), (33, 257, 200),
                                   (64, 384, 640), (100, 130, 72), (129, 1000, 90), (257, 513, 320), (600, 300, 65)])
@pytest.mark.parametrize("trans_b", [True, False])
def test_linear_shapes(m, n, k, trans_b):
    Linear(m, n, k, act="gelu", residual=torch.bfloat16, trans_b=trans_b).call().check()


@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (2, 9, 3), (16, 1024, 272), (31, 130, 640), (130, 70, 400), (300, 520, 144)])
def test_linear_e4m3(m, n, k):
    Linear(m, n, k, torch.float8_e4m3fn, "silu", residual=torch.bfloat16).call().check()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_linear_activations(act, out, dtype):
    Linear(40, 136, 192, dtype, act, residual=torch.float32, out=out, pre=True).call().check()


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("residual", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("m", [5, 300])
def test_linear_parts(bias, residual, pre, m):
    Linear(m, 264, 128, act="gelu_tanh", bias=bias, residual=residual, pre=pre).call().check()


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (5, 3), (16, 8)])
@pytest.mark.parametrize("m", [4, 200, 500])
@pytest.mark.parametrize("trans_b", [True, False])
def test_linear_pitches_and_offsets(pad, shift, m, trans_b):
    Linear(m, 272, 160, act="relu", residual=torch.bfloat16, pre=True, trans_b=trans_b, pad=pad, shift=shift).call().check()


@pytest.mark.parametrize("pad,shift", [(16, 0), (1, 0), (0, 5)])
def test_linear_e4m3_pitches(pad, shift):
    Linear(50, 144, 160, torch.float8_e4m3fn, "relu", pad=pad, shift=shift).call().check()


def test_linear_f32_operands():
    Linear(70, 136, 96, torch.float32, "gelu", residual=torch.float32, out=torch.float32).call().check()
    Linear(7, 33, 21, torch.float32, "none", trans_b=False, out=torch.float32).call().check()


@pytest.mark.parametrize("m,n", [(1, 1), (3, 130), (300, 520)])
def test_linear_without_k(m, n):
    """K = 0: z is the bias alone."""
    Linear(m, n, 0, act="silu", residual=torch.bfloat16, pre=True).call().check()


def test_linear_in_place_on_the_residual():
    for m in (4, 400):
        c = Linear(m, 320, 128, act="none", residual=torch.bfloat16)
        c.out.copy_(c.residual)
        want = c.residual.clone()
        c.residual = c.out
        c.call()
        c.residual = want
        c.check()


@pytest.mark.parametrize("tile,splits", [(16, 1), (16, 2), (16, 4), (16, 8), (32, 1), (32, 4), (64, 1), (64, 8), (128, 1),
                                         (128, 2), (256, 1), (256, 4), (256, 8)])
@pytest.mark.parametrize("dtype,trans_b", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float8_e4m3fn, True)])
def test_linear_one_cta_kernel(tile, splits, dtype, trans_b):
    """Every tile and split, with fewer and with more stages of k than CTAs that share a tile."""
    _lib.check(_lib.lib().tforge_debug_linear_kernel(1, tile, splits))
    Linear(150, 260, 900, dtype, "gelu", residual=torch.bfloat16, pre=True, trans_b=trans_b).call().check()
    Linear(9, 140, 70, dtype, "gelu", residual=torch.float32, out=torch.float32, trans_b=trans_b).call().check()


@pytest.mark.parametrize("dtype,trans_b", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float8_e4m3fn, True)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pre", [True, False])
@pytest.mark.parametrize("pad,shift", [(0, 0), (16, 0), (3, 1)])
def test_linear_pair_kernel(dtype, trans_b, out, pre, pad, shift):
    """The 256 x 256 kernel, with tiles that end inside the matrix and fewer stages of k than its ring."""
    _lib.check(_lib.lib().tforge_debug_linear_kernel(2, 0, 0))
    Linear(300, 520, 200, dtype, "gelu", residual=out, out=out, pre=pre, trans_b=trans_b, pad=pad, shift=shift).call().check()
    Linear(5, 40, 1000, dtype, "silu", out=out, pre=pre, trans_b=trans_b, pad=pad, shift=shift).call().check()
    Linear(300, 520, 4500, dtype, "gelu", residual=out, out=out, pre=pre, trans_b=trans_b, pad=pad, shift=shift).call().check()


@pytest.mark.parametrize("dtype,trans_b", [(torch.bfloat16, False), (torch.float8_e4m3fn, True)])
def test_linear_pair_kernel_walks_tiles(dtype, trans_b):
    """More tiles than CTA pairs: both accumulators in turn, the ring across tiles."""
    _lib.check(_lib.lib().tforge_debug_linear_kernel(2, 0, 0))
    c = Linear(2570, 5200, 136, dtype, "relu", residual=torch.bfloat16, trans_b=trans_b).call()
    c.check()
    first = c.out.clone()
    assert torch.equal(c.call().out, first)


@pytest.mark.parametrize("trans_b", [True, False])
def test_linear_backward_pair_kernel(trans_b):
    _lib.check(_lib.lib().tforge_debug_linear_kernel(2, 0, 0))
    check_linear_backward(300, 520, 264, trans_b=trans_b)
    check_linear_backward(77, 131, 65, trans_b=trans_b, grad=torch.float32)


@pytest.mark.parametrize("force", [(0, 0, 0), (1, 16, 2), (1, 64, 8), (2, 0, 0)])
@pytest.mark.parametrize("trans_b", [True, False])
def test_linear_f32_output_of_a_long_k(force, trans_b):
    """The tensor core cuts each addition to an f32 accumulator, 2^-23 of it at most, and adds 16
    products at a time.  An f32 output is off by no more than a piece of 768 can be (48 additions) and
    the joining of the pieces, where one sum over 16384 would be 1.9e-5 off."""
    m, n, k = 40, 264, 16384
    _lib.check(_lib.lib().tforge_debug_linear_kernel(*force))
    c = Linear(m, n, k, bias=False, out=torch.float32, trans_b=trans_b, pre=True, residual=torch.float32).call()
    want = c.a.double() @ (c.b.double().T if trans_b else c.b.double())
    bound = 48 * 2.0 ** -23 + 22 * 2.0 ** -24
    assert float((c.pre.double() - want).norm()) <= bound * float(want.norm())
    want = want + c.residual.double()
    assert float((c.out.double() - want).norm()) <= bound * float(want.norm())


def test_linear_backward_f32_gradients_of_a_long_batch():
    """The same for the gradients' products: dB sums over the batch."""
    m, n, k = 12000, 72, 136
    a, dout = rand(m, k, dtype=torch.bfloat16), rand(m, n, dtype=torch.bfloat16, seed=1)
    db = torch.empty(n, k, device="cuda")
    for force in ((0, 0, 0), (2, 0, 0)):
        _lib.check(_lib.lib().tforge_debug_linear_kernel(*force))
        _lib.linear_backward(ptr(dout), ptr(a), None, m, n, k, dB=ptr(db), grad_dtype=_lib.F32, trans_b=True,
                             stream=torch.cuda.current_stream().cuda_stream)
        want = dout.double().T @ a.double()
        assert float((db.double() - want).norm()) <= (48 * 2.0 ** -23 + 22 * 2.0 ** -24) * float(want.norm())


def test_linear_infinities_and_nan():
    """An infinite operand reaches its row as the formula says; the other rows do not see it."""
    c = Linear(20, 96, 64, act="relu", out=torch.float32)
    clean = c.call().out.clone()
    c.a[7, 3] = float("inf")
    c.a[9, 5] = float("nan")
    c.call()
    keep = [i for i in range(20) if i not in (7, 9)]
    assert torch.equal(c.out[keep], clean[keep])
    assert bool(c.out[9].isnan().all())
    want = torch.where(c.b[:, 3] > 0, float("inf"), 0.0)
    assert torch.equal(c.out[7], want.float())


def test_linear_same_bits_every_time():
    for m, n, k in ((8, 512, 2048), (300, 512, 640)):
        c = Linear(m, n, k, act="gelu", residual=torch.bfloat16)
        first = c.call().out.clone()
        for _ in range(5):
            assert torch.equal(c.call().out, first)


# ---- its gradient -------------------------------------------------------------------------------


def check_linear_backward(m, n, k, act="gelu", trans_b=True, dtype=torch.bfloat16, grad=torch.bfloat16, pad=0, shift=0,
                          wants="ABb", op=torch.bfloat16):
    a = rand(m, k, dtype=op, pad=pad, shift=shift)
    b = rand(*((n, k) if trans_b else (k, n)), dtype=op, seed=1, scale=1 / math.sqrt(k), pad=pad, shift=shift)
    dout = rand(m, n, dtype=dtype, seed=2, pad=pad, shift=shift)
    pre = rand(m, n, dtype=dtype, seed=3, scale=1.5, pad=pad, shift=shift)
    da, da_ok = out_like(m, k, grad, pad, shift)
    db, db_ok = out_like(*b.shape, grad, pad, shift)
    dbias = torch.full((n,), 7.0, device="cuda")
    ld = lambda t: t.stride(0)  # noqa: E731
    _lib.linear_backward(ptr(dout), ptr(a), ptr(b), m, n, k, act, ptr(pre) if act != "none" else None,
                         ptr(da) if "A" in wants else None, ptr(db) if "B" in wants else None,
                         ptr(dbias) if "b" in wants else None, CODE[op], CODE[op], CODE[dtype], CODE[grad], trans_b, ld(dout),
                         ld(pre), ld(a), ld(b), ld(da), ld(db), torch.cuda.current_stream().cuda_stream)
    dz = dout.double() * act64(pre.double(), act)[1]
    # The slope is off by at most 2^-20 (1 + |z|); dz is rounded to bf16 before the products.
    edz = 2.0 ** -20 * dout.double().abs() * (1 + pre.double().abs())
    ez = edz + half_step(torch.bfloat16) * (dz.abs() + edz)
    a64, b64 = a.bfloat16().double(), b.bfloat16().double() if trans_b else b.bfloat16().double().T
    hs = half_step(grad)
    if "A" in wants:
        want, mag = dz @ b64, dz.abs() @ b64.abs()
        e = ez @ b64.abs() + (n + 4) * 2.0 ** -23 * mag
        assert_within(da, want, e * (1 + hs) + hs * want.abs())
    if "B" in wants:
        want, mag = dz.T @ a64, dz.abs().T @ a64.abs()
        e = ez.T @ a64.abs() + (m + 4) * 2.0 ** -23 * mag
        if not trans_b:
            want, e = want.T, e.T
        assert_within(db, want, e * (1 + hs) + hs * want.abs())
    if "b" in wants:
        assert_within(dbias, dz.sum(0), edz.sum(0) + (m + 4) * 2.0 ** -23 * dz.abs().sum(0))
    da_ok()
    db_ok()
    for t, w in ((da, "A"), (db, "B"), (dbias, "b")):
        if w not in wants:
            assert bool((t == 7.0).all())


@pytest.mark.parametrize("m,n,k", [(1, 8, 16), (5, 7, 3), (64, 128, 192), (130, 264, 72), (300, 65, 520), (513, 300, 257)])
@pytest.mark.parametrize("trans_b", [True, False])
def test_linear_backward_shapes(m, n, k, trans_b):
    check_linear_backward(m, n, k, trans_b=trans_b)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_backward_activations(act, dtype):
    check_linear_backward(96, 136, 80, act, dtype=dtype, grad=dtype)


@pytest.mark.parametrize("wants", ["A", "B", "b", "AB", "Ab", "Bb"])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_linear_backward_parts(wants, act):
    check_linear_backward(70, 136, 80, act, wants=wants)


@pytest.mark.parametrize("pad,shift", [(8, 0), (3, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("act", ["none", "gelu_tanh"])
@pytest.mark.parametrize("trans_b", [True, False])
def test_linear_backward_pitches(pad, shift, act, trans_b):
    check_linear_backward(90, 136, 80, act, trans_b, pad=pad, shift=shift)


def test_linear_backward_f32_operands():
    check_linear_backward(90, 136, 80, op=torch.float32, dtype=torch.float32, grad=torch.float32)


def test_linear_backward_of_nothing():
    """No rows: dB and dbias are zeros; no columns: dA is."""
    s = torch.cuda.current_stream().cuda_stream
    db, dbias = torch.full((24, 16), 7.0, device="cuda"), torch.full((16,), 7.0, device="cuda")
    _lib.linear_backward(None, None, None, 0, 16, 24, dB=ptr(db), dbias=ptr(dbias), grad_dtype=_lib.F32, stream=s)
    assert not db.any() and not dbias.any()
    da = torch.full((5, 24), 7.0, device="cuda")
    _lib.linear_backward(None, None, None, 5, 0, 24, dA=ptr(da), grad_dtype=_lib.F32, stream=s)
    assert not da.any()


@pytest.mark.parametrize("act", ACTS[1:])
def test_linear_backward_against_differences(act):
    """The gradient of sum(out * w) by central differences of the 64-bit definition, at places away
    from the rectifier's corner."""
    m, n, k = 6, 16, 8
    a, b = rand(m, k, dtype=torch.bfloat16), rand(n, k, dtype=torch.bfloat16, seed=1)
    bias = rand(n, seed=2)
    w = rand(m, n, seed=3)
    z = a.double() @ b.double().T + bias.double()
    z = torch.where(z.abs() < 0.05, z + 0.1, z)
    pre = z.float()
    da = torch.empty(m, k, device="cuda")
    _lib.linear_backward(ptr(w), ptr(a), ptr(b), m, n, k, act, ptr(pre), dA=ptr(da), dtype=_lib.F32, grad_dtype=_lib.F32,
                         trans_b=True, stream=torch.cuda.current_stream().cuda_stream)
    h = 1e-4
    for i in range(k):
        step = h * b.double()[:, i]
        d = ((act64(z + step, act)[0] - act64(z - step, act)[0]) * w.double()).sum(1) / (2 * h)
        mag = (w.double().abs() * b.double()[:, i].abs()).sum(1)
        # bf16 dz: half a step of each term (slopes up to 1.13); the differences themselves are 1e-7 off.
        assert bool(((da[:, i].double() - d).abs() <= 1.2 * mag * half_step(torch.bfloat16)).all())


# ---- the norm -----------------------------------------------------------------------------------


WIDTHS = [1, 7, 8, 32, 200, 256, 257, 264, 1000, 1024, 1111, 2048, 2056, 4096, 4100, 8192, 8200, 16384, 16392, 20001, 32760, 32770, 40000]


def check_rms_norm(m, n, dtype=torch.bfloat16, out=torch.bfloat16, residual=True, weight=torch.float32, pad=0, shift=0,
                   eps=1e-5, scale=1.0, in_place=""):
    x = rand(m, n, dtype=dtype, pad=pad, shift=shift, scale=scale)
    r = rand(m, n, dtype=dtype, seed=1, pad=pad, shift=shift, scale=scale) if residual else None
    if m > 2:
        x[1] = 0  # a padded row
        if residual:
            r[1] = 0
    w = rand(n, seed=2).to(weight) if weight is not None else None
    s64 = x.double() + (r.double() if residual else 0.0)
    y, y_ok = out_like(m, n, out, pad, shift)
    so, so_ok = out_like(m, n, dtype, pad, shift)
    if in_place:
        so, so_ok = {"x": x, "residual": r}[in_place], lambda: None
    sc, rstd = torch.full((m,), 7.0, device="cuda"), torch.full((m,), 7.0, device="cuda")
    ld = lambda t: t.stride(0)  # noqa: E731
    _lib.rms_norm(ptr(x), ptr(y), m, n, eps, ptr(w), ptr(r), ptr(so), ptr(rstd), ptr(sc) if out == torch.float8_e4m3fn else None,
                  CODE[dtype], CODE[weight] if weight is not None else _lib.F32, CODE[out], ld(x), ld(r) if residual else 0, ld(so),
                  ld(y), torch.cuda.current_stream().cuda_stream)
    # f32: the sum one rounding (2^-24), the mean of squares at most 2^-23 n off in theory and
    # 2^-23 (n / 32 + 40) with 32 or more partial sums; its root halves that.
    r64 = (s64.square().mean(1) + eps).rsqrt()
    er = 2.0 ** -23 * (n / 64 + 24)
    y64 = s64 * r64[:, None] * (w.double() if w is not None else 1.0)
    ey = (er + 2.0 ** -22) * y64.abs()
    assert_within(rstd, r64, er * r64)
    assert_within(so, s64, (half_step(dtype) + 2.0 ** -23) * s64.abs())
    if out == torch.float8_e4m3fn:
        s8 = (y64.abs().amax(1) / 448).clamp(min=TINY)
        assert_within(sc, s8, (er + 2.0 ** -21) * s8)
        v = y64 / s8[:, None]
        # Half a step of 2^-4 relative, or of the smallest step 2^-9 (2^-10), from where the exact value may lie.
        assert_within(y.float(), v, 2 * (er + 2.0 ** -21) * v.abs() * (1 + 2.0 ** -4) + torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10))
        assert bool((sc > 0).all())
    else:
        hs = half_step(out)
        assert_within(y, y64, ey * (1 + hs) + hs * y64.abs())
    y_ok()
    so_ok()


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float8_e4m3fn])
def test_rms_norm_widths(n, out):
    check_rms_norm(11, n, out=out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("weight", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [200, 1111])
def test_rms_norm_types(dtype, out, residual, weight, n):
    check_rms_norm(9, n, dtype, out, residual, weight)


@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1), (7, 5)])
@pytest.mark.parametrize("out", [torch.float32, torch.float8_e4m3fn])
@pytest.mark.parametrize("n", [264, 20008])
def test_rms_norm_pitches(pad, shift, out, n):
    check_rms_norm(6, n, out=out, pad=pad, shift=shift)


@pytest.mark.parametrize("where", ["x", "residual"])
@pytest.mark.parametrize("n", [264, 1111, 20008])
def test_rms_norm_sum_in_place(where, n):
    check_rms_norm(5, n, out=torch.float8_e4m3fn, in_place=where)


@pytest.mark.parametrize("m", [1, 7, 8, 9, 1000])
def test_rms_norm_rows(m):
    check_rms_norm(m, 128, out=torch.float8_e4m3fn)
    check_rms_norm(m, 1024)


# Several rows a block of the gradient at every width class, the last round only partly filled.
MANY = [(19000, 264), (19003, 300), (20001, 511), (5000, 1024), (5003, 1111), (5000, 2048), (2400, 4096), (2401, 4099),
        (1200, 5001), (1300, 8192), (700, 10007), (600, 16384)]


@pytest.mark.parametrize("m,n", MANY)
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn),
                                       (torch.float32, torch.float32)])
def test_rms_norm_many_rows(m, n, dtype, out):
    check_rms_norm(m, n, dtype, out)
    check_rms_norm(m, n, dtype, out, residual=False, pad=3, shift=1)


@pytest.mark.parametrize("pad,shift", [(8, 8), (1, 0), (0, 1), (7, 5), (2, 4)])
@pytest.mark.parametrize("m,n", [(19003, 300), (5003, 1111)])
def test_rms_norm_many_rows_pitches(m, n, pad, shift):
    for where in ("", "x", "residual"):
        check_rms_norm(m, n, torch.bfloat16, torch.float8_e4m3fn, pad=pad, shift=shift, in_place=where)
    check_rms_norm_backward(m, n, pad=pad, shift=shift)
    check_rms_norm_backward(m, n, pad=pad, shift=shift, in_place=True)


@pytest.mark.parametrize("m,n", MANY)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rms_norm_backward_many_rows(m, n, dtype):
    check_rms_norm_backward(m, n, dtype)
    check_rms_norm_backward(m, n, dtype, ds=False, dweight=False, pad=3, shift=1)


@pytest.mark.parametrize("m,n", [(70, 16), (33, 64), (100, 72), (17, 128), (4099, 40)])
def test_rms_norm_narrow_rows(m, n):
    """Several rows a warp, the last warp only partly filled."""
    check_rms_norm(m, n, out=torch.float8_e4m3fn)
    check_rms_norm(m, n, torch.float32, torch.float32)
    check_rms_norm_backward(m, n)
    check_rms_norm_backward(m, n, torch.float32)


def test_quantize_many_rows():
    for m, n, dtype in ((19003, 300, torch.bfloat16), (2401, 4096, torch.float32)):
        x = rand(m, n, dtype=dtype)
        q, sc = torch.empty(m, n, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(m, device="cuda")
        _lib.quantize_e4m3(ptr(x), ptr(q), ptr(sc), m, n, CODE[dtype], stream=torch.cuda.current_stream().cuda_stream)
        v, s64 = quantize64(x.double())
        assert_within(sc, s64, 2.0 ** -24 * s64)
        assert_within(q.float(), v, v.abs() * (2.0 ** -21) + torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10))


def test_linear_waits_are_bounded():
    L, s = _lib.lib(), torch.cuda.current_stream().cuda_stream
    L.tforge_set_wait_limit_ns(20_000_000)
    try:
        for force in ((1, 16, 1), (1, 64, 4), (2, 0, 0)):
            for dtype, trans_b in ((torch.bfloat16, False), (torch.float8_e4m3fn, True)):
                _lib.check(L.tforge_debug_linear_kernel(*force))
                c = Linear(300, 520, 640, dtype, "gelu", trans_b=trans_b)
                L.tforge_debug_skip_load(1)
                c.call()
                assert _lib.device_status(s) == _lib.ERR_TIMEOUT
                L.tforge_debug_skip_load(0)
                c.call().check()
    finally:
        L.tforge_debug_skip_load(0)
        L.tforge_set_wait_limit_ns(0)


@pytest.mark.parametrize("scale", [1e-12, 1e-4, 1e4, 1e12])
def test_rms_norm_magnitudes(scale):
    check_rms_norm(5, 520, torch.float32, torch.float32, scale=scale)
    check_rms_norm(5, 520, torch.float32, torch.float8_e4m3fn, scale=scale)


def test_rms_norm_poisoned_rows():
    """A NaN or an infinity makes its own row's scale and values NaN (8 bits), and no other's."""
    for n in (200, 1111, 20001):
        x = rand(6, n, dtype=torch.bfloat16)
        q, sc = torch.zeros(6, n, device="cuda").to(torch.float8_e4m3fn), torch.zeros(6, device="cuda")
        s = torch.cuda.current_stream().cuda_stream
        args = dict(scale=ptr(sc), out_dtype=_lib.E4M3, stream=s)
        _lib.rms_norm(ptr(x), ptr(q), 6, n, 1e-5, **args)
        clean, clean_sc = q.float().clone(), sc.clone()
        x[2, n // 2], x[4, n - 1] = float("nan"), float("inf")
        _lib.rms_norm(ptr(x), ptr(q), 6, n, 1e-5, **args)
        for i in range(6):
            if i in (2, 4):
                assert bool(sc[i].isnan()) and bool(q[i].float().isnan().all())
            else:
                assert torch.equal(q[i].float(), clean[i]) and sc[i] == clean_sc[i]


@pytest.mark.parametrize("m,n", [(1, 1), (5, 7), (9, 200), (300, 264), (64, 1111), (40, 4096), (7, 20001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize(m, n, dtype):
    for pad, shift in ((0, 0), (8, 0), (3, 1)):
        x = rand(m, n, dtype=dtype, pad=pad, shift=shift)
        if m > 2:
            x[1] = 0
        q, q_ok = out_like(m, n, torch.float8_e4m3fn, pad, shift)
        sc = torch.empty(m, device="cuda")
        _lib.quantize_e4m3(ptr(x), ptr(q), ptr(sc), m, n, CODE[dtype], x.stride(0), q.stride(0),
                           torch.cuda.current_stream().cuda_stream)
        v, s64 = quantize64(x.double())
        assert_within(sc, s64, 2.0 ** -24 * s64)
        assert_within(q.float(), v, v.abs() * (2.0 ** -21) + torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10))
        q_ok()


# ---- the norm's gradient ------------------------------------------------------------------------


def check_rms_norm_backward(m, n, dtype=torch.bfloat16, ds=True, weight=torch.float32, dweight=True, pad=0, shift=0, in_place=False):
    s, dy = rand(m, n, dtype=dtype, pad=pad, shift=shift), rand(m, n, dtype=dtype, seed=1, pad=pad, shift=shift)
    if m > 2:
        s[1] = 0
    stream_grad = rand(m, n, dtype=dtype, seed=2, pad=pad, shift=shift) if ds else None
    w = rand(n, seed=3).to(weight) if weight is not None else None
    rstd = (s.double().square().mean(1) + 1e-5).rsqrt().float()
    dx, dx_ok = out_like(m, n, dtype, pad, shift)
    d64 = stream_grad.double() if ds else torch.zeros(m, n, device="cuda", dtype=torch.float64)
    if in_place:
        dx, dx_ok = stream_grad, lambda: None
    dw = torch.full((n,), 7.0, device="cuda")
    _lib.rms_norm_backward(ptr(dy), ptr(s), ptr(rstd), ptr(dx), m, n, ptr(w), ptr(stream_grad), ptr(dw) if dweight else None,
                           CODE[dtype], CODE[weight] if weight is not None else _lib.F32, dy.stride(0), s.stride(0),
                           stream_grad.stride(0) if ds else 0, dx.stride(0), torch.cuda.current_stream().cuda_stream)
    r = rstd.double()[:, None]
    h, y64 = s.double() * r, dy.double()
    g = y64 * (w.double() if w is not None else 1.0)
    c = (g * h).mean(1, keepdim=True)
    want = r * (g - h * c) + d64
    ec = 2.0 ** -23 * (n / 32 + 40) * (g * h).abs().mean(1, keepdim=True)
    e = r * (h.abs() * ec + 2.0 ** -21 * (g.abs() + (h * c).abs())) + 2.0 ** -23 * (want.abs() + d64.abs())
    hs = half_step(dtype)
    assert_within(dx, want, e * (1 + hs) + hs * want.abs())
    if dweight:
        assert_within(dw, (y64 * h).sum(0), (m + 8) * 2.0 ** -23 * (y64 * h).abs().sum(0))
    else:
        assert bool((dw == 7.0).all())
    dx_ok()


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rms_norm_backward_widths(n, dtype):
    check_rms_norm_backward(13, n, dtype)


@pytest.mark.parametrize("ds", [True, False])
@pytest.mark.parametrize("weight", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dweight", [True, False])
@pytest.mark.parametrize("n", [200, 1111, 17000])
def test_rms_norm_backward_parts(ds, weight, dweight, n):
    check_rms_norm_backward(10, n, ds=ds, weight=weight, dweight=dweight)


@pytest.mark.parametrize("m", [1, 8, 9, 3000])
@pytest.mark.parametrize("n", [96, 520])
def test_rms_norm_backward_rows(m, n):
    check_rms_norm_backward(m, n)


@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (0, 1)])
@pytest.mark.parametrize("n", [264, 17000])
def test_rms_norm_backward_pitches(pad, shift, n):
    check_rms_norm_backward(9, n, pad=pad, shift=shift)


@pytest.mark.parametrize("n", [264, 1111, 17000])
def test_rms_norm_backward_in_place(n):
    check_rms_norm_backward(9, n, in_place=True)


def test_rms_norm_backward_of_nothing():
    dw = torch.full((16,), 7.0, device="cuda")
    _lib.rms_norm_backward(None, None, None, None, 0, 16, dweight=ptr(dw), stream=torch.cuda.current_stream().cuda_stream)
    assert not dw.any()


def test_rms_norm_backward_against_differences():
    """The gradient of sum(y * w) by central differences of the 64-bit norm."""
    m, n, h = 3, 24, 1e-4
    s, dy, w = rand(m, n), rand(m, n, seed=1), rand(n, seed=2)
    rstd = (s.double().square().mean(1) + 1e-5).rsqrt().float()
    dx = torch.empty(m, n, device="cuda")
    _lib.rms_norm_backward(ptr(dy), ptr(s), ptr(rstd), ptr(dx), m, n, ptr(w), dtype=_lib.F32, stream=torch.cuda.current_stream().cuda_stream)

    def value(x):
        return (x * (x.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w.double() * dy.double()).sum(1)

    for i in range(n):
        d = torch.zeros(m, n, device="cuda", dtype=torch.float64)
        d[:, i] = h
        want = (value(s.double() + d) - value(s.double() - d)) / (2 * h)
        # f32 arithmetic on a sum of 24 terms of size up to about 10, and h^2 of third derivatives.
        assert bool(((dx[:, i].double() - want).abs() <= 1e-5 + 2.0 ** -18 * dy.double().abs().sum(1)).all())


# ---- together -----------------------------------------------------------------------------------


def block(d, h, act, mode, seed=0):
    from tensorforge_b200.mlp import FeedForward

    w1, w2 = rand(d, h, seed=seed, scale=1 / math.sqrt(d)), rand(h, d, seed=seed + 1, scale=1 / math.sqrt(h))
    b1, b2, g = rand(h, seed=seed + 2, scale=0.1), rand(d, seed=seed + 3, scale=0.1), 1 + rand(d, seed=seed + 4, scale=0.1)
    return FeedForward(w1, b1, w2, b2, g, act, mode)


def block64(m, x, r):
    """The block in 64 bits from its own weights, as a differentiable function."""
    s = x + r if r is not None else x
    n = s * (s.square().mean(1, keepdim=True) + m.eps).rsqrt() * m.p["g"]
    return s + act64(n @ m.p["w1"] + m.p["b1"], m.activation)[0] @ m.p["w2"] + m.p["b2"]


def weights64(m):
    if m.mode == "fp8":
        w1, w2 = (m.w1.double() * m.s1.double()[:, None]).T, (m.w2.double() * m.s2.double()[:, None]).T
    else:
        w1, w2 = m.w1.double(), m.w2.double()
    m.p = {"w1": w1, "w2": w2, "b1": m.b1.double(), "b2": m.b2.double(), "g": m.norm_weight.double()}


@pytest.mark.parametrize("mode", ["bf16", "fp8"])
@pytest.mark.parametrize("act", ["gelu_tanh", "silu", "none"])
@pytest.mark.parametrize("rows,d,h", [(1, 256, 512), (37, 200, 328), (300, 512, 1024)])
@pytest.mark.parametrize("residual", [True, False])
def test_block(mode, act, rows, d, h, residual):
    """A feed-forward block: norm, product, (quantizer,) product and residual, from one token up."""
    m = block(d, h, act, mode)
    x = rand(rows, d, dtype=torch.bfloat16, seed=7)
    r = rand(rows, d, dtype=torch.bfloat16, seed=8) if residual else None
    out, s = m(x, r)
    weights64(m)
    want = block64(m, x.double(), r.double() if residual else None)
    # The branch's values are rounded three times (n, hid, out), in 8 bits by half a step of 2^-3
    # relative (2^-4), in bf16 2^-8, each the root of a sum over many: three halves of a step cover
    # the norm of a row, and s itself one rounding of bf16.
    half = 2.0 ** -4 if mode == "fp8" else 2.0 ** -8
    branch = want - (x.double() + (r.double() if residual else 0.0))
    assert float((out.double() - want).norm()) <= 3 * half * float(branch.norm()) + 2 * 2.0 ** -8 * float(want.norm())
    assert torch.equal(s, (x.float() + r.float()).bfloat16() if residual else x)


@pytest.mark.parametrize("act", ["gelu_tanh", "gelu", "silu", "relu"])
@pytest.mark.parametrize("rows,d,h", [(5, 128, 256), (130, 256, 520)])
def test_block_gradient(act, rows, d, h):
    """The block's gradients against the 64-bit function's own."""
    m = block(d, h, act, "bf16")
    x, r = rand(rows, d, dtype=torch.bfloat16, seed=7), rand(rows, d, dtype=torch.bfloat16, seed=8)
    dout = rand(rows, d, dtype=torch.bfloat16, seed=9)
    m(x, r, keep=True)
    got = m.backward(dout)
    weights64(m)
    x64 = x.double().requires_grad_()
    for v in m.p.values():
        v.requires_grad_()
    block64(m, x64, r.double()).backward(dout.double())
    want = {"dx": x64.grad, "dw1": m.p["w1"].grad, "db1": m.p["b1"].grad, "dw2": m.p["w2"].grad, "db2": m.p["b2"].grad,
            "dnorm_weight": m.p["g"].grad}
    for name, w in want.items():
        # At most six values on the way are in bf16 (n, pre, hid, dhid, dz, dn): half a step each.
        # The rectifier's slope jumps: where pre rounds across 0 no bound holds, which at these sizes
        # touches under one value in a hundred of the branch.
        rel = float((got[name].double() - w).norm() / w.norm())
        assert rel <= 6 * 2.0 ** -8 + (0.1 if act == "relu" else 0.0), (name, rel)
    with pytest.raises(ValueError):
        m.backward(dout)  # nothing kept


def test_block_refusals():
    m = block(64, 128, "silu", "fp8")
    x = rand(4, 64, dtype=torch.bfloat16)
    for bad in (lambda: m(x.float()), lambda: m(rand(4, 32, dtype=torch.bfloat16)), lambda: m(x, x.float()), lambda: m(x, keep=True),
                lambda: m(rand(64, 4, dtype=torch.bfloat16).T), lambda: block(64, 128, "tanh", "bf16"),
                lambda: block(64, 128, "silu", "fp4")):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("mode", ["bf16", "fp8"])
def test_block_captured_and_replayed(mode):
    """Two captured graphs of one block, replayed in turn with new inputs and beside eager calls."""
    m = block(256, 512, "gelu_tanh", mode)
    st = torch.cuda.Stream()
    graphs = []
    for rows in (3, 200):
        x, r = rand(rows, 256, dtype=torch.bfloat16, seed=rows), rand(rows, 256, dtype=torch.bfloat16, seed=rows + 1)
        with torch.cuda.stream(st):
            m(x, r)
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                out, _ = m(x, r)
        graphs.append((g, x, r, out))
    for k in range(3):
        for g, x, r, out in graphs:
            x.copy_(rand(*x.shape, dtype=torch.bfloat16, seed=50 + k))
            want = m(x, r)[0].clone()
            out.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


def test_gradient_captured_and_replayed():
    m = block(256, 512, "silu", "bf16")
    x, dout = rand(100, 256, dtype=torch.bfloat16), rand(100, 256, dtype=torch.bfloat16, seed=1)
    st = torch.cuda.Stream()

    def step():
        m(x, keep=True)
        return m.backward(dout)

    with torch.cuda.stream(st):
        step()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            got = step()
    for seed in (3, 4):
        x.copy_(rand(100, 256, dtype=torch.bfloat16, seed=seed))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), k


def test_two_streams_at_once():
    """Calls that overlap on the GPU share nothing: scratch comes from the pool in stream order."""
    calls = [Linear(200, 264, 133, act="gelu", residual=torch.bfloat16, seed=k) for k in range(2)]
    want = []
    for c in calls:
        c.call()
        torch.cuda.synchronize()
        want.append(c.out.clone())
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(30):
        for c, s in zip(calls, streams):
            c.call(s.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert torch.equal(c.out, w)


def test_first_call_inside_a_capture():
    """A process whose very first calls are captured: everything the library makes on first use is
    made outside the capture."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from tensorforge_b200 import _lib
a, b = torch.randn(40, 136, device="cuda").bfloat16(), torch.randn(72, 136, device="cuda").bfloat16()
out, y, rstd = torch.zeros(40, 72, device="cuda"), torch.zeros(40, 136, device="cuda"), torch.ones(40, device="cuda")
db, dw, dx = torch.zeros(72, 136, device="cuda"), torch.zeros(136, device="cuda"), torch.zeros(40, 136, device="cuda").bfloat16()
dout = torch.randn(40, 72, device="cuda")
torch.cuda.synchronize()
st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
with torch.cuda.stream(st):
    with torch.cuda.graph(g, stream=st):
        s = st.cuda_stream
        _lib.linear(a.data_ptr(), b.data_ptr(), out.data_ptr(), 40, 72, 136, out_dtype=_lib.F32, trans_b=True, stream=s)
        _lib.rms_norm(a.data_ptr(), y.data_ptr(), 40, 136, 1e-5, out_dtype=_lib.F32, stream=s)
        _lib.linear_backward(dout.data_ptr(), a.data_ptr(), b.data_ptr(), 40, 72, 136, dB=db.data_ptr(), dtype=_lib.F32,
                             grad_dtype=_lib.F32, trans_b=True, stream=s)
        _lib.rms_norm_backward(a.data_ptr(), a.data_ptr(), rstd.data_ptr(), dx.data_ptr(), 40, 136, dweight=dw.data_ptr(), stream=s)
g.replay()
torch.cuda.synchronize()
assert torch.allclose(out.double(), a.double() @ b.double().T, atol=1e-3)
assert torch.allclose(y.double(), a.double() * (a.double().square().mean(1, keepdim=True) + 1e-5).rsqrt(), atol=1e-5)
assert torch.allclose(db.double(), dout.bfloat16().double().T @ a.double(), atol=1e-3)
assert torch.allclose(dw.double(), (a.double() * a.double()).sum(0), rtol=1e-5)
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---- calls that the documentation allows ---------------------------------------------------------


def slices(rows, widths, dtype):
    """Matrices that are neighbouring column slices of one buffer, each width a column apart, and the
    check that the columns between them stay NaN."""
    whole = torch.full((rows, sum(widths) + len(widths)), float("nan"), device="cuda", dtype=dtype)
    views, gaps, c = [], [], 0
    for w in widths:
        views.append(whole[:, c:c + w])
        gaps.append(c + w)
        c += w + 1
    return views, lambda: bool(whole[:, gaps].isnan().all())


@pytest.mark.parametrize("m,n,k", [(5, 64, 48), (130, 33, 200), (700, 264, 72)])
def test_slices_of_one_buffer(m, n, k):
    """Operands and outputs that lie side by side in one buffer."""
    (a, res, out, pre, da, s, y), gaps = slices(m, (k, n, n, n, k, k, k), torch.bfloat16)
    a.copy_(rand(m, k))
    res.copy_(rand(m, n, seed=1))
    b, bias = rand(n, k, dtype=torch.bfloat16, seed=2, scale=1 / math.sqrt(k)), rand(n, seed=3)
    ld, st = a.stride(0), torch.cuda.current_stream().cuda_stream
    ref, refp, refd = torch.empty_like(res.contiguous()), torch.empty_like(res.contiguous()), torch.empty(m, k, device="cuda").bfloat16()
    ac, rc = a.contiguous(), res.contiguous()
    _lib.linear(ptr(a), ptr(b), ptr(out), m, n, k, "silu", ptr(bias), ptr(res), ptr(pre), trans_b=True, lda=ld, ldr=ld, ldo=ld,
                ldp=ld, stream=st)
    _lib.linear(ptr(ac), ptr(b), ptr(ref), m, n, k, "silu", ptr(bias), ptr(rc), ptr(refp), trans_b=True, stream=st)
    _lib.linear_backward(ptr(out), None, ptr(b), m, n, k, "silu", ptr(pre), dA=ptr(da), trans_b=True, lddo=ld, ldp=ld, ldda=ld, stream=st)
    _lib.linear_backward(ptr(ref), None, ptr(b), m, n, k, "silu", ptr(refp), dA=ptr(refd), trans_b=True, stream=st)
    assert torch.equal(out, ref) and torch.equal(pre, refp) and torch.equal(da, refd)
    rstd, refs, refy = torch.empty(m, device="cuda"), torch.empty_like(ac), torch.empty_like(ac)
    _lib.rms_norm(ptr(a), ptr(y), m, k, 1e-5, residual=ptr(da), sum_out=ptr(s), rstd=ptr(rstd), ldx=ld, ldr=ld, lds=ld, ldo=ld, stream=st)
    _lib.rms_norm(ptr(ac), ptr(refy), m, k, 1e-5, residual=ptr(refd), sum_out=ptr(refs), rstd=ptr(rstd), stream=st)
    assert torch.equal(s, refs)
    # The unaligned rows' sums are taken in another order: a step of bf16 at most.
    assert bool(((y.double() - refy.double()).abs() <= 2.0 ** -7 * refy.double().abs()).all())
    assert gaps()


def test_inputs_written_just_before():
    """A call sees what the launches before it wrote, though its blocks may start before they end:
    small vectors and whole operands, from torch's kernels and from the library's own."""
    m, n, k = 48, 512, 256
    st = torch.cuda.current_stream().cuda_stream
    x, b = rand(m, k, dtype=torch.bfloat16), rand(n, k, dtype=torch.bfloat16, seed=1, scale=1 / 16)
    weight, bias, dw = torch.ones(k, device="cuda"), torch.zeros(n, device="cuda"), torch.empty(k, device="cuda")
    y, out, dx = torch.empty_like(x), torch.empty(m, n, device="cuda").bfloat16(), torch.empty_like(x)
    rstd = torch.empty(m, device="cuda")
    outs = []
    for i in range(40):
        f = 2.0 ** (i % 5)
        weight.fill_(f)
        bias.fill_(256 * f)
        rstd.zero_()
        _lib.rms_norm(ptr(x), ptr(y), m, k, 1e-5, weight=ptr(weight), rstd=ptr(rstd), stream=st)
        _lib.linear(ptr(y), ptr(b), ptr(out), m, n, k, bias=ptr(bias), trans_b=True, stream=st)
        _lib.rms_norm_backward(ptr(x), ptr(x), ptr(rstd), ptr(dx), m, k, weight=ptr(weight), dweight=ptr(dw), stream=st)
        outs.append([(t.float() / f).sum() for t in (y, out, dx)] + [dw.sum()])
    torch.cuda.synchronize()
    # Powers of two scale through every one of them without a rounding.
    for o in outs[1:]:
        for got, want in zip(o, outs[0]):
            assert float(got) == float(want)


@pytest.mark.parametrize("mode", ["bf16", "fp8"])
def test_block_of_no_rows(mode):
    m = block(64, 128, "silu", mode)
    x = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16)
    out, s = m(x, x.clone(), keep=mode == "bf16")
    assert out.shape == x.shape and s.shape == x.shape
    if mode == "bf16":
        g = m.backward(x)
        assert all(bool((g[k] == 0).all()) for k in ("dw1", "db1", "dw2", "db2", "dnorm_weight")) and g["dx"].shape == x.shape


def test_block_refuses_other_places():
    """Rows, residuals and gradients that are not on the weights' GPU; a gradient on another stream."""
    m = block(64, 128, "silu", "bf16")
    x = rand(4, 64, dtype=torch.bfloat16)
    for bad in (lambda: m(x.cpu()), lambda: m(x, x.cpu())):
        with pytest.raises(ValueError):
            bad()
    m(x, keep=True)
    with pytest.raises(ValueError):
        m.backward(x.cpu())
    with torch.cuda.stream(torch.cuda.Stream()), pytest.raises(ValueError):
        m.backward(x)
    assert m.backward(x)["dx"].shape == x.shape  # what was kept is still there


@pytest.mark.parametrize("m,n,k", [(300, 264, 1500), (129, 77, 1000)])
@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 1)])
def test_sums_in_pieces_with_the_whole_epilogue(m, n, k, residual, pad, shift):
    """f32 outputs whose sums are taken in pieces by CTA pairs: bias, pre, activation and residual after."""
    _lib.check(_lib.lib().tforge_debug_linear_kernel(2, 0, 0))
    for pre in (False, True):
        Linear(m, n, k, act="gelu", residual=residual, out=torch.float32, pre=pre, pad=pad, shift=shift).call().check()


@pytest.mark.parametrize("m,n,k", [(40, 264, 136), (300, 520, 1000), (2304, 2560, 2048)])
@pytest.mark.parametrize("bias", [True, False])
def test_gradients_in_a_row(m, n, k, bias):
    """The gradient's products run beside its column sums and one another; whoever comes next -- here a
    norm that reads dA and dB, and the next gradient, which overwrites them -- finds all complete."""
    st = torch.cuda.current_stream().cuda_stream
    first = rand(m, n, dtype=torch.bfloat16)
    dout, pre = torch.empty_like(first), rand(m, n, dtype=torch.bfloat16, seed=1)
    a, b = rand(m, k, dtype=torch.bfloat16, seed=2), rand(n, k, dtype=torch.bfloat16, seed=3)
    da, db, dbias = torch.empty_like(a), torch.empty_like(b), torch.empty(n, device="cuda")
    ya, yb = torch.empty_like(a), torch.empty_like(b)
    outs = []
    for i in range(12):
        f = 2.0 ** (i % 5)
        torch.mul(first, f, out=dout)
        da.zero_()
        db.zero_()
        _lib.linear_backward(ptr(dout), ptr(a), ptr(b), m, n, k, "relu", ptr(pre), dA=ptr(da), dB=ptr(db),
                             dbias=ptr(dbias) if bias else None, trans_b=True, stream=st)
        _lib.rms_norm(ptr(da), ptr(ya), m, k, 0.0, stream=st)
        _lib.rms_norm(ptr(db), ptr(yb), n, k, 0.0, stream=st)
        outs.append([(da / f).clone(), (db / f).clone(), ya.clone(), yb.clone()] + ([dbias / f] if bias else []))
    for o in outs[1:]:
        for got, want in zip(o, outs[0]):  # powers of two go through without a rounding
            assert torch.equal(got, want)
    dz = torch.where(pre > 0, first, torch.zeros_like(first)).double()
    for got, want, length in ((outs[0][0], dz @ b.double(), n), (outs[0][1], dz.T @ a.double(), m)):
        mag = (dz.abs() @ b.double().abs()) if got is outs[0][0] else (dz.abs().T @ a.double().abs())
        assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + (length + 4) * 2.0 ** -23 * mag).all())


EDGES = [64, 72, 128, 136, 256, 264, 512, 520, 768, 776, 1024, 1032, 1536, 1544, 2048, 2056, 2560, 4096, 4104, 6144, 6152, 8192,
         8200, 12288, 12296, 16384, 16392, 24576, 24584, 32768]


@pytest.mark.parametrize("n", EDGES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rms_norm_at_every_kernels_edges(n, dtype):
    """The widths at which the kernels for 16-byte pieces change, and between them for single elements,
    with few rows (148) and more."""
    for m in (148, 149):
        for w in (n, n + 3):
            check_rms_norm(m, w, dtype, torch.bfloat16 if m == 148 else torch.float8_e4m3fn)
            check_rms_norm_backward(m, w, dtype)


def test_offsets_beyond_32_bits():
    """Arrays of more than 2^31 elements: the first rows and the last."""
    m, n, k = (1 << 17) + 8, (1 << 14) + 8, 64
    st = torch.cuda.current_stream().cuda_stream
    rows = torch.tensor([0, 1, m // 2, m - 2, m - 1], device="cuda")
    a, b = rand(m, k, dtype=torch.bfloat16), rand(n, k, dtype=torch.bfloat16, seed=1, scale=1 / 8)
    for ld in (n, n + 3):  # by TMA, and element by element
        out = torch.empty(m * ld, device="cuda", dtype=torch.bfloat16).view(m, ld)[:, :n]
        _lib.linear(ptr(a), ptr(b), ptr(out), m, n, k, trans_b=True, ldo=ld, stream=st)
        want = a[rows].double() @ b.double().T
        assert_within(out[rows], want, 2.0 ** -8 * want.abs() + (k + 4) * 2.0 ** -23 * (a[rows].double().abs() @ b.double().abs().T))
        y, sc, rstd = torch.empty(m * ld, device="cuda", dtype=torch.float8_e4m3fn).view(m, ld)[:, :n], *torch.empty(2, m, device="cuda")
        _lib.rms_norm(ptr(out), ptr(y), m, n, 1e-5, rstd=ptr(rstd), scale=ptr(sc), out_dtype=_lib.E4M3, ldx=ld, ldo=ld, stream=st)
        s64 = out[rows].double()
        r64 = (s64.square().mean(1) + 1e-5).rsqrt()
        assert_within(rstd[rows], r64, 2.0 ** -23 * (n / 64 + 24) * r64)
        v = s64 * r64[:, None] / sc[rows].double()[:, None]
        assert_within(y[rows].float(), v, 2.0 ** -23 * (n / 16) * v.abs() + torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10))
        dx, dw = torch.empty(m * ld, device="cuda", dtype=torch.bfloat16).view(m, ld)[:, :n], torch.empty(n, device="cuda")
        _lib.rms_norm_backward(ptr(out), ptr(out), ptr(rstd), ptr(dx), m, n, dweight=ptr(dw), lddy=ld, lds=ld, lddx=ld, stream=st)
        r = rstd[rows].double()[:, None]
        h = s64 * r
        c = (s64 * h).mean(1, keepdim=True)
        want = r * (s64 - h * c)
        e = r * h.abs() * 2.0 ** -23 * (n / 32 + 40) * (s64 * h).abs().mean(1, keepdim=True) + 2.0 ** -21 * r * (s64.abs() + (h * c).abs())
        assert_within(dx[rows], want, e * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs())
        cols = torch.tensor([0, n - 1], device="cuda")
        z = out[:, cols].double()
        assert_within(dw[cols], (z * z * rstd.double()[:, None]).sum(0), (m + 8) * 2.0 ** -23 * (z * z * rstd.double()[:, None]).sum(0))
        del y, dx
        da, db = torch.empty_like(a), torch.empty_like(b)
        _lib.linear_backward(ptr(out), ptr(a), ptr(b), m, n, k, dA=ptr(da), dB=ptr(db), trans_b=True, lddo=ld, stream=st)
        want = s64 @ b.double()
        assert_within(da[rows], want, 2.0 ** -8 * want.abs() + (n + 4) * 2.0 ** -23 * (s64.abs() @ b.double().abs()))
        want = z.T @ a.double()
        assert_within(db[cols], want, 2.0 ** -8 * want.abs() + (m + 4) * 2.0 ** -23 * (z.abs().T @ a.double().abs()))
        del out


def test_two_threads_at_once():
    """Two host threads, each on its own stream."""
    import threading

    calls = [Linear(200, 264, 133, act="gelu", residual=torch.bfloat16, seed=k) for k in range(2)]
    want = []
    for c in calls:
        c.call()
        torch.cuda.synchronize()
        want.append(c.out.clone())
        c.out.zero_()
    torch.cuda.synchronize()
    failed = []

    def work(c):
        try:
            st = torch.cuda.Stream()
            for _ in range(100):
                c.call(st.cuda_stream)
            st.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for c, w in zip(calls, want):
        assert torch.equal(c.out, w)
