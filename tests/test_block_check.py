"""The feed-forward command's check of its outputs and gradients, on the CPU: exact ones pass, and a
mistake in any of them does not."""

import types

import pytest

torch = pytest.importorskip("torch")

from tensorforge_b200.mlp import block_bound, block_errors  # noqa: E402

M, D, H = 37, 24, 56
NAMES = ("dx", "dw1", "db1", "dw2", "db2", "dnorm_weight")


def exact(mode="bf16", with_residual=True):
    """A block in 64 bits, its inputs, output and autograd's gradients."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    p = {"w1": r(D, H) / D ** 0.5, "b1": 0.1 * r(H), "w2": r(H, D) / H ** 0.5, "b2": 0.1 * r(D), "norm_weight": 1 + 0.2 * r(D)}
    x, residual, dout = r(M, D), r(M, D) if with_residual else None, r(M, D)
    for v in p.values():
        v.requires_grad_()
    s = (x + residual if with_residual else x.clone()).requires_grad_()
    n = torch.nn.functional.rms_norm(s, (D,), p["norm_weight"], 1e-5)
    out = s + torch.nn.functional.gelu(n @ p["w1"] + p["b1"], approximate="tanh") @ p["w2"] + p["b2"]
    out.backward(dout)
    grads = {"dx": s.grad, **{"d" + k: v.grad for k, v in p.items()}}
    model = types.SimpleNamespace(mode=mode, eps=1e-5, activation="gelu_tanh", **{k: v.detach() for k, v in p.items()})
    if mode == "fp8":  # rows a feature, with scales
        model.s1, model.s2 = 0.5 + torch.rand(H, generator=g), 0.5 + torch.rand(D, generator=g)
        model.w1, model.w2 = model.w1.t() / model.s1.double()[:, None], model.w2.t() / model.s2.double()[:, None]
    return model, x, residual, out.detach(), dout, grads


ROWS, UNITS = torch.tensor([0, 5, 36]), torch.tensor([1, 30, 55])


@pytest.mark.parametrize("with_residual", [True, False])
@pytest.mark.parametrize("chunk", [8, 1024])
def test_exact_outputs_pass(with_residual, chunk):
    model, x, residual, out, dout, grads = exact(with_residual=with_residual)
    errors = block_errors(model, x, residual, out, ROWS, dout, grads, UNITS, chunk)
    assert set(errors) == {"out", *NAMES} and max(errors.values()) < 1e-12


def test_exact_output_of_8_bit_weights_passes():
    model, x, residual, out, _, _ = exact("fp8")
    assert block_errors(model, x, residual, out, ROWS).keys() == {"out"}
    assert block_errors(model, x, residual, out, ROWS)["out"] < 1e-12


@pytest.mark.parametrize("name", ("out", *NAMES))
@pytest.mark.parametrize("mistake", [lambda t: t * 1.05, torch.zeros_like, lambda t: t.roll(1, 0), lambda t: t * float("nan")])
def test_mistakes_do_not_pass(name, mistake):
    model, x, residual, out, dout, grads = exact()
    if name == "out":
        out = mistake(out)
    else:
        grads[name] = mistake(grads[name])
    errors = block_errors(model, x, residual, out, ROWS, dout, grads, UNITS)
    assert not errors[name] <= block_bound("bf16", name)
    assert all(e < 1e-12 for k, e in errors.items() if k != name)
