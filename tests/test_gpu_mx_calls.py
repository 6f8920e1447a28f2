"""Calls on 4-bit weights at the edges of what they take."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import mx_reference as ref

pytestmark = pytest.mark.gpu


def layer_of(qb, cuda, dtype="bf16", M=5, seed=3):
    d = ref.draw(dtype, M, 64, 32, rank=4, bias=True, seed=seed, device=cuda)
    return d, qb.quantize_quaternion_weights(*d["w"])


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", ["x", "bias", "a", "b"])
def test_forward_mode_derivatives_are_refused(qb, cuda, which, grad):
    d, q = layer_of(qb, cuda)
    with fwd.dual_level():
        v = {k: d[k].clone().requires_grad_(grad) for k in ("x", "bias", "a", "b")}
        v[which] = fwd.make_dual(v[which], torch.ones_like(v[which]))
        with pytest.raises(RuntimeError):
            qb.mx_quaternion_linear(v["x"], q, v["bias"], v["a"], v["b"], 2.0)
        # tensors without a tangent, inside a level
        y = qb.mx_quaternion_linear(d["x"], q, d["bias"], d["a"], d["b"], 2.0)
    assert torch.equal(y, qb.mx_quaternion_linear(d["x"], q, d["bias"], d["a"], d["b"], 2.0))


def test_function_transforms_are_refused(qb, cuda):
    """None of them comes back with a wrong value."""
    d, q = layer_of(qb, cuda, "f32")
    f, x = (lambda v: qb.mx_quaternion_linear(v, q)), d["x"]
    with pytest.raises(RuntimeError):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda v: f(v).sum())(x)
