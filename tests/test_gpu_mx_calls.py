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


# ------------------------------------------------------------- model conversion
def test_quantize_model_takes_hooks_along(qb, cuda):
    net = torch.nn.Sequential(qb.QuaternionLinear(64, 32, bias=True), torch.nn.ReLU()).to(cuda)
    seen = []
    handles = [net[0].register_forward_hook(lambda m, a, out: out + 1.0),
               net[0].register_forward_pre_hook(lambda m, a: seen.append(type(m).__name__)),
               net[0].register_full_backward_hook(lambda m, gi, go: seen.append("backward"))]
    qb.quantize_model(net)
    x = torch.randn(3, 64, device=cuda, requires_grad=True)
    want = qb.mx_quaternion_linear(x, net[0].weights, net[0].bias) + 1.0
    got = net[0](x)
    assert torch.equal(got, want) and seen == ["MXQuaternionLinear"]
    got.sum().backward()
    assert seen[1:] == ["backward"]
    for h in handles:
        h.remove()
    assert torch.equal(net[0](x), qb.mx_quaternion_linear(x, net[0].weights, net[0].bias))
    assert len(seen) == 2


def test_quantize_model_says_what_it_leaves(qb, cuda):
    class Doubled(qb.QuaternionLinear):
        def forward(self, x):
            return 2 * super().forward(x)

    class Named(qb.QuaternionLinear):
        pass

    net = torch.nn.ModuleDict({"own": Doubled(32, 32), "named": Named(32, 32), "plain": qb.QuaternionLinear(32, 32),
                               "unit": qb.UnitQuaternionLinear(32, 32)}).to(cuda)
    before = {k: net[k] for k in ("own", "unit")}
    assert sorted(qb.quantize_model(net)) == ["named", "plain"]
    assert all(net[k] is m for k, m in before.items())
    alone = qb.QuaternionLinear(32, 32).to(cuda)
    with pytest.raises(ValueError):
        qb.quantize_model(alone)
    assert isinstance(alone.wr, torch.nn.Parameter)


# ---------------------------------------------------------------- far apart scales
@pytest.mark.parametrize("M", [1, 3, 16, 32, 64, 65, 200])
def test_fp16_rows_far_below_the_largest_weight(qb, cuda, M):
    """Every row of an fp16 layer counts, down to fp16's smallest weights beside ones of
    4096, with any number of tokens and in the input gradient."""
    N_g, K_g = 48, 96
    g = torch.Generator().manual_seed(M)
    levels = torch.tensor([2.0 ** -8, 2.0 ** -16, 2.0 ** -22]).repeat_interleave(16)[:, None]
    w = [(torch.randn(N_g, K_g, generator=g) * levels).half() for _ in range(4)]
    for t in w:
        t[0, :32] = torch.randn(32, generator=g).half() * 2048  # x is zero there
    q = qb.quantize_quaternion_weights(*(t.to(cuda) for t in w))
    v = torch.stack(q.dequantize(torch.float32)).double().cpu().numpy()
    x = torch.randn(M, 4 * K_g, generator=g) * 256
    x[:, :128] = 0
    x = x.half().to(cuda)
    y = qb.mx_quaternion_linear(x, q)
    want = ref.layer(ref.f64(x), v)
    small = 2.0 ** -25 / 2.0 ** -12  # half of fp16's smallest step, results of at least 2^-12
    for k in range(3):
        rows = slice(64 * k, 64 * k + 64)
        assert ref.rel(ref.f64(y)[:, rows], want[:, rows]) <= ref.tolerance("f16", 4 * K_g) + small, k
    # the gradient: columns of one level at a time
    for k in range(3):
        gy = torch.zeros(M, 4 * N_g)
        gy[:, 64 * k + 4:64 * k + 64] = torch.randn(M, 60, generator=g) * 256
        gy = gy.half().to(cuda)
        xg = x.clone().requires_grad_(True)
        (dx,) = torch.autograd.grad(qb.mx_quaternion_linear(xg, q), xg, gy)
        want = ref.gradients(ref.f64(gy), ref.f64(x), v)[0]
        assert ref.rel(ref.f64(dx), want) <= ref.tolerance("f16", 4 * N_g) + small, k
