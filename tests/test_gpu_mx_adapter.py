"""LoRA adapters on 4-bit weights where the adapter's own products decide the
result: one output rounding over the types' whole range."""

import numpy as np
import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu


def rounded(want, dtype):
    with np.errstate(over="ignore"):
        return ref.f64(torch.from_numpy(np.ascontiguousarray(want)).to(ref.TORCH[dtype]))


def bound(want, dtype, terms):
    """2-norm of an error: that of the one rounding to the type, a tenth more for values
    that an earlier error moves to the other neighbour, and fp32 sums of `terms` terms
    as in ref.tolerance."""
    return 1.1 * np.linalg.norm(rounded(want, dtype) - want) + \
        2.0 ** -23 * (2 + terms) ** 0.5 * np.linalg.norm(want)


def one_rounding(got, want, dtype, terms, what=""):
    want = np.asarray(want)
    assert np.isfinite(rounded(want, dtype)).all(), "the exact result is in range"
    got = ref.f64(got)
    assert np.isfinite(got).all(), what
    assert np.linalg.norm(got - want) <= bound(want, dtype, terms), what


def zero_base(qb, fin, fout, device):
    return qb.quantize_quaternion_weights(*(torch.zeros(fout // 4, fin // 4, device=device) for _ in range(4)))


def values_of(q):
    return np.stack([ref.f64(w) for w in q.dequantize(torch.float32)])


def backward(qb, q, d, gy):
    leaves = {k: d[k].clone().requires_grad_(True) for k in ("x", "a", "b")}
    y = qb.mx_quaternion_linear(leaves["x"], q, None, leaves["a"], leaves["b"], d["scale"])
    return dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))


def expected(q, d, gy):
    dx, da, db, _ = ref.gradients(ref.f64(gy), ref.f64(d["x"]), values_of(q), ref.f64(d["a"]), ref.f64(d["b"]),
                                  d["scale"])
    return {"x": dx, "a": da, "b": db}


# ------------------------------------------------- small gradients and factors
@pytest.mark.parametrize("gy_std", [1.0, 1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("M", [24, 500])
def test_adapter_gradients_of_small_fp16_values(qb, cuda, gy_std, M):
    """A LoRA factor near zero and gradients down to fp16's smallest numbers, tokens
    of very different size among them."""
    d = ref.draw("f16", M, 512, 1024, rank=8, seed=M, device=cuda)
    d["b"] = (d["b"].float() * (1e-4 / 0.05)).half()
    q = qb.quantize_quaternion_weights(*d["w"])
    gy = ref.draw("f16", M, 1024, 4, seed=5, device=cuda)["x"].float() * gy_std
    for far in (0, 12):
        g = gy * torch.exp2(-(torch.arange(M, device=cuda) % (far + 1)).float())[:, None]
        g = g.half()
        got, want = backward(qb, q, d, g), expected(q, d, g)
        one_rounding(got["a"], want["a"], "f16", M + 1024, "a")
    # the other factor: a small scale makes t small
    d["a"] = (d["a"].float() * 1e-3).half()
    d["scale"] = 2.0 * gy_std
    g = ref.draw("f16", M, 1024, 4, seed=5, device=cuda)["x"]
    got, want = backward(qb, q, d, g), expected(q, d, g)
    one_rounding(got["b"], want["b"], "f16", M + 512, "b")


def test_adapter_gradients_of_far_apart_token_groups(qb, cuda):
    """Whole groups of tokens zero, and others far below the rest: their ranks' sums
    neither vanish nor spill over."""
    M = 320
    d = ref.draw("f16", M, 256, 256, rank=20, seed=1, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    level = torch.tensor([0.0, 1.0, 2.0 ** -10, 2.0 ** -20, 0.0] * 4, device=cuda).repeat_interleave(16)[:, None]
    base = ref.draw("f16", M, 256, 4, seed=2, device=cuda)["x"].float()
    for gy in ((base * level).half(), (base * level.flip(0)).half()):
        got, want = backward(qb, q, d, gy), expected(q, d, gy)
        one_rounding(got["a"], want["a"], "f16", M + 256, "a")
        one_rounding(got["b"], want["b"], "f16", M + 256, "b")
    # only the smallest tokens
    gy = (ref.draw("f16", M, 256, 4, seed=2, device=cuda)["x"].float() * 2.0 ** -20).half()
    got, want = backward(qb, q, d, gy), expected(q, d, gy)
    one_rounding(got["a"], want["a"], "f16", M + 256, "a")
    zero = torch.zeros_like(gy)
    got = backward(qb, q, d, zero)
    assert not any(bool(t.any()) for t in got.values())


def test_nonfinite_tokens_in_adapter_gradients(qb, cuda):
    """A token with an infinity or a NaN makes the sums it is part of non-finite, no others."""
    M = 100
    for dtype in ("f16", "bf16"):
        d = ref.draw(dtype, M, 128, 128, rank=8, seed=1, device=cuda)
        q = qb.quantize_quaternion_weights(*d["w"])
        clean = ref.draw(dtype, M, 128, 4, seed=2, device=cuda)["x"]
        want = backward(qb, q, d, clean)
        for bad in (float("inf"), float("nan")):
            gy = clean.clone()
            gy[40, 5] = bad
            got = backward(qb, q, d, gy)
            keep = torch.arange(M, device=cuda) != 40
            assert torch.equal(got["x"][keep], want["x"][keep])
            assert not bool(got["x"][40].isfinite().any())
            assert not bool(got["a"].isfinite().any())
            others = torch.arange(128, device=cuda) != 5
            assert torch.equal(got["b"][others], want["b"][others])
            assert not bool(got["b"][5].isfinite().any())


# ------------------------------------------------------------ range of fp16 factors
def scaled(t, factor):
    return (t.float() * factor).to(t.dtype)


@pytest.mark.parametrize("M", [1, 24, 32, 33, 64, 65, 130, 300])
def test_fp16_range_of_an_adapter_does_not_depend_on_the_tokens(qb, cuda, M):
    """Large B, large and small down projections: y and dx are finite and right with
    any number of tokens."""
    d = ref.draw("f16", M, 512, 320, rank=12, seed=M, device=cuda)
    gy = ref.draw("f16", M, 320, 4, seed=5, device=cuda)["x"]
    a, b, x = d["a"], d["b"], d["x"]
    for q in (qb.quantize_quaternion_weights(*d["w"]), zero_base(qb, 512, 320, cuda)):
        v = values_of(q)
        for fa, fb, fx, scale in ((1e-2, 40000.0, 1e-2, 2.0),    # |B| up to 8000, t about 2e-4
                                  (200.0, 2e-3, 1.0, 1000.0),    # t about 2e5, B about 1e-4
                                  (1.0, 400.0, 1e-3, 1e-3)):     # t about 1e-6, B about 20
            d.update(a=scaled(a, fa), b=scaled(b, fb), x=scaled(x, fx), scale=scale)
            y = qb.mx_quaternion_linear(d["x"], q, None, d["a"], d["b"], scale)
            want = ref.layer(ref.f64(d["x"]), v, None, ref.f64(d["a"]), ref.f64(d["b"]), scale)
            one_rounding(y, want, "f16", 512, (fa, fb))
        for fa, fb, fg, scale in ((40000.0, 1e-2, 1e-2, 2.0), (2e-3, 200.0, 1.0, 1000.0), (400.0, 1.0, 1e-3, 1e-3)):
            d.update(a=scaled(a, fa), b=scaled(b, fb), x=scaled(x, 1e-3), scale=scale)
            g = scaled(gy, fg)
            got, want = backward(qb, q, d, g), expected(q, d, g)
            for k in ("x", "a", "b"):
                if np.isfinite(rounded(want[k], "f16")).all():
                    one_rounding(got[k], want[k], "f16", 512 + M, (k, fa, fb))


# --------------------------------------------------- adapters that decide the result
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("M,fin,fout,rank", [(70, 256, 256, 32), (130, 512, 260, 64), (300, 260, 512, 40),
                                             (257, 128, 132, 100), (100, 256, 192, 300), (500, 64, 64, 7)])
def test_one_rounding_where_the_adapter_decides(qb, cuda, dtype, M, fin, fout, rank):
    """A base of zeros: the bound rejects a down projection, or B, rounded to one 16-bit part."""
    d = ref.draw(dtype, M, fin, fout, rank=rank, seed=rank, device=cuda)
    q = zero_base(qb, fin, fout, cuda)
    gy = ref.draw(dtype, M, fout, 4, seed=5, device=cuda)["x"]
    x, a, b, g = (ref.f64(t) for t in (d["x"], d["a"], d["b"], gy))
    t, u = d["scale"] * x @ a.T, d["scale"] * g @ b
    got = backward(qb, q, d, gy)
    got["y"] = qb.mx_quaternion_linear(d["x"], q, None, d["a"], d["b"], d["scale"])
    want = {"y": t @ b.T, "x": u @ a, "a": u.T @ x, "b": g.T @ t}
    th, uh = rounded(t, dtype), rounded(u, dtype)
    one_part = {"y": th @ b.T, "x": uh @ a, "a": uh.T @ x, "b": g.T @ th}
    if dtype == "f16":  # what bf16 parts of the factors would lose
        one_part.update(y=t @ rounded(b, "bf16").T, x=u @ rounded(a, "bf16"))
    terms = {"y": fin + rank, "x": fout + rank, "a": M + fout, "b": M + fin}
    for k, w in want.items():
        one_rounding(got[k], w, dtype, terms[k], k)
        assert np.linalg.norm(rounded(one_part[k], dtype) - w) > bound(w, dtype, terms[k]), k


@pytest.mark.parametrize("dtype,tie,above", [("bf16", 2.0 ** -8, 2.0 ** -20), ("f16", 2.0 ** -11, 2.0 ** -22)])
def test_every_bit_of_a_down_projection_counts(qb, cuda, dtype, tie, above):
    """t = u = 1 + tie + above, just past the middle between two numbers of the type, by
    sums and products that are exact: every result is the upper one."""
    M, F, rank = 70, 64, 8
    T = ref.TORCH[dtype]
    rows = torch.zeros(M, F, device=cuda)
    rows[:, 0:8], rows[:, 8:16], rows[:, 16:24] = 1.0, tie, above
    ones = (torch.arange(F, device=cuda)[:, None] % rank == torch.arange(rank, device=cuda)).float()  # [F, rank]
    pick = torch.eye(F, device=cuda).new_zeros(M, F)
    pick[:F] = torch.eye(F, device=cuda)  # each column from one token
    q = zero_base(qb, F, F, cuda)
    upper = 1 + 2 * tie
    d = dict(x=rows.to(T), a=ones.t().contiguous().to(T), b=ones.to(T), scale=1.0)
    y = qb.mx_quaternion_linear(d["x"], q, None, d["a"], d["b"], 1.0)
    assert bool((y == upper).all())
    assert bool((backward(qb, q, d, pick.to(T))["b"] == upper).all())
    d["x"] = pick.to(T)
    got = backward(qb, q, d, rows.to(T))
    assert bool((got["x"] == upper).all())
    assert bool((got["a"] == upper).all())
