"""Global gradient norm and clipping against 64-bit sums."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def params_of(shapes, dtypes, device, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for k, s in enumerate(shapes):
        dt = dtypes[k % len(dtypes)]
        p = torch.nn.Parameter(torch.empty(s, dtype=dt, device=device))
        p.grad = (torch.randn(s, generator=g) * std).to(dt).to(device)
        out.append(p)
    return out


def check(qb, params, max_norm):
    before = [p.grad.double() for p in params]
    want = float(torch.stack([g.square().sum() for g in before]).sum().sqrt())
    norm = qb.clip_grad_norm(params, max_norm)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and norm.device == params[0].device
    # squares of a piece's share in fp32 (16 terms at most), the rest in fp64, one rounding
    assert abs(float(norm) - want) <= 16 * 2.0 ** -24 * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for p, g in zip(params, before):
        if factor == 1.0:
            assert torch.equal(p.grad.double(), g)
            continue
        err = (p.grad.double() - g * factor).abs()
        # the factor (norm, sum and quotient rounded), the product, the type's rounding
        # (below the smallest normal number half a step of it)
        lim = (g * factor).abs() * (20 * 2.0 ** -24 + HALF_STEP[p.dtype]) + torch.finfo(p.dtype).smallest_normal * \
            HALF_STEP[p.dtype] * 2
        assert bool((err <= lim).all())


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float16,),
                                    (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("shapes", [[(1,)], [(8192,)], [(8193,), (8191,), (3,)], [(64, 4096), (4096, 64)],
                                    [(5, 7)] * 70, [(0,), (10,), (0,), (0, 4), (30000,), (0,)], [(1,)] * 600,
                                    [(257, 129)] * 20])
def test_clip(qb, cuda, dtypes, shapes):
    for max_norm in (0.5, 1e6):
        check(qb, params_of(shapes, dtypes, cuda), max_norm)


def test_large_tensors(qb, cuda):
    check(qb, params_of([(40_000_003,), (9_999_999,)], (torch.float32,), cuda), 1.0)
    check(qb, params_of([(40_000_003,), (9_999_999,)], (torch.bfloat16,), cuda), 1.0)


def test_unaligned_and_strided_gradients(qb, cuda):
    for dt in (torch.float32, torch.bfloat16):
        params = params_of([(100,), (20000,), (60, 70), (60, 70)], (dt,), cuda)
        flat = torch.randn(30001, device=cuda).to(dt)
        params[0].grad = flat[1:101]                     # not on a 16-byte boundary
        params[1].grad = flat[3001:23001]
        params[2].grad = torch.randn(70, 60, device=cuda).to(dt).t()      # dense, transposed
        wide = torch.randn(60, 90, device=cuda).to(dt)
        params[3].grad = wide[:, 10:80]                  # gaps between its rows
        rest = wide[:, :10].clone(), wide[:, 80:].clone(), flat[:1].clone(), flat[101:3001].clone()
        check(qb, params, 0.7)
        assert torch.equal(wide[:, :10], rest[0]) and torch.equal(wide[:, 80:], rest[1])
        assert torch.equal(flat[:1], rest[2]) and torch.equal(flat[101:3001], rest[3])


def test_wide_values(qb, cuda):
    """Squares past fp32's range, and a zero gradient."""
    check(qb, params_of([(20000,), (100,)], (torch.float32,), cuda, std=1e25), 1.0)
    params = params_of([(20000,), (100,)], (torch.float32,), cuda, std=0.0)
    assert float(qb.clip_grad_norm(params, 1.0)) == 0.0
    assert not any(bool(p.grad.any()) for p in params)
    params = params_of([(300,)], (torch.float32,), cuda)
    qb.clip_grad_norm(params, 0.0)
    assert not bool(params[0].grad.any())


def test_nonfinite(qb, cuda):
    for n in (9000, 50):
        params = params_of([(n,), (40,)], (torch.float32,), cuda)
        params[0].grad[7] = float("nan")
        before = params[1].grad.clone()
        with pytest.raises(RuntimeError):
            qb.clip_grad_norm(params, 1.0, error_if_nonfinite=True)
        assert torch.equal(params[1].grad, before)
        assert bool(qb.clip_grad_norm(params, 1.0).isnan())
        assert all(bool(p.grad.isnan().all()) for p in params)
        params = params_of([(n,), (40,)], (torch.float32,), cuda)
        params[0].grad[7] = float("-inf")
        assert float(qb.clip_grad_norm(params, 1.0)) == float("inf")
        assert not bool(params[1].grad.any())
        assert bool(params[0].grad[7].isnan())


def test_which_parameters_count(qb, cuda):
    params = params_of([(300,), (20,)], (torch.float32,), cuda)
    none = torch.nn.Parameter(torch.zeros(4, device=cuda))
    want = float(torch.cat([p.grad for p in params]).double().norm())
    twice = [params[0], none, params[1], params[0]]
    got = qb.clip_grad_norm(iter(twice), 1e9)
    assert abs(float(got) - want) <= 16 * 2.0 ** -24 * want
    one = float(qb.clip_grad_norm(params[0], 1e9))
    assert abs(one - float(params[0].grad.double().norm())) <= 16 * 2.0 ** -24 * one
    assert float(qb.clip_grad_norm([none], 1.0)) == 0.0
    assert float(qb.clip_grad_norm([], 1.0)) == 0.0


def test_same_gradients_give_the_same_bits(qb, cuda):
    shapes = [(1000, 333)] * 9 + [(77,)] * 40
    runs = []
    for _ in range(3):
        params = params_of(shapes, (torch.bfloat16, torch.float32), cuda)
        runs.append((qb.clip_grad_norm(params, 0.3), [p.grad for p in params]))
    for norm, grads in runs[1:]:
        assert torch.equal(norm, runs[0][0])
        assert all(torch.equal(a, b) for a, b in zip(grads, runs[0][1]))


def test_captured_and_replayed(qb, cuda):
    params = params_of([(5000,), (64, 64)], (torch.float32,), cuda)
    kept = [p.grad.clone() for p in params]
    want = qb.clip_grad_norm(params, 1.0)
    clipped = [p.grad.clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = qb.clip_grad_norm(params, 1.0)
    for _ in range(3):
        for p, g in zip(params, kept):
            p.grad.copy_(g)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        assert all(torch.equal(p.grad, c) for p, c in zip(params, clipped))


def test_refusals(qb, cuda):
    params = params_of([(30,)], (torch.float32,), cuda)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            qb.clip_grad_norm(params, bad)
    with pytest.raises(TypeError):
        qb.clip_grad_norm(3, 1.0)
    host = params_of([(30,)], (torch.float32,), "cpu")
    with pytest.raises(RuntimeError):
        qb.clip_grad_norm(host, 1.0)
    with pytest.raises(RuntimeError):
        qb.clip_grad_norm(params + host, 1.0)
    with pytest.raises(RuntimeError):
        qb.clip_grad_norm(params_of([(30,)], (torch.float64,), cuda), 1.0)
    s = torch.nn.Parameter(torch.zeros(4, 4, device=cuda))
    s.grad = torch.eye(4, device=cuda).to_sparse()
    with pytest.raises(RuntimeError):
        qb.clip_grad_norm([s], 1.0)
