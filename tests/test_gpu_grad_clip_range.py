"""Gradient clipping: values whose squares leave fp32's range, gradients that cannot
be written."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def param(grad):
    p = torch.nn.Parameter(torch.empty_like(grad))
    p.grad = grad
    return p


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std", [1e-18, 1e-20, 1e-22, 1e-24, 1e-30, 1e-36])
def test_norm_of_small_gradients(qb, cuda, dtype, std):
    """Whole aligned pieces, their rests and unaligned tensors alike."""
    g = torch.Generator().manual_seed(1)
    flat = (torch.randn(60001, generator=g) * std).to(dtype).to(cuda)
    for grads in ([flat], [flat[1:]], [flat[:8192], flat[8192:8200], flat[8201:50000]],
                  [flat[:16384], torch.zeros(16384, dtype=dtype, device=cuda)]):
        want = float(torch.cat([v.double() for v in grads]).norm())
        got = float(qb.clip_grad_norm([param(v.clone() if v.data_ptr() % 16 == 0 else v) for v in grads], 1.0))
        # (as for other sizes: squares of a thread's share of a piece in fp32, 16 terms at most)
        assert abs(got - want) <= 16 * 2.0 ** -24 * want


def test_a_refused_call_changes_nothing(qb, cuda):
    """Gradients that cannot be written in place, among others that can."""
    def first():
        return param(torch.full((5000,), 3.0, device=cuda))

    shared = torch.nn.Parameter(torch.zeros(40, 30, device=cuda))
    shared.grad = torch.ones(1, 30, device=cuda).expand(40, 30)  # rows share their memory
    with torch.inference_mode():
        frozen = torch.ones(40, device=cuda)
    made = torch.nn.Parameter(torch.zeros(40, device=cuda))
    made.grad = frozen
    for bad in (shared, made):
        for order in (0, 1):
            good = first()
            before = bad.grad.clone()
            with pytest.raises(RuntimeError):
                qb.clip_grad_norm([good, bad] if order else [bad, good], 0.5)
            assert torch.equal(good.grad, torch.full_like(good.grad, 3.0))
            assert torch.equal(bad.grad, before)
