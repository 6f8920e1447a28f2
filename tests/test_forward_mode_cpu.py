"""A forward-mode tangent through the quaternion layer is refused, not dropped."""

import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.mark.parametrize("which", range(8))
def test_a_tangent_is_refused(qb, which):
    shapes = [(2, 16)] + [(3, 4)] * 4 + [(12,), (2, 16), (12, 2)]
    with fwd.dual_level():
        t = [torch.randn(*s) for s in shapes]
        t[which] = fwd.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            qb.fused_quaternion_linear(*t, 2.0)
        # plain tensors inside a level get the usual answer (here: no CPU path)
        with pytest.raises(RuntimeError, match="CUDA"):
            qb.fused_quaternion_linear(*(fwd.unpack_dual(v).primal for v in t), 2.0)
