"""4-bit quaternion weights: a frozen base at a quarter of its 16-bit bytes.

The four weight components are held as OCP microscaling MXFP4: e2m1 elements
(0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) with one power-of-two scale
for every 32 consecutive input quaternions of a component row, about 4.25
bits a weight.  They serve inference and, with
:class:`~.lora.LoRAQuaternionLinear` on top, fine-tuning: the 4-bit base is a
constant, gradients reach the input, the bias and the LoRA factors.

``x``, bias, LoRA factors and outputs are float32, bfloat16 or float16, sums
are fp32; with float32 inputs the products are those of fp32 arithmetic.  The
weights enter exactly; with float16 inputs of three tokens or more that holds
for blocks whose scale is at least 2^-36 of the layer's largest (all float16
weights below 8192), others are rounded at 2^-37 of it.  CPU tensors raise
``RuntimeError`` -- there is no CPU path.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .linear import QuaternionLinear

__all__ = [
    "MXQuaternionWeights",
    "MXQuaternionLinear",
    "quantize_quaternion_weights",
    "mx_quaternion_linear",
    "quantize_model",
]


def _ext():
    if _lib._torch_ext is None:
        _lib.load()
        if _lib._torch_ext is None:
            raise RuntimeError("the torch extension (lib/_qlin_torch*.so) is not built; run "
                               "`python quaternion-based-math-1_b200/build.py`")
    return _lib._torch_ext


class MXQuaternionWeights:
    """The 4-bit weights of one layer: ``data``, an opaque uint8 buffer in the
    kernels' layout, and the layer's ``out_groups`` and ``in_groups``."""

    __slots__ = ("data", "out_groups", "in_groups")

    def __init__(self, data: torch.Tensor, out_groups: int, in_groups: int):
        self.data = data
        self.out_groups = out_groups
        self.in_groups = in_groups

    def dequantize(self, dtype: torch.dtype = torch.float32):
        """The values the codes stand for, rounded to ``dtype``: ``(wr, wi, wj, wk)``."""
        return tuple(_ext().mx_dequantize(self.data, self.out_groups, self.in_groups, dtype))

    def __repr__(self) -> str:
        return (f"MXQuaternionWeights(out_groups={self.out_groups}, in_groups={self.in_groups}, "
                f"device={self.data.device})")


def quantize_quaternion_weights(wr, wi, wj, wk) -> MXQuaternionWeights:
    """The components ``[out_groups, in_groups]`` as 4-bit weights.

    Every run of 32 input quaternions of a component row gets the scale
    ``2^(floor(log2(max |w|)) - 2)``; elements are rounded to nearest, ties to
    even, and saturate at 6 scales.  A run that holds an infinity or a NaN
    stands for NaNs.
    """
    return MXQuaternionWeights(_ext().mx_quantize(wr, wi, wj, wk), wr.shape[0], wr.shape[1])


def mx_quaternion_linear(x, weights: MXQuaternionWeights, bias=None, lora_a=None, lora_b=None,
                         lora_scale: float = 0.0):
    """``quaternion_linear(x) + bias + lora_scale * (x A^T) B^T`` on 4-bit weights.

    ``x``: ``[..., in_features]``; bias ``[out_features]``; LoRA A
    ``[r, in_features]`` and B ``[out_features, r]``, all of x's dtype.
    Differentiable once in x, bias, A and B, in reverse mode only (a forward-mode
    tangent raises ``RuntimeError``).
    """
    return _ext().mx_linear(x, weights.data, weights.out_groups, weights.in_groups, bias, lora_a, lora_b,
                            float(lora_scale))


class MXQuaternionLinear(nn.Module):
    """A :class:`~.linear.QuaternionLinear` with its weights frozen in 4 bits.

    Buffer ``weight_mx`` (the codes and scales) and parameter ``bias``; made
    by :meth:`from_linear` or :func:`quantize_model`.  A LoRA adapter goes on
    top with :class:`~.lora.LoRAQuaternionLinear`.
    """

    def __init__(self, in_features: int, out_features: int, weight_mx: torch.Tensor,
                 bias: torch.Tensor | None = None, dtype: torch.dtype | None = None):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.in_groups = in_features // 4
        self.out_groups = out_features // 4
        self.register_buffer("weight_mx", weight_mx)
        # the type an adapter's factors take; follows .to() and the like
        self.register_buffer("type_of", torch.empty(0, dtype=dtype, device=weight_mx.device), persistent=False)
        if bias is None:
            self.register_parameter("bias", None)
        else:
            self.bias = nn.Parameter(bias.detach().clone())

    @classmethod
    def from_linear(cls, layer: QuaternionLinear) -> "MXQuaternionLinear":
        q = quantize_quaternion_weights(*(w.detach() for w in (layer.wr, layer.wi, layer.wj, layer.wk)))
        return cls(layer.in_features, layer.out_features, q.data, layer.bias, layer.wr.dtype)

    @property
    def weights(self) -> MXQuaternionWeights:
        return MXQuaternionWeights(self.weight_mx, self.out_groups, self.in_groups)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return mx_quaternion_linear(x, self.weights, self.bias)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, weights=mxfp4")


# what a replaced layer hands on besides its parameters: the hooks around its forward and backward
_HOOKS = ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks",
          "_forward_pre_hooks_with_kwargs", "_backward_hooks", "_backward_pre_hooks", "_is_full_backward_hook")


def quantize_model(model: nn.Module):
    """Replace every ``QuaternionLinear`` of ``model`` (LoRA bases too) by an
    ``MXQuaternionLinear`` in place; return the replaced names.  A layer that
    appears under several names stays shared; forward and backward hooks of a
    layer go over to its replacement (hooks on its state dict do not).

    Left as they are: subclasses with a ``forward`` of their own, and layers
    that hold their weights in another form (``FactorizedQuaternionLinear``,
    ``UnitQuaternionLinear``, ``ColumnParallelQuaternionLinear``).  A ``model``
    that is itself a ``QuaternionLinear`` cannot be replaced in place:
    ``ValueError`` (:meth:`MXQuaternionLinear.from_linear` makes its
    replacement).
    """
    if isinstance(model, QuaternionLinear):
        raise ValueError("the model is a QuaternionLinear itself and cannot be replaced in place; "
                         "use MXQuaternionLinear.from_linear")
    made: dict[QuaternionLinear, MXQuaternionLinear] = {}
    replaced = []
    for name, mod in list(model.named_modules(remove_duplicate=False)):
        if not isinstance(mod, QuaternionLinear) or type(mod).forward is not QuaternionLinear.forward:
            continue
        if mod not in made:
            made[mod] = MXQuaternionLinear.from_linear(mod)
            made[mod].train(mod.training)
            for hooks in _HOOKS:
                setattr(made[mod], hooks, getattr(mod, hooks))
            if mod.bias is not None:
                made[mod].bias.requires_grad_(mod.bias.requires_grad)
        parent_name, _, leaf = name.rpartition(".")
        setattr(model.get_submodule(parent_name) if parent_name else model, leaf, made[mod])
        replaced.append(name)
    return replaced
