"""The 4-bit quaternion layer in 64 bits (numpy): quantisation by definition,
the layer as the product with the real block matrix, its gradients."""

from __future__ import annotations

import numpy as np
import torch

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# half a step of each type, relative to the value
HALF_STEP = {k: torch.finfo(t).eps / 2 for k, t in TORCH.items()}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def quantized_values(w: np.ndarray) -> np.ndarray:
    """[..., K_g] float -> the values of its 4-bit codes, float64."""
    w = np.asarray(w, np.float64)
    K = w.shape[-1]
    pad = np.zeros((*w.shape[:-1], -K % 32))
    b = np.concatenate((w, pad), -1).reshape(*w.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1, keepdims=True)
    b = np.where(bad, 0.0, b)
    top = np.abs(b).max(-1, keepdims=True)
    e = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)
    unit = np.ldexp(1.0, np.maximum(e, -127))
    a = np.abs(b) / unit
    # nearest grid value; of two equally near ones that with the even index
    d = np.abs(a[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    index = np.where(near, np.arange(8) + 8 * (np.arange(8) % 2), 99).argmin(-1)
    out = np.sign(b) * GRID[index] * unit
    return np.where(bad, np.nan, out).reshape(*w.shape[:-1], -1)[..., :K]


SIGN = ((1, -1, -1, -1), (1, 1, -1, 1), (1, 1, 1, -1), (1, -1, 1, 1))


def real_matrix(w: np.ndarray) -> np.ndarray:
    """[4, N_g, K_g] -> [4 N_g, 4 K_g]: row 4o+a, column 4i+q is +-W_{a^q}[o, i]."""
    _, n, k = w.shape
    out = np.empty((n, 4, k, 4))
    for a in range(4):
        for q in range(4):
            out[:, a, :, q] = SIGN[a][q] * w[a ^ q]
    return out.reshape(4 * n, 4 * k)


def f64(t) -> np.ndarray | None:
    return None if t is None else t.detach().double().cpu().numpy()


def layer(x, values, bias=None, a=None, b=None, scale=0.0):
    y = x @ real_matrix(values).T
    if a is not None:
        y = y + scale * (x @ a.T) @ b.T
    return y if bias is None else y + bias


def gradients(gy, x, values, a=None, b=None, scale=0.0):
    dx = gy @ real_matrix(values)
    da = db = None
    if a is not None:
        up = scale * (gy @ b)
        dx = dx + up @ a
        da, db = up.T @ x, scale * gy.T @ (x @ a.T)
    return dx, da, db, gy.sum(0)


def rel(got, want) -> float:
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    n = np.linalg.norm(want)
    d = np.linalg.norm(got - want)
    return float(d / n) if n else float(d)


def tolerance(dtype: str, terms: int, roundings: int = 1) -> float:
    """2-norm of the error over that of the result: `roundings` roundings to
    the type (half a step each), and fp32 sums of `terms` terms whose
    rounding errors (at most 2^-23 each, truncation included) add up as
    independent ones, the running sum being of the result's size."""
    return roundings * HALF_STEP[dtype] + 2.0 ** -23 * (2 + terms) ** 0.5


def draw(dtype, M, fin, fout, rank=0, bias=False, seed=0, device="cuda", w_std=None):
    """Inputs of one layer as tensors of the type."""
    g = torch.Generator().manual_seed(seed)

    def t(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, dtype=torch.float64) * std).to(TORCH[dtype]).to(device)

    w = [t(fout // 4, fin // 4, std=w_std or fin ** -0.5) for _ in range(4)]
    return dict(x=t(M, fin), w=w, bias=t(fout, std=0.1) if bias else None,
                a=t(rank, fin, std=0.05) if rank else None, b=t(fout, rank, std=0.05) if rank else None,
                scale=2.0 if rank else 0.0)
