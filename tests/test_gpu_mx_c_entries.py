"""The C entries of the 4-bit layer on rows with gaps and a workspace of the asked
size: the results of the Python calls, nothing else written."""

import ctypes

import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu

CODE = {"f32": 0, "bf16": 1, "f16": 2}
GUARD = 4096


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


class Workspace:
    """`size` bytes at the front of a buffer whose rest is watched."""

    def __init__(self, size):
        self.size = size
        self.bytes = torch.full((size + GUARD,), 0xA5, dtype=torch.uint8, device="cuda")

    def whole(self):
        return bool((self.bytes[self.size:] == 0xA5).all())


def asked(fn, *args):
    n = ctypes.c_size_t(0)
    assert fn(*args, ctypes.byref(n)) == 0
    return n.value


def gapped(M, n, gap, dtype):
    """Rows of n elements with `gap` more between them, all marked."""
    buf = torch.full((M, n + gap), -77.0, dtype=dtype, device="cuda")
    return buf, buf[:, :n]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M", [1, 2, 7, 16, 30, 64, 65, 200])
@pytest.mark.parametrize("fin,fout,rank,gap", [(68, 36, 5, 4), (512, 260, 40, 8), (256, 192, 41, 12), (128, 64, 0, 20)])
def test_strided_rows_and_exact_workspaces(qb, cuda, dtype, M, fin, fout, rank, gap):
    lib = qb._lib.load()
    d = ref.draw(dtype, M, fin, fout, rank=rank, bias=True, seed=M + rank, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    T, K_g, N_g, code = ref.TORCH[dtype], fin // 4, fout // 4, CODE[dtype]
    gy = ref.draw(dtype, M, fout, 4, seed=5, device=cuda)["x"]
    leaves = {k: d[k].clone().requires_grad_(True) for k in ("x", "bias", "a", "b") if d[k] is not None}
    want = qb.mx_quaternion_linear(leaves["x"], q, leaves["bias"], leaves.get("a"), leaves.get("b"), d["scale"])
    grads = dict(zip(leaves, torch.autograd.grad(want, list(leaves.values()), gy)))

    xs, x = gapped(M, fin, gap, T)
    x.copy_(d["x"])
    ybuf, y = gapped(M, fout, gap, T)
    ws = Workspace(asked(lib.qlin_mx_workspace_size, code, M, K_g, N_g, rank))
    st = lib.qlin_mx_forward(code, ptr(xs), fin + gap, ptr(q.data), ptr(d["bias"]), ptr(d["a"]), ptr(d["b"]), rank,
                             d["scale"], ptr(ybuf), fout + gap, M, K_g, N_g, ptr(ws.bytes), ws.size, stream())
    assert st == 0 and ws.whole()
    assert torch.equal(y, want.detach())
    assert bool((ybuf[:, fout:] == -77).all())

    gs, g = gapped(M, fout, gap, T)
    g.copy_(gy)
    ws = Workspace(asked(lib.qlin_mx_backward_workspace_size, code, M, K_g, N_g, rank))
    for only in (None, "x", "a", "b", "bias"):
        if only in ("a", "b") and rank == 0:
            continue
        dbuf, dx = gapped(M, fin, gap, T)
        out = {"x": dbuf, "bias": torch.empty(fout, dtype=T, device=cuda)}
        if rank:
            out.update(a=torch.empty_like(d["a"]), b=torch.empty_like(d["b"]))
        if only:
            out = {only: out[only]}
        st = lib.qlin_mx_backward(code, ptr(gs), fout + gap, ptr(xs), fin + gap, ptr(q.data), ptr(d["a"]), ptr(d["b"]),
                                  rank, d["scale"], ptr(out.get("x")), fin + gap, ptr(out.get("a")), ptr(out.get("b")),
                                  ptr(out.get("bias")), M, K_g, N_g, ptr(ws.bytes), ws.size, stream())
        assert st == 0 and ws.whole(), only
        for k, t in out.items():
            got = dx if k == "x" else t
            if only is None:
                assert torch.equal(got, grads[k]), k
            else:  # (alone a bias sum runs in another order)
                assert ref.rel(ref.f64(got), ref.f64(grads[k])) <= 2 * ref.tolerance(dtype, M), (only, k)
        if "x" in out:
            assert bool((dbuf[:, fin:] == -77).all())
