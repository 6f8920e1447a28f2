"""4-bit weights and gradient clipping without a device: sizes, refusals of
the C entries and of the Python calls, the test oracle itself."""

import ctypes

import numpy as np
import pytest
import torch

import mx_reference as ref


def size(fn, *args):
    n = ctypes.c_size_t(0)
    assert fn(*args, ctypes.byref(n)) == 0
    return n.value


def test_oracle_rounding():
    w = np.zeros(32)
    w[:10] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7.9, -0.26]
    assert ref.quantized_values(w)[:10].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 6, -0.5]
    assert ref.quantized_values(w / 16)[:9].tolist() == [v / 16 for v in (6, 0, 1, 1, 2, 2, 4, 4, 6)]
    # 8 starts the next scale: steps of 1 in place of 0.5 around 1
    assert ref.quantized_values(np.array([8.0, 1.25, 0.5, 0.51]))[:4].tolist() == [8, 1, 0, 1]


def test_real_matrix_is_hamiltons_table(oracle):
    rng = np.random.default_rng(0)
    w, x = rng.standard_normal((4, 3, 5)), rng.standard_normal((2, 20))
    w, x = w.astype(np.float32), x.astype(np.float32)  # the oracle takes fp32 values
    want = oracle.forward_rows(x, *w)
    w, x = w.astype(np.float64), x.astype(np.float64)
    assert np.allclose(ref.layer(x, w), want, rtol=1e-12, atol=1e-12)


def test_buffer_sizes(qb):
    lib = qb._lib.load()
    f = lib.qlin_mx_weights_size
    assert size(f, 32, 16) == 128 + 1088
    assert size(f, 1, 1) == 128 + 1088
    assert size(f, 33, 17) == 128 + 4 * 1088
    assert size(f, 1024, 1024) == 128 + 64 * 32 * 1088  # 4.25 bits a weight
    n = ctypes.c_size_t(0)
    for k, g in ((0, 4), (4, 0), (-1, 4), (2 ** 40, 4)):
        assert f(k, g, ctypes.byref(n)) == 1
    assert f(4, 4, None) == 8


def test_c_entries_refuse_before_device_use(qb):
    lib = qb._lib.load()
    P, A = None, 256  # A: a non-null address, never dereferenced
    n = ctypes.c_size_t(0)
    # quantise: type, sizes, leading dimension, null, alignment
    assert lib.qlin_mx_quantize(7, A, A, A, A, 8, 8, 8, A, P) == 2
    assert lib.qlin_mx_quantize(0, A, A, A, A, 8, 0, 8, A, P) == 1
    assert lib.qlin_mx_quantize(0, A, A, A, A, 7, 8, 8, A, P) == 1
    assert lib.qlin_mx_quantize(0, A, A, P, A, 8, 8, 8, A, P) == 8
    assert lib.qlin_mx_quantize(0, A, A, A, A, 8, 8, 8, A + 64, P) == 3
    assert lib.qlin_mx_dequantize(7, A, 8, 8, A, A, A, A, 8, P) == 2
    assert lib.qlin_mx_dequantize(0, A, 8, 8, A, A, A, A, 7, P) == 1
    assert lib.qlin_mx_dequantize(0, P, 8, 8, A, A, A, A, 8, P) == 8
    assert lib.qlin_mx_dequantize(0, A + 1, 8, 8, A, A, A, A, 8, P) == 3
    # forward
    for args, want in (
            ((7, A, 32, A, P, P, P, 0, 0.0, A, 32, 2, 8, 8), 2),
            ((1, A, 31, A, P, P, P, 0, 0.0, A, 32, 2, 8, 8), 1),
            ((1, A, 32, A, P, P, P, 0, 0.0, A, 31, 2, 8, 8), 1),
            ((1, A, 32, A, P, P, P, -1, 0.0, A, 32, 2, 8, 8), 1),
            ((1, A, 32, A, P, P, P, 0, 0.0, A, 32, -2, 8, 8), 1),
            ((1, A, 32, A, P, P, P, 4, 1.0, A, 32, 2, 8, 8), 8),
            ((1, P, 32, A, P, P, P, 0, 0.0, A, 32, 2, 8, 8), 8),
            ((1, A, 32, P, P, P, P, 0, 0.0, A, 32, 2, 8, 8), 8),
            ((1, A, 32, A + 16, P, P, P, 0, 0.0, A, 32, 2, 8, 8), 3),
            ((1, P, 32, P, P, P, P, 0, 0.0, P, 32, 0, 8, 8), 0)):
        assert lib.qlin_mx_forward(*args, P, 0, P) == want, args
    # a workspace that is missing, and one that is not aligned
    need = size(lib.qlin_mx_workspace_size, 1, 300, 64, 64, 8)
    assert need > 0
    big = (1, A, 256, A, P, A, A, 8, 1.0, A, 256, 300, 64, 64)
    assert lib.qlin_mx_forward(*big, P, need, P) == 4
    assert lib.qlin_mx_forward(*big, A, need - 1, P) == 4
    assert lib.qlin_mx_forward(*big, A + 8, need, P) == 4
    assert size(lib.qlin_mx_workspace_size, 1, 0, 64, 64, 8) == 0
    assert lib.qlin_mx_workspace_size(9, 1, 8, 8, 0, ctypes.byref(n)) == 2
    assert lib.qlin_mx_workspace_size(1, 1, 8, 8, 0, None) == 8
    # backward
    for args, want in (
            ((7, A, 32, A, 32, A, P, P, 0, 0.0, A, 32, P, P, P, 2, 8, 8), 2),
            ((1, A, 31, A, 32, A, P, P, 0, 0.0, A, 32, P, P, P, 2, 8, 8), 1),
            ((1, A, 32, A, 32, A, P, P, 0, 0.0, A, 31, P, P, P, 2, 8, 8), 1),
            ((1, A, 32, A, 31, A, A, A, 4, 1.0, P, 0, A, A, P, 2, 8, 8), 1),
            ((1, A, 32, A, 32, A, P, P, 0, 0.0, A, 32, A, P, P, 2, 8, 8), 8),
            ((1, P, 32, A, 32, A, P, P, 0, 0.0, A, 32, P, P, P, 2, 8, 8), 8),
            ((1, A, 32, A, 32, P, P, P, 0, 0.0, A, 32, P, P, P, 2, 8, 8), 8),
            ((1, A, 32, P, 32, A, A, A, 4, 1.0, P, 32, A, P, P, 2, 8, 8), 8),
            ((1, A, 32, A, 32, A + 4, P, P, 0, 0.0, A, 32, P, P, P, 2, 8, 8), 3),
            ((1, P, 32, P, 32, P, P, P, 0, 0.0, P, 32, P, P, P, 0, 8, 8), 0)):
        assert lib.qlin_mx_backward(*args, P, 0, P) == want, args
    need = size(lib.qlin_mx_backward_workspace_size, 1, 300, 64, 64, 8)
    assert lib.qlin_mx_backward(1, A, 256, A, 256, A, A, A, 8, 1.0, A, 256, A, A, P, 300, 64, 64, A, need - 1, P) == 4
    # clipping
    one = (ctypes.c_void_p * 1)(A)
    f32, bad = (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(5)
    ten, neg = (ctypes.c_int64 * 1)(10), (ctypes.c_int64 * 1)(-1)
    need = size(lib.qlin_grad_clip_workspace_size, 1)
    clip = lib.qlin_grad_clip
    assert clip(-1, one, ten, f32, 1.0, A, A, need, P) == 1
    assert clip(1, one, neg, f32, 1.0, A, A, need, P) == 1
    assert clip(1, one, ten, bad, 1.0, A, A, need, P) == 2
    assert clip(1, one, ten, f32, 1.0, P, A, need, P) == 8
    assert clip(1, one, ten, f32, -1.0, A, A, need, P) == 8
    assert clip(1, one, ten, f32, float("nan"), A, A, need, P) == 8
    assert clip(1, (ctypes.c_void_p * 1)(None), ten, f32, 1.0, A, A, need, P) == 8
    assert clip(1, (ctypes.c_void_p * 1)(A + 2), ten, f32, 1.0, A, A, need, P) == 3
    assert clip(1, one, ten, f32, 1.0, A, A, need - 1, P) == 4
    assert clip(1, one, ten, f32, 1.0, A, P, need, P) == 4


def test_cpu_tensors_are_refused(qb):
    w = [torch.zeros(4, 8) for _ in range(4)]
    with pytest.raises(RuntimeError):
        qb.quantize_quaternion_weights(*w)
    n = size(qb._lib.load().qlin_mx_weights_size, 8, 4)
    q = qb.MXQuaternionWeights(torch.zeros(n, dtype=torch.uint8), 4, 8)
    with pytest.raises(RuntimeError):
        qb.mx_quaternion_linear(torch.zeros(2, 32), q)
    with pytest.raises(ValueError):
        qb.mx_quaternion_linear(torch.zeros(2, 30), q)
    with pytest.raises(RuntimeError):
        q.dequantize()
    layer = qb.MXQuaternionLinear(32, 16, q.data, torch.zeros(16), torch.float16)
    assert set(layer.state_dict()) == {"weight_mx", "bias"}
    adapted = qb.LoRAQuaternionLinear(layer, rank=2)
    assert adapted.lora_A.dtype == torch.float16 and adapted.lora_A.shape == (2, 32)
    assert qb.LoRAQuaternionLinear(layer.float(), rank=2).lora_A.dtype == torch.float32
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError):
        qb.clip_grad_norm([p], 1.0)
    assert float(qb.clip_grad_norm([torch.nn.Parameter(torch.zeros(3))], 1.0)) == 0.0
