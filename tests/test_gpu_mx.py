"""4-bit quaternion weights on the device against the definition in 64 bits."""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import mx_reference as ref

pytestmark = pytest.mark.gpu


def values_of(q):
    return np.stack([ref.f64(w) for w in q.dequantize(torch.float32)])


# ---------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 32), (17, 33), (5, 250), (64, 192), (259, 250), (130, 1024)])
def test_quantisation_is_the_definition(qb, cuda, dtype, n, k):
    w = ref.draw(dtype, 1, 4 * k, 4 * n, seed=n + k, device=cuda)["w"]
    q = qb.quantize_quaternion_weights(*w)
    want = ref.quantized_values(np.stack([ref.f64(t) for t in w]))
    assert np.array_equal(values_of(q), want)
    for d in ("f32", "bf16", "f16"):
        got = q.dequantize(ref.TORCH[d])
        for g, v in zip(got, want):  # one rounding of the value
            assert torch.equal(g.cpu(), torch.from_numpy(v).to(ref.TORCH[d]))


def test_quantisation_ties_and_extremes(qb, cuda):
    rows = []
    # every midpoint and value of the grid at several scales (6 fixes the scale)
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9])
    for e in (-126, -100, -3, 0, 5, 100, 125):
        r = np.zeros(32)
        r[: len(mids)] = mids
        r[10:18] = -ref.GRID
        r[20:29] = np.nextafter(mids.astype(np.float32), np.float32(9)).astype(np.float64)
        rows.append(np.ldexp(r, e))
    rows.append(np.zeros(32))
    rows.append(np.full(32, 2.0 ** -149))                       # the smallest fp32 values
    rows.append(np.linspace(-1, 1, 32) * 2.0 ** -125)
    rows.append(np.full(32, float(np.finfo(np.float32).max)))
    with np.errstate(all="ignore"):
        m = np.stack(rows).astype(np.float32)
    w = [torch.from_numpy(np.roll(m, p, 0)).to(cuda) for p in range(4)]
    q = qb.quantize_quaternion_weights(*w)
    assert np.array_equal(values_of(q), ref.quantized_values(np.stack([ref.f64(t) for t in w])))


def test_blocks_with_infinities_or_nans_stand_for_nans(qb, cuda):
    w = ref.draw("f32", 1, 4 * 96, 4 * 20, seed=3, device=cuda)["w"]
    w[1][3, 40] = float("inf")
    w[2][7, 95] = float("nan")
    q = qb.quantize_quaternion_weights(*w)
    got = values_of(q)
    bad = np.zeros_like(got, bool)
    bad[1, 3, 32:64] = True
    bad[2, 7, 64:96] = True
    assert np.array_equal(np.isnan(got), bad)
    want = ref.quantized_values(np.stack([ref.f64(t) for t in w]))
    assert np.array_equal(got[~bad], want[~bad])
    # only the outputs that read those weights are NaN
    for M in (1, 9, 130):
        x = torch.ones(M, 384, device=cuda)
        for dt in (torch.float32, torch.bfloat16, torch.float16):
            y = qb.mx_quaternion_linear(x.to(dt), q).isnan().cpu().numpy()
            rows = np.zeros(80, bool)
            rows[12:16] = rows[28:32] = True
            assert np.array_equal(y, np.broadcast_to(rows, y.shape)), (M, dt)


def test_quantisation_of_strided_components(qb, cuda):
    base = torch.randn(40, 77, 4, device=cuda)
    views = [base[..., p] for p in range(4)]            # element stride 4
    wide = [torch.randn(40, 90, device=cuda)[:, 5:82] for _ in range(4)]  # row stride 90, unaligned
    mixed = [wide[0], wide[1].contiguous(), wide[2], wide[3]]
    turned = [torch.randn(77, 40, device=cuda).t() for _ in range(4)]
    for w in (views, wide, mixed, turned):
        got = values_of(qb.quantize_quaternion_weights(*w))
        assert np.array_equal(got, ref.quantized_values(np.stack([ref.f64(t) for t in w])))


# --------------------------------------------------------------------- forward
def check_forward(qb, d, dtype, roundings):
    q = qb.quantize_quaternion_weights(*d["w"])
    y = qb.mx_quaternion_linear(d["x"], q, d["bias"], d["a"], d["b"], d["scale"])
    assert y.dtype == d["x"].dtype and y.shape == (*d["x"].shape[:-1], 4 * q.out_groups)
    want = ref.layer(ref.f64(d["x"]), values_of(q), *(ref.f64(d[k]) for k in ("bias", "a", "b")), d["scale"])
    K = d["x"].shape[-1]
    assert ref.rel(ref.f64(y), want) <= ref.tolerance(dtype, K, roundings)
    return y, want


# LoRA: the down projection is rounded to 16 bits once more
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64, 65, 100, 129, 300])
def test_forward_over_token_counts(qb, cuda, dtype, M):
    check_forward(qb, ref.draw(dtype, M, 512, 320, bias=True, seed=M, device=cuda), dtype, 1)
    check_forward(qb, ref.draw(dtype, M, 512, 320, rank=8, seed=M, device=cuda), dtype, 2)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("fin,fout", [(4, 4), (4, 260), (36, 4), (100, 68), (252, 132), (1000, 1036), (2056, 60),
                                      (768, 2304)])
@pytest.mark.parametrize("M", [1, 6, 40, 70, 260])
def test_forward_over_odd_sizes(qb, cuda, dtype, fin, fout, M):
    check_forward(qb, ref.draw(dtype, M, fin, fout, bias=True, rank=5, seed=fin + fout + M, device=cuda), dtype, 2)


@pytest.mark.parametrize("rank", [1, 4, 7, 16, 32, 33, 64, 65, 100, 130, 300])
@pytest.mark.parametrize("M", [1, 12, 150])
def test_forward_over_ranks(qb, cuda, rank, M):
    check_forward(qb, ref.draw("bf16", M, 256, 192, rank=rank, seed=rank, device=cuda), "bf16", 2)
    check_forward(qb, ref.draw("f32", M, 256, 192, rank=rank, seed=rank, device=cuda), "f32", 2)


@pytest.mark.parametrize("dtype,M,fin,fout,rank", [
    ("bf16", 1, 4096, 4096, 32), ("bf16", 1, 5120, 27648, 0), ("f16", 16, 4096, 4096, 32),
    ("bf16", 2, 11008, 4096, 16), ("bf16", 16, 11008, 4096, 16), ("f32", 3, 4096, 4096, 8)])
def test_forward_of_served_layers(qb, cuda, dtype, M, fin, fout, rank):
    check_forward(qb, ref.draw(dtype, M, fin, fout, rank=rank, bias=True, seed=7, device=cuda), dtype, 2)


def test_forward_over_far_scales(qb, cuda):
    """Blocks whose scales are 2^20 apart (bf16, fp32) and 2^10 apart (fp16: all
    products representable)."""
    for dtype, spread in (("bf16", 20), ("f32", 20), ("f16", 10)):
        d = ref.draw(dtype, 1, 1024, 256, seed=5, device=cuda)
        e = torch.arange(8, device=cuda).float().mul(-spread / 7).round().exp2().repeat_interleave(32)
        d["w"] = [(w.float() * e).to(w.dtype) for w in d["w"]]
        for M in (1, 8, 40, 200):
            d["x"] = ref.draw(dtype, M, 1024, 256, seed=M, device=cuda)["x"]
            check_forward(qb, d, dtype, 1)


@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** 60])
def test_forward_of_very_small_and_large_weights(qb, cuda, factor):
    for dtype in ("bf16", "f32"):
        for M in (1, 8, 200):
            d = ref.draw(dtype, M, 256, 256, seed=9, device=cuda)
            d["w"] = [w * factor for w in d["w"]]
            check_forward(qb, d, dtype, 1)


def test_zero_weights(qb, cuda):
    w = [torch.zeros(20, 40, device=cuda) for _ in range(4)]
    q = qb.quantize_quaternion_weights(*w)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        bias = torch.randn(80, device=cuda).to(dt)
        for M in (1, 5, 100):
            x = torch.randn(M, 160, device=cuda).to(dt)
            assert torch.equal(qb.mx_quaternion_linear(x, q, bias), bias.expand(M, 80))


def test_wide_ranging_inputs_fp32(qb, cuda):
    """fp32 inputs keep fp32's range and precision: values near its ends, and
    ones whose low bits matter."""
    d = ref.draw("f32", 4, 128, 64, seed=1, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    v = values_of(q)
    for f in (2.0 ** -100, 2.0 ** 120):
        x = d["x"] * f
        assert ref.rel(ref.f64(qb.mx_quaternion_linear(x, q)) / f, ref.layer(ref.f64(x) / f, v)) <= ref.tolerance("f32", 128)
    x = 1 + d["x"] * 2.0 ** -20
    assert ref.rel(ref.f64(qb.mx_quaternion_linear(x, q)), ref.layer(ref.f64(x), v)) <= ref.tolerance("f32", 128)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M", [1, 2, 8, 40, 200])
def test_nonfinite_tokens_stay_in_their_rows(qb, cuda, dtype, M):
    d = ref.draw(dtype, M, 256, 128, rank=8, bias=True, seed=2, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    args = (q, d["bias"], d["a"], d["b"], d["scale"])
    clean = qb.mx_quaternion_linear(d["x"], *args)
    x = d["x"].clone()
    x[M // 2, 17] = float("nan")
    got = qb.mx_quaternion_linear(x, *args)
    keep = torch.arange(M, device=cuda) != M // 2
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[M // 2].isnan().all())
    x[M // 2, 17] = float("inf")
    got = qb.mx_quaternion_linear(x, *args)
    assert torch.equal(got[keep], clean[keep])
    assert not bool(got[M // 2].isfinite().all())


def test_layouts_of_x(qb, cuda):
    for dtype in ("bf16", "f16", "f32"):
        d = ref.draw(dtype, 24, 136, 72, seed=4, device=cuda)
        q = qb.quantize_quaternion_weights(*d["w"])
        x = d["x"]
        want = qb.mx_quaternion_linear(x, q)
        assert torch.equal(qb.mx_quaternion_linear(x.view(2, 3, 4, 136), q), want.view(2, 3, 4, 72))
        assert torch.equal(qb.mx_quaternion_linear(x[0], q), qb.mx_quaternion_linear(x[:1], q)[0])
        wide = torch.full((24, 300), float("nan"), dtype=x.dtype, device=cuda)
        for at in (0, 1, 3, 8):  # rows with a stride, and unaligned starts
            wide[:, at:at + 136] = x
            assert torch.equal(qb.mx_quaternion_linear(wide[:, at:at + 136], q), want), (dtype, at)
            wide.fill_(float("nan"))
        assert torch.equal(qb.mx_quaternion_linear(x.t().contiguous().t(), q), want)
        assert torch.equal(qb.mx_quaternion_linear(x[:1].expand(24, 136), q), qb.mx_quaternion_linear(x[:1].repeat(24, 1), q))
        for shape in ((0, 136), (2, 0, 136)):
            assert qb.mx_quaternion_linear(x.new_empty(shape), q).shape == (*shape[:-1], 72)


def test_same_inputs_give_the_same_bits(qb, cuda):
    for dtype, M in (("bf16", 1), ("bf16", 16), ("bf16", 300), ("f32", 40)):
        d = ref.draw(dtype, M, 2048, 1024, rank=16, seed=6, device=cuda)
        q = qb.quantize_quaternion_weights(*d["w"])
        assert torch.equal(q.data, qb.quantize_quaternion_weights(*d["w"]).data)
        y = [qb.mx_quaternion_linear(d["x"], q, None, d["a"], d["b"], 2.0) for _ in range(4)]
        assert all(torch.equal(y[0], o) for o in y[1:])


def test_tokens_do_not_depend_on_their_batch(qb, cuda):
    """A token's result next to others is within the rounding of its result alone."""
    d = ref.draw("f32", 40, 640, 320, seed=8, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    all_of = qb.mx_quaternion_linear(d["x"], q)
    one = torch.cat([qb.mx_quaternion_linear(d["x"][m:m + 1], q) for m in range(40)])
    assert ref.rel(ref.f64(all_of), ref.f64(one)) <= 2 * ref.tolerance("f32", 640)


# ------------------------------------------------------------ streams, graphs
def test_streams_and_graphs(qb, cuda):
    for dtype, M in (("bf16", 1), ("bf16", 12), ("f16", 200), ("f32", 20)):
        d = ref.draw(dtype, M, 512, 512, rank=8, bias=True, seed=11, device=cuda)
        q = qb.quantize_quaternion_weights(*d["w"])

        def chain(x):
            for _ in range(3):
                x = qb.mx_quaternion_linear(x, q, d["bias"], d["a"], d["b"], d["scale"])
            return x

        want = chain(d["x"])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = chain(d["x"])
        side.synchronize()
        assert torch.equal(got, want)
        static = torch.zeros_like(d["x"])
        graphs = []
        for _ in range(2):  # two graphs, replayed one after the other and interleaved
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = chain(static)
            graphs.append((g, out))
        for k in range(3):
            static.copy_(d["x"] if k % 2 == 0 else d["x"] * 2)
            want = chain(static.clone())
            for g, out in graphs:
                g.replay()
            torch.cuda.synchronize()
            for g, out in graphs:
                assert torch.equal(out, want)


# ------------------------------------------------------------------- gradients
def check_gradients(qb, d, dtype, M, fout):
    q = qb.quantize_quaternion_weights(*d["w"])
    leaves = {k: d[k].clone().requires_grad_(True) for k in ("x", "bias", "a", "b") if d[k] is not None}
    y = qb.mx_quaternion_linear(leaves["x"], q, leaves.get("bias"), leaves.get("a"), leaves.get("b"), d["scale"])
    g = torch.Generator().manual_seed(99)
    gy = torch.randn(*y.shape, generator=g, dtype=torch.float64).to(y.dtype).to(y.device)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))
    dx, da, db, dbias = ref.gradients(ref.f64(gy), ref.f64(d["x"]), values_of(q), ref.f64(d["a"]), ref.f64(d["b"]),
                                      d["scale"])
    K = d["x"].shape[-1]
    want = {"x": (dx, fout, 2), "a": (da, M + fout, 1), "b": (db, M + K, 1), "bias": (dbias, M, 1)}
    for k, got in grads.items():
        w, terms, roundings = want[k]
        assert got.shape == w.shape and got.dtype == y.dtype
        assert ref.rel(ref.f64(got), w) <= ref.tolerance(dtype, terms, roundings), k


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,fin,fout,rank", [(1, 64, 64, 4), (7, 36, 68, 3), (33, 256, 128, 8), (64, 128, 512, 1),
                                             (130, 1000, 1036, 12), (300, 512, 260, 32), (257, 72, 1024, 64),
                                             (70, 132, 100, 70)])
def test_gradients(qb, cuda, dtype, M, fin, fout, rank):
    check_gradients(qb, ref.draw(dtype, M, fin, fout, rank=rank, bias=True, seed=M, device=cuda), dtype, M, fout)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradients_of_a_training_batch(qb, cuda, dtype):
    check_gradients(qb, ref.draw(dtype, 1024, 1024, 768, rank=16, bias=True, seed=1, device=cuda), dtype, 1024, 768)
    check_gradients(qb, ref.draw(dtype, 90, 512, 768, seed=1, device=cuda), dtype, 90, 768)


def test_gradients_against_differences(qb, cuda):
    """The layer is linear in x, A, B and bias each: a difference over a whole
    step is the derivative, up to fp32 rounding of the two results."""
    d = ref.draw("f32", 9, 96, 64, rank=4, bias=True, seed=3, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    gy = torch.randn(9, 64, device=cuda)
    names = ("x", "bias", "a", "b")
    leaves = {k: d[k].clone().requires_grad_(True) for k in names}

    def f(v):
        return qb.mx_quaternion_linear(v["x"], q, v["bias"], v["a"], v["b"], d["scale"])

    grads = dict(zip(names, torch.autograd.grad(f(leaves), [leaves[k] for k in names], gy)))
    base = f(d)
    for k in names:
        step = torch.randn_like(d[k])
        moved = f({**d, k: d[k] + step})
        want = float(((moved.double() - base.double()) * gy.double()).sum())
        got = float((grads[k].double() * step.double()).sum())
        # 576 outputs of size up to about 5, each off by a few units of 2^-24
        assert abs(got - want) <= 576 ** 0.5 * 5 * 8 * 2.0 ** -24 * 10 + 1e-5 * abs(want), k


def test_only_wanted_gradients(qb, cuda):
    d = ref.draw("bf16", 70, 128, 64, rank=4, bias=True, seed=3, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    for want in ("x", "bias", "a", "b"):
        leaves = {k: d[k].clone().requires_grad_(k == want) for k in ("x", "bias", "a", "b")}
        y = qb.mx_quaternion_linear(leaves["x"], q, leaves["bias"], leaves["a"], leaves["b"], 2.0)
        y.sum().backward()
        for k, t in leaves.items():
            assert (t.grad is not None) == (k == want)
    # without an adapter, and without a bias
    for drop, left in ((("a", "b"), ("x", "bias")), (("bias",), ("x", "a", "b"))):
        leaves = {k: None if k in drop else d[k].clone().requires_grad_(True) for k in ("x", "bias", "a", "b")}
        qb.mx_quaternion_linear(leaves["x"], q, leaves["bias"], leaves["a"], leaves["b"], 2.0).sum().backward()
        assert all(leaves[k].grad is not None for k in left)
    # a broadcast gradient (sum) and one with a stride
    x = d["x"].clone().requires_grad_(True)
    y = qb.mx_quaternion_linear(x, q)
    gy = torch.randn(64, 70, device=cuda).bfloat16().t()
    (g1,) = torch.autograd.grad(y, x, gy, retain_graph=True)
    (g2,) = torch.autograd.grad(y, x, gy.contiguous())
    assert torch.equal(g1, g2)


def test_gradients_of_empty_batches(qb, cuda):
    d = ref.draw("f32", 1, 64, 32, rank=4, bias=True, seed=3, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    leaves = {k: d[k].clone().requires_grad_(True) for k in ("bias", "a", "b")}
    x = torch.empty(0, 64, device=cuda, requires_grad=True)
    y = qb.mx_quaternion_linear(x, q, leaves["bias"], leaves["a"], leaves["b"], 2.0)
    grads = torch.autograd.grad(y, [x, *leaves.values()], torch.empty(0, 32, device=cuda))
    assert grads[0].shape == (0, 64)
    for g in grads[1:]:
        assert not bool(g.any())


def test_twice_differentiating_is_refused(qb, cuda):
    d = ref.draw("f32", 3, 64, 32, seed=3, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    x = d["x"].requires_grad_(True)
    (g,) = torch.autograd.grad(qb.mx_quaternion_linear(x, q).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


# ---------------------------------------------------------------- refusals
def test_refusals(qb, cuda):
    d = ref.draw("bf16", 3, 64, 32, rank=4, bias=True, seed=3, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    f, x = qb.mx_quaternion_linear, d["x"]
    for bad in (x[:, :60], x[:, :62], torch.zeros((), device=cuda)):
        with pytest.raises(ValueError):
            f(bad, q)
    for kw in (dict(bias=d["bias"][:-1]), dict(lora_a=d["a"]), dict(lora_b=d["b"]),
               dict(lora_a=d["a"][:, :-4], lora_b=d["b"]), dict(lora_a=d["a"][:3], lora_b=d["b"])):
        with pytest.raises(ValueError):
            f(x, q, **kw)
    for bad in (x.cpu(), x.double(), x.to(torch.int32)):
        with pytest.raises(RuntimeError):
            f(bad, q)
    with pytest.raises(RuntimeError):
        f(x, q, d["bias"].float())
    with pytest.raises(RuntimeError):
        f(x, q, None, d["a"].half(), d["b"].half())
    W = qb.MXQuaternionWeights
    for data in (q.data[:-1], q.data.view(-1, 2), q.data.to(torch.int8), torch.cat((q.data, q.data))[::2]):
        with pytest.raises(ValueError):
            f(x, W(data, 8, 16))
    with pytest.raises(ValueError):
        f(x, W(q.data, 0, 16))
    with pytest.raises(RuntimeError):
        f(x, W(q.data.cpu(), 8, 16))
    shifted = torch.empty(q.data.numel() + 16, dtype=torch.uint8, device=cuda)[16:]
    with pytest.raises(RuntimeError):  # the buffer's alignment
        f(x, W(shifted.copy_(q.data), 8, 16))
    w = d["w"]
    with pytest.raises(ValueError):
        qb.quantize_quaternion_weights(w[0], w[1], w[2], w[3][:-1])
    with pytest.raises(ValueError):
        qb.quantize_quaternion_weights(*(t[0] for t in w))
    with pytest.raises(ValueError):
        qb.quantize_quaternion_weights(*(t[:0] for t in w))
    with pytest.raises(RuntimeError):
        qb.quantize_quaternion_weights(*(t.cpu() for t in w))
    with pytest.raises(RuntimeError):
        qb.quantize_quaternion_weights(w[0], w[1], w[2], w[3].float())
    with pytest.raises(RuntimeError):
        q.dequantize(torch.float64)


# ------------------------------------------------------------------- modules
def test_modules_and_adapters(qb, cuda):
    torch.manual_seed(0)
    net = torch.nn.Sequential(qb.QuaternionLinear(64, 128, bias=True), torch.nn.GELU(),
                              qb.QuaternionLinear(128, 64)).to(cuda).bfloat16()
    names = qb.quantize_model(net)
    assert names == ["0", "2"] and all(isinstance(net[i], qb.MXQuaternionLinear) for i in (0, 2))
    x = torch.randn(5, 64, device=cuda).bfloat16()
    want = net(x)
    assert qb.inject_lora(net, rank=4) == ["0", "2"]
    assert torch.equal(net(x), want)  # B starts at zero
    assert net[0].lora_A.dtype == net[2].lora_A.dtype == torch.bfloat16
    qb.mark_only_lora_trainable(net)
    with torch.no_grad():
        for _, p in qb.lora_parameters(net):
            p.normal_(std=0.1)
    copy = torch.nn.Sequential(qb.QuaternionLinear(64, 128, bias=True), torch.nn.GELU(),
                               qb.QuaternionLinear(128, 64)).to(cuda).bfloat16()
    qb.quantize_model(copy)
    qb.inject_lora(copy, rank=4)
    copy.load_state_dict(net.state_dict())
    assert torch.equal(copy(x), net(x))
    # adapters put on first, the base quantised afterwards
    other = torch.nn.Sequential(qb.QuaternionLinear(64, 128, bias=True)).to(cuda)
    qb.inject_lora(other, rank=4)
    assert qb.quantize_model(other) == ["0.base"]
    assert other(x.float()).shape == (5, 128)
    # a layer under two names stays one
    shared = qb.QuaternionLinear(32, 32).to(cuda)
    pair = torch.nn.ModuleDict({"a": shared, "b": shared})
    assert qb.quantize_model(pair) == ["a", "b"] and pair["a"] is pair["b"]


def test_a_training_step_on_the_frozen_base(qb, cuda):
    """Quantise, adapt, forward, backward, clip, step: the gradients are those
    of the layers' formulas, the clipped ones have the asked norm."""
    torch.manual_seed(1)
    net = torch.nn.Sequential(qb.QuaternionLinear(64, 96, bias=True), qb.QuaternionLinear(96, 64, bias=True)).to(cuda)
    qb.quantize_model(net)
    qb.inject_lora(net, rank=4)
    qb.mark_only_lora_trainable(net)
    params = [p for _, p in qb.lora_parameters(net)]
    with torch.no_grad():
        for p in params:
            p.normal_(std=0.2)
    x, target = torch.randn(20, 64, device=cuda), torch.randn(20, 64, device=cuda)
    loss = (net(x) - target).square().mean()
    loss.backward()
    # in 64 bits
    v = [values_of(m.base.weights) for m in net]
    A, B, bias = ([ref.f64(getattr(m, k)) for m in net] for k in ("lora_A", "lora_B", "bias"))
    s = net[0].scale
    h = ref.layer(ref.f64(x), v[0], bias[0], A[0], B[0], s)
    out = ref.layer(h, v[1], bias[1], A[1], B[1], s)
    gout = 2 * (out - ref.f64(target)) / out.size
    gh, dA1, dB1, _ = ref.gradients(gout, h, v[1], A[1], B[1], s)
    _, dA0, dB0, _ = ref.gradients(gh, ref.f64(x), v[0], A[0], B[0], s)
    wants = [dA0, dB0, dA1, dB1]
    for p, w in zip(params, wants):
        # a handful of fp32 results of up to 96 terms follow one another
        assert ref.rel(ref.f64(p.grad), w) <= 6 * ref.tolerance("f32", 200)
    norm = float(np.sqrt(sum((w * w).sum() for w in wants)))
    got = qb.clip_grad_norm(params, norm / 2)
    assert abs(float(got) - norm) <= 6 * ref.tolerance("f32", 200) * norm
    after = float(torch.stack([p.grad.double().square().sum() for p in params]).sum().sqrt())
    assert abs(after - norm / 2) <= 12 * ref.tolerance("f32", 200) * norm
    torch.optim.SGD(params, lr=0.1).step()
    assert all(m.base.weight_mx.grad is None for m in net)


# --------------------------------------------- order, devices, repeated calls
def test_inputs_written_right_before_a_call(qb, cuda):
    """Dependent launches see what was queued just before them: x, the codes, bias
    and the adapter, rows of any alignment among them."""
    for dtype, M, fin in (("bf16", 1, 512), ("bf16", 12, 516), ("bf16", 150, 516), ("f32", 20, 512), ("f16", 150, 512)):
        d = ref.draw(dtype, M, fin, 256, rank=5, bias=True, seed=1, device=cuda)
        e = ref.draw(dtype, M, fin, 256, rank=5, bias=True, seed=2, device=cuda)

        def call(v, q):
            return qb.mx_quaternion_linear(v["x"], q, v["bias"], v["a"], v["b"], 2.0)

        want = call(e, qb.quantize_quaternion_weights(*e["w"]))
        q = qb.quantize_quaternion_weights(*d["w"])
        for _ in range(5):
            call(d, q)
            new = qb.quantize_quaternion_weights(*e["w"])
            q.data.copy_(new.data)
            v = {k: t.clone() for k, t in d.items() if k in ("x", "bias", "a", "b")}
            for k in v:
                v[k].copy_(e[k])
            assert torch.equal(call(v, q), want)
            q = qb.quantize_quaternion_weights(*d["w"])


def test_two_streams_at_once(qb, cuda):
    d = ref.draw("bf16", 90, 512, 512, rank=8, seed=1, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs = [d["x"], d["x"] * 0.5]
    want = [qb.mx_quaternion_linear(x, q, None, d["a"], d["b"], 2.0) for x in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for s, x, out in zip(streams, xs, got):
            with torch.cuda.stream(s):
                out.append(qb.mx_quaternion_linear(x, q, None, d["a"], d["b"], 2.0))
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        assert all(torch.equal(o, w) for o in out)


def test_backward_in_a_graph_beside_an_eager_one(qb, cuda):
    """A captured forward and backward on leaves of its own; the eager pass of other
    leaves goes on as before."""
    d = ref.draw("bf16", 70, 256, 128, rank=8, bias=True, seed=1, device=cuda)
    q = qb.quantize_quaternion_weights(*d["w"])
    gy = torch.randn(70, 128, device=cuda).bfloat16()

    def step(leaves):
        y = qb.mx_quaternion_linear(leaves[0], q, leaves[1], leaves[2], leaves[3], 2.0)
        return torch.autograd.grad(y, leaves, gy)

    def leaves():
        return [d[k].clone().requires_grad_(True) for k in ("x", "bias", "a", "b")]

    want = step(leaves())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = leaves()
        step(mine)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(mine)
    for _ in range(3):
        graph.replay()
        eager = step(leaves())
        torch.cuda.synchronize()
        for a, b, w in zip(got, eager, want):
            assert torch.equal(a, w) and torch.equal(b, w)


def test_no_device_errors_left(qb, cuda):
    assert qb.device_error(cuda) == 0


@pytest.mark.parametrize("M,fin,rank", [(1, 4 * 3840, 88), (2, 4 * 3200, 88), (1, 4 * 3830, 88), (2, 4 * 3200, 256),
                                        (1, 4 * 3789, 8)])
def test_one_or_two_tokens_of_the_longest_rows(qb, cuda, M, fin, rank):
    """x, a ring, the rows of lora_b and t together at the most that shared memory holds."""
    check_forward(qb, ref.draw("bf16", M, fin, 260, rank=rank, bias=True, seed=rank, device=cuda), "bf16", 2)


def test_first_calls_inside_a_capture(qb, cuda):
    """Nothing that a first call sets up breaks a capture."""
    code = """
import importlib, sys, torch
sys.path.insert(0, {repo!r})
sys.path.insert(0, {repo!r} + "/tests")
import mx_reference as ref
qb = importlib.import_module("quaternion-based-math-1_b200")
for dtype, M in (("bf16", 1), ("f16", 12), ("bf16", 200), ("f32", 20)):
    d = ref.draw(dtype, M, 512, 256, rank=8, bias=True, seed=1, device="cuda")
    leaves = [d[k].requires_grad_(True) for k in ("x", "bias", "a", "b")]
    gy = torch.ones(M, 256, device="cuda", dtype=d["x"].dtype)
    def step():
        q = qb.quantize_quaternion_weights(*d["w"])
        y = qb.mx_quaternion_linear(leaves[0], q, leaves[1], leaves[2], leaves[3], 2.0)
        for p, g in zip(leaves, torch.autograd.grad(y, leaves, gy)):
            p.grad = g
        norm = qb.clip_grad_norm(leaves, 0.5)
        return [y, norm, *(p.grad for p in leaves), *q.dequantize(torch.float32)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)
    del graph
print("same")
"""
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code.format(repo=repo)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "same" in res.stdout, res.stderr[-2000:]


@pytest.mark.parametrize("dtype,M", [("bf16", 600), ("f16", 70), ("f32", 200)])
def test_gradients_of_buffers_that_change_between_calls(qb, cuda, dtype, M):
    """Every kernel of a backward pass is done with its inputs when the next work of
    the stream starts: the same buffers, refilled right behind each call."""
    sets = []
    for seed in (1, 2):
        d = ref.draw(dtype, M, 1024, 768, rank=8, bias=True, seed=seed, device=cuda)
        d["gy"] = ref.draw(dtype, M, 768, 4, seed=seed + 5, device=cuda)["x"]
        sets.append(d)
    q = qb.quantize_quaternion_weights(*sets[0]["w"])
    names = ("x", "bias", "a", "b", "gy")

    def step(v):
        leaves = [v[k].detach().requires_grad_(True) for k in names[:4]]
        y = qb.mx_quaternion_linear(leaves[0], q, leaves[1], leaves[2], leaves[3], 2.0)
        return torch.autograd.grad(y, leaves, v["gy"])

    want = []
    for d in sets:
        want.append(step(d))
        torch.cuda.synchronize()
    v = {k: sets[0][k].detach().clone() for k in names}
    got = []
    for n in range(12):
        got.append(step(v))
        for k in names:
            v[k].copy_(sets[(n + 1) % 2][k])
    for n, grads in enumerate(got):
        for a, b in zip(grads, want[n % 2]):
            assert torch.equal(a, b)
