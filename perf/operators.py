"""Measured cases of the 4-bit (MXFP4) quaternion weights and the operators around them.

A quaternion layer's frozen base is held as OCP microscaling 4-bit floating
point: e2m1 elements, one power-of-two (E8M0) scale for each run of 32 input
quaternions of one component row.  The operators:

``quantize``  the four weight components -> 4-bit codes and scales -> the
              values they stand for;
``linear``    the quaternion layer on such weights, with bias and LoRA
              residual, from single tokens to prefill;
``train``     that layer's forward and its gradients (input, LoRA A and B,
              bias) over the frozen base;
``clip``      the global norm of many gradient tensors, and their clipping.

``run`` computes them in plain torch (``own`` false) or by the package's
calls (``own`` true) on what ``prepare`` gives.
"""

import importlib
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BLOCK = 32
# e2m1: sign, two exponent bits, one mantissa bit
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# rows: output component a; columns: input component q; the weight component is a ^ q
_SIGN = ((1, -1, -1, -1), (1, 1, -1, 1), (1, 1, 1, -1), (1, -1, 1, 1))


def _package():
    return importlib.import_module("quaternion-based-math-1_b200")


def _linear(name, dtype, tokens, fin, fout, bias, rank, op="linear"):
    return {"name": name, "op": op, "dtype": dtype, "tokens": tokens, "in": fin, "out": fout, "bias": bias,
            "rank": rank}


def listed():
    return [
        # the decode layer of the benchmark, one token: latency of a served step
        _linear("decode_1_4096", "bf16", 1, 4096, 4096, True, 32),
        # the largest layer of the benchmark, one token: bound by the weights' bytes
        _linear("decode_1_27648", "bf16", 1, 5120, 27648, False, 0),
        # a batch of decode requests in fp16
        _linear("decode_16_4096", "f16", 16, 4096, 4096, True, 32),
        # a short prompt through a layer whose sizes fit no tile
        _linear("ragged_333", "f16", 333, 1000, 1036, True, 12),
        # the prefill layer of the benchmark
        _linear("prefill_2048", "bf16", 2048, 4096, 11008, False, 0),
        # prefill of the largest layer with its adapter
        _linear("prefill_27648", "bf16", 2048, 5120, 27648, True, 32),
        # fine-tuning step of one adapted layer over the frozen base
        _linear("train_2048", "bf16", 2048, 4096, 4096, True, 32, op="train"),
        # the same in fp32, a GPT-2-small projection
        _linear("train_f32", "f32", 512, 768, 2304, True, 8, op="train"),
        # converting a layer's weights
        {"name": "quantize_11008", "op": "quantize", "dtype": "bf16", "in": 4096, "out": 11008},
        # rows that end inside a block
        {"name": "quantize_ragged", "op": "quantize", "dtype": "f32", "in": 1000, "out": 1036},
        # adapters of 24 layers, fp32 gradients
        {"name": "clip_adapters", "op": "clip", "dtype": "f32", "layers": 24, "in": 4096, "out": 4096, "rank": 32,
         "max_norm": 1.0},
        # all components of 12 layers, bf16 gradients
        {"name": "clip_components", "op": "clip", "dtype": "bf16", "layers": 12, "in": 4096, "out": 11008, "rank": 0,
         "max_norm": 1.0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear", "train", "train", "quantize", "clip"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    fin, fout = 4 * _log_int(rng, 16, 1280), 4 * _log_int(rng, 16, 2752)
    if op == "quantize":
        return {"op": op, "dtype": dtype, "in": fin, "out": fout}
    if op == "clip":
        rank = rng.choice((0, 8, 16, 32))
        layers = rng.randint(1, 15 if rank == 0 else 31)
        return {"op": op, "dtype": dtype, "layers": layers, "in": fin, "out": fout, "rank": rank,
                "max_norm": rng.choice((0.5, 1.0, 1e6))}
    tokens = _log_int(rng, 1, 512 if dtype == "f32" else 2048)
    rank = rng.choice((4, 8, 16, 32, 64)) if op == "train" else rng.choice((0, 0, 4, 8, 20, 32, 64))
    return {"op": op, "dtype": dtype, "tokens": tokens, "in": fin, "out": fout, "bias": rng.random() < 0.5,
            "rank": rank}


def _power(exponent):
    return torch.exp2(exponent.double()).float()


def _round_values(w):
    """e2m1 magnitudes' indices, scales' exponents of blocks [..., blocks, 32] (fp32)."""
    amax = w.abs().amax(-1, keepdim=True)
    exponent = (torch.frexp(amax)[1] - 3).clamp(-127, 127)
    exponent = torch.where(amax == 0, torch.full_like(exponent, -127), exponent)
    a = w.abs() / _power(exponent)
    # to nearest, ties to the even code
    index = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return index, exponent


def _quantize(weights):
    """[4, N_g, K_g] -> codes [4, N_g, blocks, 16] (two per byte, the even element low), exponents [4, N_g, blocks, 1]."""
    w = weights.float()
    w = torch.nn.functional.pad(w, (0, -w.shape[-1] % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    index, exponent = _round_values(w)
    code = index + 8 * (w < 0)
    return code[..., 0::2] | (code[..., 1::2] << 4), exponent


def _values(codes, exponent, in_groups):
    """The fp32 values [4, N_g, K_g] of packed codes and exponents."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=codes.device)
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (table[code.int()] * _power(exponent)).flatten(-2)[..., :in_groups]


def _real_matrix(w):
    """The real [out, in] matrix of the components [4, N_g, K_g]."""
    rows = [torch.stack([_SIGN[a][q] * w[a ^ q] for q in range(4)], -1) for a in range(4)]
    return torch.stack(rows, 1).flatten(2).flatten(0, 1)


def _randn(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda") * std


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    kg, ng = case["in"] // 4, case["out"] // 4
    if case["op"] == "clip":
        shapes = ([(ng, kg)] * 4 if case["rank"] == 0 else [(case["rank"], 4 * kg), (4 * ng, case["rank"])])
        params = []
        for shape in shapes * case["layers"]:
            p = torch.nn.Parameter(torch.empty(shape, dtype=dtype, device="cuda"))
            p.grad = _randn(gen, *shape, std=0.02).to(dtype)
            params.append(p)
        return {"op": "clip", "params": params, "max_norm": case["max_norm"]}
    w = _randn(gen, 4, ng, kg, std=1.0 / math.sqrt(case["in"])).to(dtype)
    if case["op"] == "quantize":
        return {"op": "quantize", "dtype": dtype, "weights": tuple(w.unbind(0))}
    state = {"op": case["op"], "dtype": dtype, "in_groups": kg, "bias": None, "a": None, "b": None, "scale": 0.0}
    # the frozen base: what a program that serves or trains on it keeps in hand
    state["codes"], state["exponent"] = _quantize(w)
    state["base"] = _package().quantize_quaternion_weights(*w.unbind(0)) if own else None
    state["x"] = _randn(gen, case["tokens"], case["in"]).to(dtype)
    if case["bias"]:
        state["bias"] = _randn(gen, case["out"], std=0.02).to(dtype)
    if case["rank"]:
        state["a"] = _randn(gen, case["rank"], case["in"], std=0.01).to(dtype)
        state["b"] = _randn(gen, case["out"], case["rank"], std=0.01).to(dtype)
        state["scale"] = 2.0
    if case["op"] == "train":
        state["gy"] = _randn(gen, case["tokens"], case["out"]).to(dtype)
        for k in ("x", "bias", "a", "b"):
            if state[k] is not None:
                state[k].requires_grad_(True)
    return state


def _wide(t):
    return None if t is None else t.detach().float()


def _plain_linear(s):
    x, a, b, bias = (_wide(s[k]) for k in ("x", "a", "b", "bias"))
    matrix = _real_matrix(_values(s["codes"], s["exponent"], s["in_groups"]))
    y = x @ matrix.t()
    if a is not None:
        y += s["scale"] * ((x @ a.t()) @ b.t())
    if bias is not None:
        y += bias
    if s["op"] == "linear":
        return {"y": y.to(s["dtype"])}
    gy = s["gy"].float()
    up = s["scale"] * (gy @ b)
    grads = {"dx": gy @ matrix + up @ a, "da": up.t() @ x, "db": gy.t() @ (s["scale"] * (x @ a.t()))}
    if bias is not None:
        grads["dbias"] = gy.sum(0)
    return {k: v.to(s["dtype"]) for k, v in {"y": y, **grads}.items()}


def run(state):
    s = state
    if s["op"] == "quantize":
        if own:
            return list(_package().quantize_quaternion_weights(*s["weights"]).dequantize(s["dtype"]))
        w = torch.stack(s["weights"])
        return list(_values(*_quantize(w), w.shape[-1]).to(s["dtype"]).unbind(0))
    if s["op"] == "clip":
        grads = [p.grad for p in s["params"]]
        if own:
            norm = _package().clip_grad_norm(s["params"], s["max_norm"])
        else:
            norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
            factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
            _ = [g.copy_(g.float() * factor) for g in grads]
        return {"norm": norm, "grads": grads}
    if not own:
        return _plain_linear(s)
    y = _package().mx_quaternion_linear(s["x"], s["base"], s["bias"], s["a"], s["b"], s["scale"])
    if s["op"] == "linear":
        return {"y": y}
    names = [k for k in ("x", "a", "b", "bias") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["gy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    k, n, r = case["in"], case["out"], case.get("rank", 0)
    weights = k * n // 4
    if case["op"] == "clip":
        count = case["layers"] * (weights if r == 0 else r * (k + n))
        return {"bytes": 2 * count * size, "flops": 3 * count}
    held = n * (k // 4 // 2 + -(-(k // 4) // _BLOCK))  # half a byte per code, one byte per scale
    if case["op"] == "quantize":
        return {"bytes": 2 * weights * size + held, "flops": 4 * weights}
    m = case["tokens"]
    adapter, bias = r * (k + n) * size, n * size if case["bias"] else 0
    if case["op"] == "linear":
        return {"bytes": held + adapter + bias + m * (k + n) * size, "flops": 2 * m * n * k + 2 * m * r * (k + n)}
    return {"bytes": held + 2 * (adapter + bias) + 2 * m * (k + n) * size,
            "flops": 4 * m * n * k + 6 * m * r * (k + n) + m * n}


def _nearest(w):
    """Blocks' values in 64 bits: the scale is 2^(floor(log2 amax) - 2); e2m1 has steps of 1/2 below 2, 1 below 4, 2 above."""
    groups = w.shape[-1]
    pad = w.new_zeros(*w.shape[:-1], -groups % _BLOCK)
    blocks = torch.cat((w, pad), -1).double().unflatten(-1, (-1, _BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(top)).clamp(-125, 129) - 2)
    a = blocks.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.sign(blocks) * (torch.round(a / step) * step).clamp(max=6.0) * unit).flatten(-2)[..., :groups]


def _hamilton(w, x):
    """y_a = sum over the products of Hamilton's table, component by component, for w [4][n, k] and x [m, k, 4]."""
    r, i, j, k = (x[..., c] for c in range(4))
    wr, wi, wj, wk = (c.t() for c in w)
    return torch.stack((r @ wr - i @ wi - j @ wj - k @ wk, r @ wi + i @ wr - j @ wk + k @ wj,
                        r @ wj + j @ wr + i @ wk - k @ wi, r @ wk + k @ wr - i @ wj + j @ wi), -1)


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if s["op"] == "quantize":
        return [_nearest(w) for w in s["weights"]]
    if s["op"] == "clip":
        grads = [p.grad.double() for p in s["params"]]
        norm = math.sqrt(sum(float((g * g).sum()) for g in grads))
        factor = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [g * factor for g in grads]}
    # the values the 4-bit codes stand for
    nibbles = torch.stack((s["codes"] % 16, s["codes"] // 16), -1).flatten(-2).long()
    low, high = nibbles % 2, (nibbles // 2) % 4
    magnitude = torch.where(high == 0, 0.5 * low, (1 + 0.5 * low) * torch.exp2(high.double() - 1))
    w = torch.where(nibbles >= 8, -magnitude, magnitude) * torch.exp2(s["exponent"].double())
    w = w.flatten(-2)[..., : s["in_groups"]]
    x = s["x"].detach().double()
    y = _hamilton(w, x.unflatten(-1, (-1, 4))).flatten(-2)
    a, b, bias = (None if s[k] is None else s[k].detach().double() for k in ("a", "b", "bias"))
    if bias is not None:
        y = y + bias
    if a is not None:
        y = y + s["scale"] * (x @ a.T) @ b.T
    if s["op"] == "linear":
        return {"y": y}
    g = s["gy"].double()
    # the adjoint of a quaternion product is the product with the conjugate
    flip = torch.tensor([1.0, -1.0, -1.0, -1.0], dtype=torch.float64, device=w.device).view(4, 1, 1)
    dx = _hamilton((w * flip).transpose(1, 2), g.unflatten(-1, (-1, 4))).flatten(-2)
    out = {"y": y, "dx": dx + s["scale"] * (g @ b) @ a, "da": s["scale"] * (g @ b).T @ x,
           "db": s["scale"] * g.T @ (x @ a.T)}
    if bias is not None:
        out["dbias"] = g.sum(0)
    return out
