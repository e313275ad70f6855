"""Cases for the operators of expert layers and of orthogonalised updates: what a training step, or a small serving step, asks of

* ``gn_kernels.grouped_scaled_mm`` with a weight stack: rows sorted by expert times that expert's matrix, ragged group sizes ("rows");
* ``gn_kernels.grouped_scaled_mm`` with two matrices: the contraction runs over each expert's rows, one weight gradient per expert ("depth");
* ``gn_kernels.quantize_int8_grouped``: column-wise absmax INT8 quantization within each expert's rows ("quant");
* ``torch.nn.functional.grouped_mm`` on a ``MixedPrecisionLinearWeight`` stack, forward and backward: the run of the three above ("linear");
* ``gn_kernels.orthogonalize``: Newton-Schulz orthogonalisation of a stack of weight updates ("ortho").

`run` computes them in elementary torch operations in 32 bits where `own` is False, and calls the package where it is True.
"""
import math
import os
import sys

import torch

own = False

STEPS = 5
COEFFS = (3.4445, -4.7750, 2.0315)      # the quintic a x + b x^3 + c x^5 of the usual Newton-Schulz iteration
NORM_EPS = 1e-7
QUANT_EPS = 1e-12

_OUT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quantized-training_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gn_kernels

    return gn_kernels


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # eight tokens of a batch that is being decoded, two experts each: the weights' bytes are what counts
        {"name": "rows decode int8", "kind": "rows", "T": 16, "E": 8, "K": 1024, "N": 4096, "dt": "int8", "out": "bf16", "layout": "nk", "pad": 0, "skew": 0.5},
        # a prompt of odd length through 16 experts in fp8, rows of padding behind the last expert
        {"name": "rows prompt e4m3", "kind": "rows", "T": 4099, "E": 16, "K": 1024, "N": 4096, "dt": "e4m3", "out": "bf16", "layout": "nk", "pad": 37, "skew": 0.5},
        # the up projection of a training step: 32768 routed rows, the 1b model's hidden and intermediate sizes
        {"name": "rows train int8", "kind": "rows", "T": 32768, "E": 8, "K": 2048, "N": 5632, "dt": "int8", "out": "bf16", "layout": "nk", "pad": 0, "skew": 0.5},
        # the gradient of the input of a training step: the same weights read the other way round, many experts
        {"name": "rows grad-input int8", "kind": "rows", "T": 16384, "E": 32, "K": 4096, "N": 1024, "dt": "int8", "out": "bf16", "layout": "kn", "pad": 0, "skew": 0.5},
        # weight gradients of a small model's step, odd number of rows
        {"name": "depth small int8", "kind": "depth", "T": 1021, "E": 8, "M": 512, "N": 256, "dt": "int8", "out": "bf16", "pad": 3, "skew": 0.5},
        # weight gradients of the training step above
        {"name": "depth train int8", "kind": "depth", "T": 32768, "E": 8, "M": 5632, "N": 2048, "dt": "int8", "out": "bf16", "pad": 0, "skew": 0.5},
        # the quantization in front of the weight gradients, small and large
        {"name": "quant small", "kind": "quant", "T": 1021, "E": 8, "C": 512, "dtype": "bf16", "pad": 3, "skew": 0.5},
        {"name": "quant train", "kind": "quant", "T": 32768, "E": 8, "C": 5632, "dtype": "bf16", "pad": 0, "skew": 0.5},
        # the whole expert projection: forward, gradient of the input and of the weights
        {"name": "linear small", "kind": "linear", "T": 509, "E": 8, "K": 256, "N": 512, "pad": 3, "skew": 0.5},
        {"name": "linear train", "kind": "linear", "T": 16384, "E": 8, "K": 2048, "N": 5632, "pad": 0, "skew": 0.5},
        # the update of one odd, tall matrix, and of eight experts' projections
        {"name": "ortho one tall", "kind": "ortho", "B": 1, "m": 999, "n": 333, "dtype": "bf16"},
        {"name": "ortho stack", "kind": "ortho", "B": 8, "m": 2048, "n": 5632, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _feature(rng, lo=64, hi=5632):
    """A feature size: a multiple of 64 mostly, of 16 or anything at times."""
    v = _log(rng, lo, hi)
    step = rng.choice((64, 64, 64, 16, 1))
    return max(lo, v // step * step)


def draw(rng):
    kind = rng.choice(("rows", "rows", "rows", "depth", "depth", "quant", "linear", "ortho", "ortho"))
    if kind == "ortho":
        m, n = _log(rng, 33, 4096), _log(rng, 33, 4096)
        lo, hi = min(m, n), max(m, n)
        b = max(1, min(_log(rng, 1, 16), int(2.2e11 / (lo * lo * hi))))
        return {"kind": kind, "B": b, "m": m, "n": n, "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    case = {"kind": kind, "T": _log(rng, 1, 32768), "E": _log(rng, 1, 64)}
    if kind == "quant":
        case |= {"C": _feature(rng), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}
    elif kind == "linear":
        case |= {"K": _feature(rng, 64, 2048), "N": _feature(rng)}
        case["T"] = min(case["T"], int(1.8e11 / (case["K"] * case["N"])))
    else:
        case |= {"K" if kind == "rows" else "M": _feature(rng), "N": _feature(rng, 64, 4096)}
        case["T"] = min(case["T"], int(3.5e11 / (case.get("K", case.get("M")) * case["N"])))
        case["dt"] = rng.choice(("int8", "int8", "int8", "e4m3", "e5m2"))
        case["out"] = rng.choice(("bf16", "bf16", "fp16", "fp32")) if case["dt"] == "int8" else "bf16"
        if kind == "rows":
            case["layout"] = rng.choice(("nk", "nk", "kn"))
            case["E"] = max(1, min(case["E"], int(6e8 / (case["K"] * case["N"]))))
        else:
            case["E"] = max(1, min(case["E"], int(3e8 / (case["M"] * case["N"]))))
    if kind == "linear":
        case["E"] = max(1, min(case["E"], int(3e8 / (case["K"] * case["N"]))))
    case["pad"] = rng.choice((0, 0, 0, rng.randint(1, 100)))
    case["skew"] = rng.choice((0.0, 0.5, 1.0))
    return case


def _sum_rows(case):
    """Rows that belong to an expert; `pad` more lie behind them."""
    return case["T"]


def _active(case):
    """Experts that a uniform router leaves with a row, on average."""
    return case["E"] * (1 - (1 - 1 / case["E"]) ** case["T"])


def work(case):
    k = case["kind"]
    if k == "ortho":
        b, lo, hi = case["B"], min(case["m"], case["n"]), max(case["m"], case["n"])
        # each step: X X^T and its square, both symmetric (half of the products), and the product with X
        return {"bytes": 2 * 2 * b * lo * hi, "flops": STEPS * b * (lo * lo * hi + lo ** 3 + 2.0 * lo * lo * hi)}
    T, E, rows = _sum_rows(case), case["E"], case["T"] + case["pad"]
    if k == "quant":
        sz = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": T * case["C"] * sz + rows * case["C"] + E * case["C"] * sz, "flops": 2.0 * T * case["C"]}
    if k == "linear":
        K, N = case["K"], case["N"]
        a = _active(case)
        return {"bytes": 2 * (T * (K + N) + a * K * N) + 2 * (rows * (N + K) + E * K * N), "flops": 6.0 * T * K * N}
    osz = 4 if case["out"] == "fp32" else 2
    if k == "rows":
        K, N = case["K"], case["N"]
        return {"bytes": T * K + _active(case) * K * N + rows * N * osz + (T + E * N) * osz, "flops": 2.0 * T * K * N}
    M, N = case["M"], case["N"]
    return {"bytes": T * (M + N) + E * M * N * osz + E * (M + N) * osz, "flops": 2.0 * T * M * N}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _groups(case, seed):
    """Ends of the groups on the GPU, as a router with a mild preference leaves them, and the largest group."""
    g = torch.Generator().manual_seed(1000003 * seed + 17)
    p = torch.softmax(case["skew"] * torch.randn(case["E"], generator=g), 0)
    sizes = torch.bincount(torch.multinomial(p, case["T"], replacement=True, generator=g), minlength=case["E"])
    return sizes.cumsum(0).to(torch.int32).cuda(), int(sizes.max())


def _quantized(x, dim, dt, out):
    """What a caller holds of an operand that is already quantized: 8-bit values and their scales in the output's type."""
    amax = x.abs().amax(dim, keepdim=True)
    if dt == "int8":
        return (x / (amax / 127).clamp_min(QUANT_EPS)).round().clamp(-128, 127).to(torch.int8), (amax / 127).to(_OUT[out])
    top = torch.finfo(_FP8[dt]).max
    return (x * (top / amax.clamp_min(QUANT_EPS))).clamp(-top, top).to(_FP8[dt]), (amax / top).to(_OUT[out])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 29)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    k = case["kind"]
    s = {"kind": k}
    if k == "ortho":
        b, m, n = case["B"], case["m"], case["n"]
        r = max(1, min(m, n) // 8)      # momentum of a weight: a few strong directions above noise
        s["G"] = (torch.bmm(randn(b, m, r), randn(b, r, n)) / math.sqrt(r) + 0.3 * randn(b, m, n)).mul_(1e-3).to(_OUT[case["dtype"]])
        return s
    s["offs"], s["tmax"] = _groups(case, seed)
    rows, E = case["T"] + case["pad"], case["E"]
    if k == "quant":
        s["x"] = randn(rows, case["C"]).to(_OUT[case["dtype"]])
    elif k == "linear":
        K, N = case["K"], case["N"]
        s["x"] = randn(rows, K).bfloat16()
        s["w"] = (randn(E, N, K) / math.sqrt(K)).bfloat16()
        s["gy"] = (randn(rows, N) * 1e-2).bfloat16()
    elif k == "rows":
        K, N = case["K"], case["N"]
        s["A"], s["sA"] = _quantized(randn(rows, K), 1, case["dt"], case["out"])
        if case["layout"] == "nk":      # weights as a Linear keeps them, (out, in) per expert
            B, sB = _quantized(randn(E, N, K), 2, case["dt"], case["out"])
            s["B"], s["sB"] = B.transpose(1, 2), sB.transpose(1, 2).contiguous()
        else:
            s["B"], s["sB"] = _quantized(randn(E, K, N), 1, case["dt"], case["out"])
    else:
        M, N = case["M"], case["N"]
        A, _ = _quantized(randn(rows, M), 0, case["dt"], case["out"])
        s["B"], _ = _quantized(randn(rows, N), 0, case["dt"], case["out"])
        s["A"] = A.t()                  # the rows lie in memory one after the other: (M, T) is a view
        s["sA"] = (torch.rand((E, M, 1), generator=g, device="cuda") * 0.02 + 0.01).to(_OUT[case["out"]])
        s["sB"] = (torch.rand((E, 1, N), generator=g, device="cuda") * 0.02 + 0.01).to(_OUT[case["out"]])
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _padded(x, offs, tmax, dtype=torch.float32):
    """(E, tmax, ...) copies of the groups' rows of x, zeros behind each group."""
    start = torch.cat([offs.new_zeros(1), offs[:-1]]).long()
    idx = start[:, None] + torch.arange(tmax, device=x.device)
    gone = idx >= offs[:, None]
    rows = x.to(dtype)[idx.clamp_(max=x.shape[0] - 1)]
    return rows.masked_fill_(gone[..., None], 0)


def _unpadded(y, offs, rows):
    """Back to rows in order; rows behind the last group are zeros."""
    t = torch.arange(rows, device=y.device)
    e = torch.searchsorted(offs.long(), t, right=True)
    gone = e >= offs.numel()
    e = e.clamp_(max=offs.numel() - 1)
    start = torch.cat([offs.new_zeros(1), offs[:-1]]).long()
    pos = (t - start[e]).clamp_(max=y.shape[1] - 1)
    return y[e, pos].masked_fill_(gone[:, None], 0)


def _plain_rows(A, B, sA, sB, offs, tmax, dtype=torch.float32):
    y = torch.bmm(_padded(A, offs, tmax, dtype), B.to(dtype).contiguous())
    y = y * _padded(sA, offs, tmax, dtype) * sB.to(dtype)
    return _unpadded(y, offs, A.shape[0])


def _plain_depth(A, B, sA, sB, offs, tmax, dtype=torch.float32):
    y = torch.bmm(_padded(A.t(), offs, tmax, dtype).transpose(1, 2).contiguous(), _padded(B, offs, tmax, dtype))
    return y * sA.to(dtype) * sB.to(dtype)


def _plain_quant(x, offs, tmax, dtype=torch.float32):
    """Column-wise absmax quantization within each group, in x's order; the scales in x's type."""
    xp = _padded(x, offs, tmax, dtype)
    scale = xp.abs().amax(1, keepdim=True) / 127
    q = (xp / scale.clamp_min(QUANT_EPS)).round_().clamp_(-128, 127)
    return _unpadded(q, offs, x.shape[0]), scale.to(x.dtype)


def _plain_quant_dim(x, dim, dtype=torch.float32):
    xf = x.to(dtype)
    scale = xf.abs().amax(dim, keepdim=True) / 127
    return (xf / scale.clamp_min(QUANT_EPS)).round_().clamp_(-128, 127), scale.to(x.dtype)


def _plain_linear(x, w, gy, offs, tmax, dtype=torch.float32):
    """INT8 mixed precision: every product's operands are quantized along the contraction."""
    xq, xs = _plain_quant_dim(x, 1, dtype)
    wq, ws = _plain_quant_dim(w, 2, dtype)
    y = _plain_rows(xq, wq.transpose(1, 2), xs, ws.transpose(1, 2), offs, tmax, dtype)
    gq, gs = _plain_quant_dim(gy, 1, dtype)
    wq, ws = _plain_quant_dim(w, 1, dtype)
    gx = _plain_rows(gq, wq, gs, ws, offs, tmax, dtype)
    xq, xs = _plain_quant(x, offs, tmax, dtype)
    gq, gs = _plain_quant(gy, offs, tmax, dtype)
    gw = _plain_depth(gq.t(), xq, gs.transpose(1, 2), xs, offs, tmax, dtype)
    return y, gx, gw


def _plain_ortho(G, dtype=torch.float32):
    a, b, c = COEFFS
    X = G.to(dtype)
    tall = X.shape[1] > X.shape[2]
    if tall:
        X = X.transpose(1, 2).contiguous()
    X = X / X.square().sum((1, 2), keepdim=True, dtype=torch.float64).sqrt().clamp_min(NORM_EPS).to(dtype)
    for _ in range(STEPS):
        A = torch.bmm(X, X.transpose(1, 2).contiguous())
        X = torch.baddbmm(X, torch.baddbmm(A, A, A, beta=b, alpha=c), X, beta=a)
    return X.transpose(1, 2).contiguous() if tall else X


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    s, k = state, state["kind"]
    if own:
        gn_kernels = _package()
        if k == "ortho":
            return gn_kernels.orthogonalize(s["G"], steps=STEPS, coefficients=COEFFS, eps=NORM_EPS)
        if k == "quant":
            return gn_kernels.quantize_int8_grouped(s["x"], s["offs"])
        if k == "linear":
            from subclasses import MixedPrecisionConfig, MixedPrecisionLinearWeight

            x = s["x"].detach().requires_grad_()
            w = torch.nn.Parameter(MixedPrecisionLinearWeight(s["w"], MixedPrecisionConfig()))
            y = torch.nn.functional.grouped_mm(x, w.transpose(-2, -1), offs=s["offs"])
            gx, gw = torch.autograd.grad(y, (x, w), s["gy"])
            return y.detach(), gx, gw
        return gn_kernels.grouped_scaled_mm(s["A"], s["B"], s["sA"], s["sB"], s["offs"])
    if k == "ortho":
        return _plain_ortho(s["G"]).to(s["G"].dtype)
    if k == "quant":
        q, scale = _plain_quant(s["x"], s["offs"], s["tmax"])
        return q.to(torch.int8), scale
    if k == "linear":
        return tuple(t.bfloat16() for t in _plain_linear(s["x"], s["w"], s["gy"], s["offs"], s["tmax"]))
    form = _plain_rows if k == "rows" else _plain_depth
    return form(s["A"], s["B"], s["sA"], s["sB"], s["offs"], s["tmax"]).to(s["sA"].dtype)


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _round8(x, dim):
    """Quantized values (still in 64 bits) and scales as they are stored."""
    step = x.double().abs().amax(dim, keepdim=True) / 127.0
    return torch.round(x.double() / torch.clamp(step, min=QUANT_EPS)).clamp(-128, 127), step.to(x.dtype).double()


def exact(case, seed):
    """The definitions group by group, in 64 bits."""
    s, k = prepare(case, seed), case["kind"]
    if k == "ortho":
        c1, c3, c5 = COEFFS
        done = []
        for G in s["G"].double():
            X = G / max(float(G.norm()), NORM_EPS)
            for _ in range(STEPS):      # the odd polynomial of X, through the smaller of its two Gram matrices
                if X.shape[0] <= X.shape[1]:
                    S = X @ X.mT
                    X = c1 * X + c3 * (S @ X) + c5 * (S @ (S @ X))
                else:
                    S = X.mT @ X
                    X = c1 * X + c3 * (X @ S) + c5 * ((X @ S) @ S)
            done.append(X)
        return torch.stack(done)
    ends = s["offs"].tolist()
    spans = list(zip([0] + ends[:-1], ends))
    if k == "quant":
        scale = torch.zeros((case["E"], 1, case["C"]), dtype=torch.float64, device="cuda")
        for e, (lo, hi) in enumerate(spans):
            if hi > lo:
                scale[e, 0] = s["x"][lo:hi].double().abs().amax(0) / 127.0
        return None, scale
    if k == "linear":
        x, w, gy = s["x"], s["w"], s["gy"]
        y = torch.zeros(gy.shape, dtype=torch.float64, device="cuda")
        gx = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        gw = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
        for e, (lo, hi) in enumerate(spans):
            if hi == lo:
                continue
            (a, sa), (b, sb) = _round8(x[lo:hi], 1), _round8(w[e], 1)
            y[lo:hi] = (a @ b.T) * sa * sb.T
            (a, sa), (b, sb) = _round8(gy[lo:hi], 1), _round8(w[e], 0)
            gx[lo:hi] = (a @ b) * sa * sb
            (a, sa), (b, sb) = _round8(gy[lo:hi], 0), _round8(x[lo:hi], 0)
            gw[e] = (a.T @ b) * sa.T * sb
        return y, gx, gw
    A, B, sA, sB = s["A"].float().double(), s["B"].float().double(), s["sA"].double(), s["sB"].double()
    if k == "rows":
        y = torch.zeros((A.shape[0], B.shape[2]), dtype=torch.float64, device="cuda")
        for e, (lo, hi) in enumerate(spans):
            y[lo:hi] = (A[lo:hi] @ B[e]) * sA[lo:hi] * sB[e]
        return y
    y = torch.zeros((len(spans), A.shape[0], B.shape[1]), dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(spans):
        y[e] = (A[:, lo:hi] @ B[lo:hi]) * sA[e] * sB[e]
    return y
