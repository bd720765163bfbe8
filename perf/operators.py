"""Operators around the logits that kernel_opt scores: what makes them and what draws from them.

Kinds of case, each one pass through a public entry point:

  "sample"    fused_sample: a token a row from logits and one uniform number a row, with
              temperature, top-k, top-p and min-p, and the token's log-probabilities under the
              whole and under the filtered distribution (a rollout's inner loop);
  "norm"      fused_add_rms_norm and its backward: the residual's addition and the
              root-mean-square norm in front of the LM head, in training;
  "norm8"     fused_add_rms_norm_fp8: the same norm in serving, its output in e4m3 with a
              float32 scale for each 128 columns;
  "quantize"  quantize_fp8: e4m3 values and scales of activations (128 columns of a row share
              a scale) or of a weight (128 x 128 elements do);
  "linear"    fp8_linear: the product of the two, an 8-bit LM head's logits.

Shapes are the benchmark's (heads of 32000, 128256, 151936, 152064 and 262144 rows, a hidden
size of 3584), powers of two near them, and, for drawn cases, any between.

What the operators compute:

  sample    y_v = (x_v - max x) / T, w_v = exp(y_v); the order is falling x, ties lowest index
            first; K the first top_k of it, P those of K whose preceding mass is below
            top_p * mass(K) (the first always), M those of P with w >= min_p (the first
            always); the token is the lowest index whose running sum of M's weights exceeds
            uniform * mass(M); logp = y - ln sum(w), sample_logp = y - ln mass(M).
  norm      h = round(x + residual), s = (mean(h^2) + eps)^-1/2, y = round(h s w).
  quantize  a = max |v| of a block, scale = a / 448 (1 for a block of zeros),
            q = e4m3(v * (448 / a)).
  linear    out[m, n] = round(sum_b xs[m, b] ws[n / 128, b] sum_{k in b} x[m, k] w[n, k]).
"""
from __future__ import annotations

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
VOCABS = (32000, 50257, 128256, 151936, 152064, 262144)
BLOCK = 128
E4M3_MAX = 448.0
EPS = 1e-6


def listed():
    return [
        # One sequence being decoded with Llama-2's vocabulary, nucleus sampling: latency.
        dict(name="sample_one", kind="sample", rows=1, vocab=32000, dtype="fp32", temperature=0.8,
             top_k=0, top_p=0.9, min_p=0.0, per_row=False),
        # A decode batch of Qwen2.5-7B's vocabulary with every filter on, each request its own
        # parameters.
        dict(name="sample_decode", kind="sample", rows=64, vocab=152064, dtype="bf16",
             temperature=0.7, top_k=50, top_p=0.95, min_p=0.02, per_row=True),
        # Unfiltered sampling, which keeps the trainer's importance ratios at 1, of a wide batch
        # of rollouts with Llama-3's vocabulary.
        dict(name="sample_wide", kind="sample", rows=1024, vocab=128256, dtype="fp16",
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, per_row=False),
        # Nucleus sampling at a high temperature over 262144 fp32 columns: thousands of tokens
        # stay in the nucleus.
        dict(name="sample_long", kind="sample", rows=200, vocab=262144, dtype="fp32",
             temperature=1.2, top_k=0, top_p=0.9, min_p=0.0, per_row=False),
        # The norm before the head of a training batch, bf16 with the residual stream.
        dict(name="norm_train", kind="norm", rows=8192, dim=4096, dtype="bf16", residual=True),
        # A small fp32 model with an odd width and no residual.
        dict(name="norm_odd", kind="norm", rows=1000, dim=1601, dtype="fp32", residual=False),
        # A decode batch's norm in front of an 8-bit head.
        dict(name="norm8_decode", kind="norm8", rows=64, dim=3584, dtype="bf16", residual=True),
        # A scoring batch's.
        dict(name="norm8_score", kind="norm8", rows=16384, dim=3584, dtype="bf16",
             residual=True),
        # Activations that no norm produces.
        dict(name="quantize_rows", kind="quantize", rows=4096, dim=3584, dtype="fp16",
             block_rows=1),
        # A head's weight, once after each optimizer step of a run that samples in 8 bits.
        dict(name="quantize_head", kind="quantize", rows=152064, dim=3584, dtype="bf16",
             block_rows=128),
        # The 8-bit head on a decode batch: the weight's bytes.
        dict(name="linear_decode", kind="linear", tokens=16, dim=3584, out=152064, dtype="bf16"),
        # The 8-bit head on a scoring batch: the matrix cores.
        dict(name="linear_score", kind="linear", tokens=4096, dim=3584, out=152064,
             dtype="bf16"),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("sample", "sample", "norm", "norm8", "quantize", "linear", "linear"))
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    if kind == "sample":
        vocab = rng.choice(VOCABS + (_log_between(rng, 1000, 262144),) * 3)
        rows = _log_between(rng, 1, min(1024, 200 * 262144 // vocab))
        return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype,
                    temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice((0, 0, _log_between(rng, 1, 1000))),
                    top_p=rng.choice((1.0, 0.8, 0.9, 0.95, 0.99)),
                    min_p=rng.choice((0.0, 0.0, 0.01, 0.1)), per_row=rng.random() < 0.5)
    if kind in ("norm", "norm8"):
        dim = rng.choice((3584, _log_between(rng, 256, 16384)))
        rows = _log_between(rng, 1, min(65536, 32 * 2**20 // dim))
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype, residual=rng.random() < 0.7)
    if kind == "quantize":
        dim = rng.choice((3584, _log_between(rng, 256, 16384)))
        rows = _log_between(rng, 1, min(152064, 2**28 // dim))
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype,
                    block_rows=rng.choice((1, 128)))
    dim = rng.choice((3584, 16 * _log_between(rng, 16, 512)))
    out = rng.choice((32000, 152064, _log_between(rng, 512, 152064)))
    tokens = _log_between(rng, 1, min(4096, 2**41 // (dim * out)))
    return dict(kind=kind, tokens=tokens, dim=dim, out=out, dtype=dtype)


# --------------------------------------------------------------------------- inputs


def _quantized(x, block_rows):
    """(e4m3 values, float32 scales) of x by the formula above, in slices of rows."""
    step = 8192  # a multiple of BLOCK
    parts = [_plain_quantize(x[i:i + step], block_rows) for i in range(0, x.shape[0], step)]
    return torch.cat([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn), \
        torch.cat([p[1] for p in parts])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    kind = case["kind"]
    s = dict(case=dict(case))
    if kind == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = normal(rows, vocab)
        # What a head gives: a bulk of unlikely tokens, and a few dozen that stand out by
        # amounts that differ from row to row.
        few = torch.randint(0, vocab, (rows, 64), generator=g, device=dev)
        x.mul_(1.5).scatter_add_(1, few, 2.0 + 6.0 * torch.rand(rows, 64, generator=g, device=dev)
                                 + 2.0 * normal(rows, 1))
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["uniform"] = torch.rand(rows, generator=g, device=dev)
        t, k, p, m = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
        if case["per_row"]:  # parameters around the case's, a request each
            def around(v):
                return v * (0.75 + 0.25 * torch.rand(rows, generator=g, device=dev))
            t = around(t)
            k = (around(float(k)).ceil().to(torch.int32)) if k else None
            p = around(p) if p < 1.0 else None
            m = around(m) if m > 0.0 else None
        else:
            k, p, m = k or None, p if p < 1.0 else None, m if m > 0.0 else None
        s["how"] = (t, k, p, m)
    elif kind in ("norm", "norm8"):
        rows, dim, dt = case["rows"], case["dim"], DTYPES[case["dtype"]]
        grads = kind == "norm"
        s["x"] = normal(rows, dim).to(dt).requires_grad_(grads)
        s["weight"] = (1.0 + 0.2 * normal(dim)).to(dt).requires_grad_(grads)
        s["residual"] = None
        if case["residual"]:
            s["residual"] = (3.0 * normal(rows, dim)).to(dt).requires_grad_(grads)
        if grads:
            s["g_y"] = normal(rows, dim).to(dt)
            s["g_h"] = normal(rows, dim).to(dt)
    elif kind == "quantize":
        spread = torch.exp(normal(case["rows"], 1))
        s["x"] = (normal(case["rows"], case["dim"]) * spread).to(DTYPES[case["dtype"]])
    else:
        m, k, n = case["tokens"], case["dim"], case["out"]
        s["xq"], s["xs"] = _quantized(normal(m, k) * torch.exp(normal(m, 1)), 1)
        s["wq"], s["ws"] = _quantized(normal(n, k).mul_(k ** -0.5), BLOCK)
    if own:
        pkg = os.path.join(ROOT, "fused-logprob-entropy-cuda-kernel-for-llm-post-training_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import kernel_opt
        s["api"] = kernel_opt
    return s


# ---------------------------------------------------------------------- plain forms


def _column(v, like):
    """A parameter as a float64 column, from its float32 value."""
    if not isinstance(v, torch.Tensor):
        v = torch.full((like.shape[0],), float(v), device=like.device)
    return v.to(torch.float32).to(torch.float64)[:, None]


def _plain_sample(logits, uniform, temperature, top_k, top_p, min_p):
    # 64 bits: a token is drawn at a border of running sums over the whole row.
    x = logits.double()
    y = (x - x.amax(1, keepdim=True)) / _column(temperature, x)
    w = y.exp()
    kept = w
    if top_k is not None or top_p is not None or min_p is not None:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        ws = w.gather(1, order)
        rank = torch.arange(x.shape[1], device=x.device)[None, :]
        if top_k is not None:
            ws = torch.where(rank < _column(top_k, x), ws, 0.0)
        if top_p is not None:
            before = ws.cumsum(1) - ws
            share = _column(top_p, x) * ws.sum(1, keepdim=True)
            ws = torch.where((before < share) | (rank == 0), ws, 0.0)
        if min_p is not None:
            ws = torch.where((ws >= _column(min_p, x)) | (rank == 0), ws, 0.0)
        kept = torch.zeros_like(w).scatter_(1, order, ws)
    run_sum = kept.cumsum(1)
    token = (run_sum <= uniform.double()[:, None] * run_sum[:, -1:]).sum(1, keepdim=True)
    y = y.gather(1, token)
    logp = y - w.sum(1, keepdim=True).log()
    sample_logp = y - run_sum[:, -1:].log()
    return token[:, 0], logp[:, 0].float(), sample_logp[:, 0].float()


def _plain_norm(x, weight, residual):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    s = torch.rsqrt(hf.square().mean(1, keepdim=True) + EPS)
    return h, hf, s, hf * s * weight.float()


def _plain_norm_grads(x, weight, residual, g_y, g_h):
    h, hf, s, y = _plain_norm(x, weight, residual)
    gy = g_y.float()
    gw = gy * weight.float()
    dot = (gw * hf).mean(1, keepdim=True)
    dx = (g_h.float() + s * (gw - hf * (s * s * dot))).to(x.dtype)
    dw = (gy * hf * s).sum(0).to(weight.dtype)
    return y.to(x.dtype), h, dx, None if residual is None else dx, dw


def _plain_quantize(x, block_rows):
    rows, dim = x.shape
    nr, nd = -(-rows // block_rows), -(-dim // BLOCK)
    v = torch.zeros(nr * block_rows, nd * BLOCK, device=x.device)
    v[:rows, :dim] = x
    v = v.view(nr, block_rows, nd, BLOCK)
    a = v.abs().amax((1, 3), keepdim=True)
    scale = torch.where(a == 0, 1.0, a / E4M3_MAX)
    q = (v * torch.where(a == 0, 1.0, E4M3_MAX / a)).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.view(nr * block_rows, nd * BLOCK)[:rows, :dim].contiguous()
    return q.to(torch.float8_e4m3fn), scale.view(nr, nd)


def _plain_linear(xq, xs, wq, ws, dtype):
    k = xq.shape[1]
    x = xq.float() * xs.repeat_interleave(BLOCK, 1)[:, :k]
    w = wq.float()
    w *= ws.repeat_interleave(BLOCK, 0)[:wq.shape[0]].repeat_interleave(BLOCK, 1)[:, :k]
    return (x @ w.t()).to(dtype)


def run(state):
    s = state
    kind = s["case"]["kind"]
    if kind == "sample":
        t, k, p, m = s["how"]
        if own:
            return s["api"].fused_sample(s["logits"], s["uniform"], t, top_k=k, top_p=p, min_p=m)
        return _plain_sample(s["logits"], s["uniform"], t, k, p, m)
    if kind == "norm":
        x, w, r, gy, gh = s["x"], s["weight"], s["residual"], s["g_y"], s["g_h"]
        if r is None:
            gh = None
        if own:
            if r is None:
                y = s["api"].fused_rms_norm(x, w, eps=EPS)
                return (y, *torch.autograd.grad(y, (x, w), gy))
            y, h = s["api"].fused_add_rms_norm(x, r, w, eps=EPS)
            return (y, h, *torch.autograd.grad((y, h), (x, r, w), (gy, gh)))
        with torch.no_grad():
            if r is None:
                y, _, dx, _, dw = _plain_norm_grads(x, w, r, gy, torch.zeros_like(gy))
                return y, dx, dw
            return _plain_norm_grads(x, w, r, gy, gh)
    if kind == "norm8":
        x, w, r = s["x"], s["weight"], s["residual"]
        if own:
            if r is None:
                return s["api"].fused_rms_norm_fp8(x, w, eps=EPS)
            return s["api"].fused_add_rms_norm_fp8(x, r, w, eps=EPS)
        h, _, _, y = _plain_norm(x, w, r)
        q, scale = _plain_quantize(y, 1)
        return (q, scale) if r is None else (q, scale, h)
    if kind == "quantize":
        if own:
            return s["api"].quantize_fp8(s["x"], block_rows=s["case"]["block_rows"])
        return _plain_quantize(s["x"].float(), s["case"]["block_rows"])
    dt = DTYPES[s["case"]["dtype"]]
    if own:
        return s["api"].fp8_linear(s["xq"], s["xs"], s["wq"], s["ws"], out_dtype=dt)
    return _plain_linear(s["xq"], s["xs"], s["wq"], s["ws"], dt)


# ---------------------------------------------------------------------------- work


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "sample":
        n = case["rows"] * case["vocab"]
        # Logits once; the number, the token, its two log-probabilities, a row's parameters.
        return dict(bytes=n * size + case["rows"] * (20 + 16 * case["per_row"]), flops=4 * n)
    if kind == "linear":
        m, k, n = case["tokens"], case["dim"], case["out"]
        nb, nn = -(-k // BLOCK), -(-n // BLOCK)
        return dict(bytes=m * k + n * k + 4 * (m * nb + nn * nb) + m * n * size,
                    flops=2 * m * n * k)
    n = case["rows"] * case["dim"]
    nb = -(-case["dim"] // BLOCK)
    if kind == "quantize":
        return dict(bytes=n * (size + 1) + 4 * nb * -(-case["rows"] // case["block_rows"]),
                    flops=3 * n)
    r = case["residual"]
    if kind == "norm8":
        return dict(bytes=n * (size * (3 if r else 1) + 1) + 4 * nb * case["rows"], flops=8 * n)
    # Forward: x (and the residual) in, y (and h) out; backward: h and the gradients in, one
    # gradient out, each once.
    return dict(bytes=n * size * (8 if r else 5) + 3 * case["dim"] * size, flops=16 * n)


# --------------------------------------------------------------------------- exact


def _exact_row(x, u, t, k, p, m):
    """Token, logp, sample_logp of one row of float64 logits, one token after the other in
    falling order."""
    by = torch.argsort(-x, stable=True)
    y = (x[by] - x[by[0]]) / t
    w = torch.exp(y)
    n = x.numel() if k is None else min(k, x.numel())
    if p is not None:
        total = w[:n].sum()
        reach = torch.cumsum(w[:n], 0)
        # Tokens before which less than p of the mass lies: those after the first that
        # completes it go.
        n = max(1, min(n, 1 + int((reach[:-1] < p * total).sum())))
    if m is not None:
        n = max(1, min(n, int((w >= m).sum())))
    mass = w[:n].sum()
    ids, back = torch.sort(by[:n])
    reach = torch.cumsum(w[:n][back], 0)
    at = int(torch.searchsorted(reach, (u * reach[-1]).reshape(1), right=True)[0])
    at = min(at, n - 1)
    chosen = y[back[at]]
    return ids[at], chosen - torch.log(w.sum()), chosen - torch.log(mass)


def _exact_codes(v, block_rows):
    """e4m3 values and scales of float64 v, and nothing of them shared with the plain form."""
    rows, dim = v.shape
    q = torch.empty(rows, dim, device=v.device, dtype=torch.float64)
    scales = torch.empty(-(-rows // block_rows), -(-dim // BLOCK), device=v.device,
                         dtype=torch.float64)
    for j in range(0, dim, BLOCK):
        part = v[:, j:j + BLOCK]
        top = part.abs().max(1).values
        if block_rows > 1:
            pad = torch.zeros(scales.shape[0] * block_rows, device=v.device, dtype=v.dtype)
            pad[:rows] = top
            top = pad.view(-1, block_rows).max(1).values
        s = top / 448.0
        s[s == 0] = 1.0
        scales[:, j // BLOCK] = s
        z = part / s.repeat_interleave(block_rows)[:rows, None]
        # Rounding to 3 bits after the leading one, ties to even, steps of 2^-9 below 2^-6.
        e = torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6)))
        step = torch.exp2(e - 3)
        q[:, j:j + BLOCK] = (torch.round(z / step) * step).clamp(-448, 448)
    return q, scales


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "sample":
            x, u = s["logits"], s["uniform"]

            def of(v, i):
                return v if v is None else float(v[i]) if isinstance(v, torch.Tensor) \
                    else float(torch.tensor(float(v)))

            got = []
            for i in range(x.shape[0]):
                t, k, p, m = (of(v, i) for v in s["how"])
                got.append(_exact_row(x[i].double(), u[i].double(), t,
                                      None if k is None else int(k), p, m))
            return tuple(torch.stack(c) for c in zip(*got))
        if kind == "linear":
            k, out = case["dim"], []
            xd = s["xq"].double()
            for j in range(0, k, BLOCK):
                xd[:, j:j + BLOCK] *= s["xs"][:, j // BLOCK, None].double()
            for i in range(0, case["out"], 64 * BLOCK):
                wd = s["wq"][i:i + 64 * BLOCK].double()
                by_row = torch.arange(i, i + wd.shape[0], device=wd.device) // BLOCK
                for j in range(0, k, BLOCK):
                    wd[:, j:j + BLOCK] *= s["ws"][by_row, j // BLOCK, None].double()
                out.append(xd @ wd.t())
            return torch.cat(out, 1)
        if kind == "quantize":
            step = 64 * BLOCK
            parts = [_exact_codes(s["x"][i:i + step].double(), case["block_rows"])
                     for i in range(0, case["rows"], step)]
            return torch.cat([a for a, _ in parts]), torch.cat([b for _, b in parts])
        x, r, w = s["x"].double(), s["residual"], s["weight"].double()
        h = x if r is None else (x + r.double()).to(r.dtype).double()  # h is what is stored
        norm = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        d = case["dim"]
        unit = h / torch.sqrt(norm * norm / d + EPS)
        if kind == "norm8":
            q, scale = _exact_codes(unit * w, 1)
            return (q, scale) if r is None else (q, scale, h)
        gy = s["g_y"].double()
        along = (gy * w * unit).sum(1, keepdim=True) / d
        dx = (gy * w - unit * along) / torch.sqrt(norm * norm / d + EPS)
        dw = (gy * unit).sum(0)
        if r is None:
            return unit * w, dx, dw
        dx = dx + s["g_h"].double()
        return unit * w, h, dx, dx, dw
