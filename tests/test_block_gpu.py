"""fused_block_norm, its 8-bit checkpoints and fused_block_norm_fp8 on the GPU,
against the float64 oracle (oracle/block_oracle.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import block_oracle, fp8_oracle, norm_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
EPS = 1e-6
U = 2.0 ** -24  # half a step of float32, relative

# (sequences, rows of each, dim): around every shape of a group.
SIZES = [(1, 1, 1), (3, 1, 7), (1, 5, 128), (3, 3, 511), (7, 1, 513), (2, 33, 1024), (5, 1, 1601),
         (1, 4, 2048), (3, 1, 2049), (4, 75, 3584), (1, 2, 4097), (3, 1, 8192), (1, 2, 8200),
         (2, 1, 16384)]


def _ko():
    import kernel_opt
    return kernel_opt


def np64(t):
    return t.detach().cpu().double().numpy()


def _data(seqs, length, dim, dtype, seed, gate="none", post=True, weight_dtype=None,
          gate_dtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    shape = (seqs, length, dim)
    d = dict(x=(r(*shape) * torch.exp(r(seqs, length, 1))).to(dtype),
             residual=(2.0 * r(*shape)).to(dtype),
             weight=(1.0 + 0.3 * r(dim)).to(weight_dtype or dtype))
    p, c, s, t = (0.8 + 0.3 * r(dim)), r(dim), r(seqs, 1, dim), r(*shape)
    if post:
        d["post_weight"] = p.to(weight_dtype or dtype)
    if gate != "none":
        d["gate"] = dict(channel=c, sequence=s, token=t)[gate].to(gate_dtype or dtype)
    return d, r(*shape).to(dtype), r(*shape).to(dtype)


def _steps(dim):
    """Roundings behind a row's sum, in units of U: a thread adds at most 64
    products one after the other, a group merges 10 levels of partial sums."""
    return min(dim, 64) + 10


def _half(dtype):
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


def _within(got, want, err, dtype, what):
    half, tiny = _half(dtype)
    bound = err + half * (np.abs(want) + err) + tiny
    off = np.abs(np64(got).reshape(want.shape) - want) - bound
    assert (off <= 0).all(), (what, float(off.max()))


def _rows_of(d, dim):
    """Operands as float64 rows, the gate broadcast to them."""
    x = np64(d["x"]).reshape(-1, dim)
    gate = np64(d["gate"].expand_as(d["x"])).reshape(-1, dim) if "gate" in d else np.ones_like(x)
    return (x, np64(d["residual"]).reshape(-1, dim), np64(d["weight"]),
            np64(d["post_weight"]) if "post_weight" in d else None, gate)


def _check_h(h, d, scale, dim, dtype):
    """The statistic's error, its four roundings, three products and the sum."""
    x, r, _, post, gate = _rows_of(d, dim)
    want, u = block_oracle.forward(x, r, post, gate, scale, EPS)
    err = np.abs(u) * (_steps(dim) / 2 + 4 + 4) * U + np.abs(want) * U
    _within(h, want, err, dtype, "h")


def _check_y(y, h, weight, dtype):
    rows = np64(h).reshape(-1, h.shape[-1])
    ref, _ = norm_oracle.forward(rows, np64(weight), EPS)
    _within(y, ref, np.abs(ref) * (_steps(h.shape[-1]) / 2 + 6) * U, dtype, "y")


def _kept(t):
    """The values of t's 8-bit checkpoint."""
    q, s = _ko().quantize_fp8(t.detach().to(DEV))
    codes = fp8_oracle.decode(q.view(torch.uint8).cpu().numpy()).reshape(-1, t.shape[-1])
    return codes * fp8_oracle.spread(np64(s).reshape(codes.shape[0], -1), 1, *codes.shape)


def _check_grads(grads, d, h, scale, gy, gh, dtype, kept):
    dim = h.shape[-1]
    x, _, weight, post, gate = _rows_of(d, dim)
    hr = np64(h).reshape(-1, dim)
    s_x, s_h = block_oracle.rstd(x, EPS), block_oracle.rstd(hr, EPS)
    if kept:
        x, hr = _kept(d["x"]), _kept(h)
    unit = (_steps(dim) / 2 + 4) * U, (_steps(dim) + 8) * U, U
    want = block_oracle.backward(x, hr, s_x, s_h, weight, post, gate, scale,
                                 np64(gy).reshape(-1, dim) if gy is not None else 0.0 * x,
                                 np64(gh).reshape(-1, dim) if gh is not None else 0.0 * x, unit)
    _within(grads["x"], *want["x"], dtype, "d_x")
    _within(grads["residual"], *want["residual"], dtype, "d_residual")
    _within(grads["weight"], *want["weight"], d["weight"].dtype, "d_weight")
    if post is not None:
        _within(grads["post_weight"], *want["post"], d["weight"].dtype, "d_post_weight")
    if "gate" in d:
        shape, full = d["gate"].shape, d["x"].shape
        value, err = (torch.from_numpy(v).reshape(full).sum_to_size(shape).numpy()
                      for v in want["gate"])
        _within(grads["gate"], value, err, d["gate"].dtype, "d_gate")


def _run(d, gy, gh, scale, checkpoint=None, f=None):
    t = {k: v.to(DEV).requires_grad_() for k, v in d.items()}
    f = f or _ko().fused_block_norm
    y, h = f(t["x"], t["residual"], t["weight"], post_weight=t.get("post_weight"),
             gate=t.get("gate"), scale=scale, eps=EPS, checkpoint=checkpoint)
    outs = [o for o, g in ((y, gy), (h, gh)) if g is not None]
    gs = [g.to(DEV) for g in (gy, gh) if g is not None]
    got = torch.autograd.grad(outs, list(t.values()), gs)
    return y, h, dict(zip(t, got))


@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("post", [True, False], ids=["post", "bare"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_forward_and_backward(dtype, post, gate):
    for seqs, length, dim in SIZES:
        d, gy, gh = _data(seqs, length, dim, dtype, dim + seqs, gate, post)
        for kept in (None, "fp8"):
            print(f"block {seqs} x {length} x {dim} {dtype} {post} {gate} {kept}", flush=True)
            y, h, grads = _run(d, gy, gh, 0.7, kept)
            assert y.shape == h.shape == d["x"].shape and y.dtype == h.dtype == dtype
            _check_h(h, d, 0.7, dim, dtype)
            _check_y(y, h, d["weight"], dtype)
            for k, g in grads.items():
                assert g.shape == d[k].shape and g.dtype == d[k].dtype
            _check_grads(grads, d, h, 0.7, gy, gh, dtype, kept)


@pytest.mark.parametrize("seqs,length", [(7, 857), (1000, 6), (2, 4097), (4100, 1), (1, 9000),
                                         (333, 27)])
def test_gates_of_many_rows(seqs, length):
    """Gates that end inside a group's rows, go on past several groups, or have
    a row each."""
    for dim, dtype in ((40, torch.float32), (520, torch.bfloat16)):
        for post in (True, False):
            d, gy, gh = _data(seqs, length, dim, dtype, seqs, "sequence", post)
            y, h, grads = _run(d, gy, gh, 1.3)
            _check_grads(grads, d, h, 1.3, gy, gh, dtype, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_float32_weights_and_gates(dtype):
    for wd, gd in ((torch.float32, None), (None, torch.float32), (torch.float32, torch.float32)):
        d, gy, gh = _data(3, 40, 3000, dtype, 5, "sequence", True, wd, gd)
        for kept in (None, "fp8"):
            y, h, grads = _run(d, gy, gh, 1.0, kept)
            _check_h(h, d, 1.0, 3000, dtype)
            _check_y(y, h, d["weight"], dtype)
            _check_grads(grads, d, h, 1.0, gy, gh, dtype, kept)


def test_plain_form_is_the_add_norm():
    """Without norm, gate and scale: fused_add_rms_norm's h exactly, y and
    gradients up to the order of sums."""
    ko = _ko()
    for dtype in DTYPES:
        d, gy, gh = _data(4, 9, 1500, dtype, 3, "none", False)
        y, h, grads = _run(d, gy, gh, 1.0)
        t = {k: v.to(DEV).requires_grad_() for k, v in d.items()}
        y2, h2 = ko.fused_add_rms_norm(t["x"], t["residual"], t["weight"], EPS)
        assert torch.equal(h, h2) and torch.equal(grads["x"], grads["residual"])
        # Each is within (steps / 2 + 6) U, by the order of its sum (as _check_y
        # counts them), and half a step of the exact one: twice that apart.
        half, tiny = _half(dtype)
        rel = 2 * (half + (_steps(1500) / 2 + 6) * U) * 1.01
        assert ((y - y2).abs().double() <= y2.abs().double() * rel + 2 * tiny).all()


def test_one_gradient_alone():
    """g_y or g_h alone, and only the gradients asked for."""
    ko = _ko()
    for gate, post in (("channel", True), ("sequence", False), ("none", True)):
        d, gy, gh = _data(3, 11, 300, torch.float32, 8, gate, post)
        for a, b in ((gy, None), (None, gh)):
            y, h, grads = _run(d, a, b, 0.5)
            _check_grads(grads, d, h, 0.5, a, b, torch.float32, False)
        _, _, full = _run(d, gy, gh, 0.5)
        for need in d:
            t = {k: v.to(DEV).requires_grad_(k == need) for k, v in d.items()}
            y, h = ko.fused_block_norm(t["x"], t["residual"], t["weight"],
                                       post_weight=t.get("post_weight"), gate=t.get("gate"),
                                       scale=0.5, eps=EPS)
            outs, gs = [y], [gy.to(DEV)]
            if h.requires_grad:
                outs, gs = [y, h], [gy.to(DEV), gh.to(DEV)]
            got, = torch.autograd.grad(outs, t[need], gs)
            assert torch.equal(got, full[need]), need


def test_gradient_against_differences():
    """Along random directions of every operand, differences of the formula in
    64 bits (float32 rows: h's rounding is 2^-24 of it)."""
    seqs, length, dim = 2, 3, 50
    d, gy, gh = _data(seqs, length, dim, torch.float32, 4, "sequence", True)
    _, _, grads = _run(d, gy, gh, 0.6)
    base = {k: np64(v) for k, v in d.items()}

    def loss(v):
        x = v["x"].reshape(-1, dim)
        gate = np.broadcast_to(v["gate"], v["x"].shape).reshape(-1, dim)
        h, _ = block_oracle.forward(x, v["residual"].reshape(-1, dim), v["post_weight"], gate, 0.6,
                                    EPS)
        y, _ = norm_oracle.forward(h, v["weight"], EPS)
        return (y * np64(gy).reshape(-1, dim)).sum() + (h * np64(gh).reshape(-1, dim)).sum()

    rng = np.random.RandomState(0)
    for _ in range(5):
        v = {k: rng.randn(*a.shape) for k, a in base.items()}
        e = 1e-5
        num = (loss({k: base[k] + e * v[k] for k in base})
               - loss({k: base[k] - e * v[k] for k in base})) / (2 * e)
        ana = sum((np64(grads[k]) * v[k]).sum() for k in base)
        size = sum(np.abs(np64(grads[k]) * v[k]).sum() for k in base)
        # float32 gradients of some hundred roundings of terms that cancel, and e^2.
        assert abs(num - ana) <= size * (2000 * U + 1e-8)


def test_layouts():
    ko = _ko()
    g = torch.Generator().manual_seed(2)
    for dtype in DTYPES:
        base = torch.randn(3, 7, 403, generator=g).to(dtype).to(DEV)
        w = torch.randn(806, generator=g).to(dtype).to(DEV)
        for x in (base, base[:, 1:, 3:200], base[..., ::2], base.transpose(0, 1), base[0, 0]):
            D = x.size(-1)
            res = torch.randn(x.shape, generator=g).to(dtype).to(DEV)
            gates = [None, w[::2][:D], torch.randn(x.shape, generator=g).to(dtype).to(DEV)]
            if x.dim() == 3:
                gates.append(torch.randn(x.size(0), 1, D, generator=g).to(dtype).to(DEV))
                gates.append(gates[-1].expand(x.shape))
            for gate in gates:
                kw = dict(post_weight=w[1:D + 1], gate=gate, scale=0.5)
                a = ko.fused_block_norm(x, res, w[:D], **kw)
                dense = None if gate is None else gate.contiguous()
                b = ko.fused_block_norm(x.contiguous(), res, w[:D].contiguous(),
                                        post_weight=w[1:D + 1].clone(), gate=dense, scale=0.5)
                assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[0].shape == x.shape
                q, s, h = ko.fused_block_norm_fp8(x, res, w[:D], **kw)
                assert torch.equal(h, a[1]) and s.shape == (*x.shape[:-1], -(-D // 128))
                leaf = x.detach().requires_grad_()
                for kept in (None, "fp8"):
                    y, _ = ko.fused_block_norm(leaf, res, w[:D], checkpoint=kept, **kw)
                    d, = torch.autograd.grad(y.float().sum(), leaf)
                    assert d.shape == x.shape
        e = torch.empty(0, 4, 16, dtype=dtype, device=DEV, requires_grad=True)
        ew = w[:16].detach().requires_grad_()
        eg = torch.empty(0, 1, 16, dtype=dtype, device=DEV, requires_grad=True)
        y, h = ko.fused_block_norm(e, e.detach(), ew, post_weight=ew, gate=eg)
        dx, dw, dg = torch.autograd.grad(y, (e, ew, eg), torch.empty_like(y))
        assert dx.shape == e.shape and not dw.any() and dg.shape == eg.shape


def test_special_rows():
    x = torch.randn(8, 300, generator=torch.Generator().manual_seed(4))
    r = torch.zeros(8, 300)
    x[1] = 0.0
    x[2] *= 1e-30
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    x[5] *= 1e15
    w = torch.ones(300)
    y, h = _ko().fused_block_norm(x.to(DEV), r.to(DEV), w.to(DEV), post_weight=w.to(DEV), eps=EPS)
    ok = [0, 1, 2, 5, 6, 7]
    _check_h(h[ok], dict(x=x[ok], residual=r[ok], weight=w, post_weight=w), 1.0, 300, torch.float32)
    _check_y(y[ok], h[ok].cpu(), w, torch.float32)
    assert y[3].isnan().all() and y[4].isnan().any() and not y[ok].isnan().any()


@pytest.mark.parametrize("post", [True, False], ids=["post", "bare"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_fp8(dtype, post):
    """h bit for bit as the other form's; scales and codes of its y."""
    ko = _ko()
    for seqs, length, dim in [(1, 1, 1), (5, 1, 127), (3, 3, 1000), (64, 1, 3584), (3, 1, 5003),
                              (1, 2, 16000)]:
        d, _, _ = _data(seqs, length, dim, dtype, dim, "sequence", post)
        t = {k: v.to(DEV) for k, v in d.items()}
        kw = dict(post_weight=t.get("post_weight"), gate=t["gate"], scale=0.3, eps=EPS)
        q, s, h = ko.fused_block_norm_fp8(t["x"], t["residual"], t["weight"], **kw)
        assert torch.equal(h, ko.fused_block_norm(t["x"], t["residual"], t["weight"], **kw)[1])
        rows = seqs * length
        y, _ = norm_oracle.forward(np64(h).reshape(rows, dim), np64(d["weight"]), EPS)
        amax = fp8_oracle.block_amax(y, 1)
        rel = (_steps(dim) / 2 + 4 + 2 + 2) * U
        ref = np.where(amax == 0, 1.0, amax / 448.0)
        assert (np.abs(np64(s).reshape(rows, -1) - ref) <= ref * rel).all()
        codes = fp8_oracle.decode(q.view(torch.uint8).cpu().numpy()).reshape(rows, dim)
        exact = y / fp8_oracle.spread(ref, 1, rows, dim)
        bound = np.maximum(np.abs(exact) * 2.0 ** -4, 2.0 ** -10) + np.abs(exact) * 2 * rel
        assert (np.abs(codes - exact) <= bound).all()


def test_statement_streams_and_graphs():
    """The same bits from the compiled function, its Python statement, repeated
    calls, another stream, and replays of a graph that holds both passes."""
    from kernel_opt.block import _FusedBlockNorm
    ko = _ko()
    for gate in ("channel", "sequence"):
        d, gy, gh = _data(4, 150, 1024, torch.bfloat16, 6, gate, True)
        gy, gh = gy.to(DEV), gh.to(DEV)
        t = {k: v.to(DEV).requires_grad_() for k, v in d.items()}
        per = 600 if gate == "channel" else 150

        def step(statement=False):
            got = []
            for kept in (None, "fp8"):
                if statement:
                    y, h = _FusedBlockNorm.apply(t["x"], t["residual"], t["weight"],
                                                 t["post_weight"], t["gate"], per, 0.5, EPS,
                                                 kept is not None)
                else:
                    y, h = ko.fused_block_norm(t["x"], t["residual"], t["weight"],
                                               post_weight=t["post_weight"], gate=t["gate"],
                                               scale=0.5, eps=EPS, checkpoint=kept)
                got += [y, h, *torch.autograd.grad((y, h), list(t.values()), (gy, gh))]
            q, s, _ = ko.fused_block_norm_fp8(t["x"], t["residual"], t["weight"], gate=t["gate"])
            return [o.detach().clone() for o in (*got, q.view(torch.uint8), s)]

        def same(a, b):
            return all(torch.equal(p, q) for p, q in zip(a, b))

        want = step()
        assert same(want, step()) and same(want, step(True))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step()
        torch.cuda.current_stream().wait_stream(s)
        assert same(want, got)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = step()
        for _ in range(3):
            with torch.no_grad():
                t["x"].copy_(torch.randn_like(t["x"], dtype=torch.float32))
                gy.mul_(0.5)
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, step())


def test_what_a_checkpoint_keeps():
    """Bytes held between the passes: 2 of 16 bits an element, or 2 codes and
    two scales for each 128."""
    ko = _ko()
    rows, dim = 2048, 2048
    w = torch.ones(dim, dtype=torch.bfloat16, device=DEV)
    held = {}
    for kept in (None, "fp8"):
        leaf = torch.randn(rows, dim, device=DEV).bfloat16().requires_grad_()
        r = torch.randn(rows, dim, device=DEV).bfloat16()
        before = torch.cuda.memory_allocated()
        x = leaf * 1.0  # a block's output, which nothing else keeps
        y, h = ko.fused_block_norm(x, r, w, post_weight=w, checkpoint=kept)
        loss = y.sum()
        del x, y, h
        torch.cuda.synchronize()
        held[kept] = torch.cuda.memory_allocated() - before
        loss.backward()
        assert leaf.grad is not None
        del loss, leaf  # its graph holds the leaf
    n = rows * dim
    assert 4 * n <= held[None] <= 4 * n + 2 ** 20
    assert 2 * n <= held["fp8"] <= 2 * n + 2 * n // 32 + 2 ** 20


def test_second_derivatives_are_refused():
    from kernel_opt.block import _FusedBlockNorm
    ko = _ko()
    d, _, _ = _data(2, 3, 40, torch.float32, 1, "channel", True)
    for f in (lambda x, r, w, p, g, k: ko.fused_block_norm(x, r, w, post_weight=p, gate=g,
                                                           checkpoint="fp8" if k else None),
              lambda x, r, w, p, g, k: _FusedBlockNorm.apply(x, r, w, p, g, 6, 1.0, EPS, k)):
        for which in d:
            t = {k: v.to(DEV).requires_grad_() for k, v in d.items()}
            y, h = f(t["x"].tanh(), t["residual"], t["weight"], t["post_weight"], t["gate"], False)
            total = y.square().sum() + h.square().sum() + t[which].pow(3).sum()
            got, = torch.autograd.grad(total, t[which], create_graph=True)
            with pytest.raises(RuntimeError, match="no second derivative"):
                torch.autograd.grad(got.square().sum(), t[which])
        t = {k: v.to(DEV).requires_grad_() for k, v in d.items()}
        y, _ = f(t["x"], t["residual"], t["weight"], t["post_weight"], t["gate"], True)
        with pytest.raises(RuntimeError, match="8-bit checkpoints"):
            torch.autograd.grad(y.sum(), t["x"], create_graph=True)


def test_refusals():
    ko = _ko()
    x = torch.zeros(4, 6, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(64, dtype=torch.bfloat16, device=DEV)
    for f in (ko.fused_block_norm, ko.fused_block_norm_fp8):
        for bad in (x[:3], x.half(), x.cpu(), x[..., :63]):
            with pytest.raises(RuntimeError, match="residual must have"):
                f(x, bad, w)
        for bad in (w[:63], w.cpu(), w[None]):
            with pytest.raises(RuntimeError, match="weight must be"):
                f(x, x, bad)
            with pytest.raises(RuntimeError, match="post_weight must be"):
                f(x, x, w, post_weight=bad)
        with pytest.raises(RuntimeError, match="both be float32"):
            f(x, x, w, post_weight=w.float())
        with pytest.raises(RuntimeError, match="both be float32"):
            f(x, x, w.half())
        for bad in (x[:, :, :63], x[:1], w[None], x[0], x[:, :3], w[:32]):
            with pytest.raises(RuntimeError, match="gate must be"):
                f(x, x, w, gate=bad)
        with pytest.raises(RuntimeError, match="gate must be float32"):
            f(x, x, w, gate=w.half())
        for bad in (float("nan"), float("inf")):
            with pytest.raises(RuntimeError, match="scale"):
                f(x, x, w, scale=bad)
        with pytest.raises(RuntimeError, match="eps"):
            f(x, x, w, eps=-1.0)
        wide = torch.zeros(1, 16385, device=DEV)
        with pytest.raises(RuntimeError, match="last dim"):
            f(wide, wide, wide[0])
        with pytest.raises(RuntimeError, match="GPU tensor"):
            f(x.cpu(), x.cpu(), w.cpu())
    with pytest.raises(ValueError, match="checkpoint"):
        ko.fused_block_norm(x, x, w, checkpoint="int8")


def test_rows_beyond_32_bits():
    ko = _ko()
    g = torch.Generator(device=DEV).manual_seed(1)
    rows, dim = 2 ** 18 + 3, 8200
    x = torch.zeros(rows, dim, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, dim, generator=g, device=DEV)
    w = torch.randn(dim, generator=g, device=DEV)
    y, h = ko.fused_block_norm(x, x, w, post_weight=w, scale=0.5)
    y1, h1 = ko.fused_block_norm(x[-3:], x[-3:], w, post_weight=w, scale=0.5)
    assert torch.equal(y[-3:], y1) and torch.equal(h[-3:], h1)
