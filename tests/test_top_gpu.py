"""fused_top_logprobs on the GPU, against the float64 oracle
(oracle/top_oracle.py)."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

from oracle import top_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
U = 2.0 ** -24  # half a step of float32, relative


def _ko():
    import kernel_opt
    return kernel_opt


def np64(t):
    return t.detach().cpu().double().numpy()


def _logits(rows, vocab, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    t = torch.randint(0, vocab, (rows,), generator=g)
    x[torch.arange(rows), t] += 4.0 * torch.rand(rows, generator=g)
    return x.to(dtype), t


def _sum_error(x, t):
    """Relative error of a row's float32 sums.  A thread of at least 256 adds
    its share of the weights one after the other, rescales them a few times and
    merges 9 levels; each weight carries the exponential's rounding and those of
    its exponent, which move it by 3 U of |y - max y|, here in the mean."""
    n = -(-x.size // 256) + 16
    y = (x[np.isfinite(x)] - x[np.isfinite(x)].max()) / t
    w = np.exp(y)
    away = float((w * np.abs(y)).sum() / w.sum())
    return (n + 40 + 4 * away) * U, away


def _check_row(got, x, target, k, T):
    lp, ent, lse, rank, ids, top = got
    want = top_oracle.forward_row(x, target, k, T)
    assert rank == want[3]
    assert (ids == want[4]).all(), (ids, want[4])
    t = float(np.float32(T))
    err, away = _sum_error(x, t)
    ln_z = want[2] - x[np.isfinite(x)].max() / t
    off = err + 4 * U * abs(ln_z)
    # x - max and its product with 1 / T: three roundings of the difference.
    assert abs(lse - want[2]) <= off + 3 * U * (abs(want[2]) + abs(want[2] - ln_z))
    assert abs(ent - want[1]) <= 2 * (err + 4 * U) * (1 + away + abs(ln_z))
    if np.isfinite(want[0]):
        big = abs(want[0]) + abs(ln_z) + (abs(want[2]) if not 0 <= target < x.size else 0.0)
        assert abs(lp - want[0]) <= off + 4 * U * big
    else:
        assert lp == want[0]
    fin = np.isfinite(want[5])
    assert (np.abs(top[fin] - want[5][fin])
            <= off + 4 * U * (np.abs(want[5][fin]) + abs(ln_z))).all()
    assert (top[~fin] == want[5][~fin]).all()


def _check(out, x, t, k, T=1.0):
    out = [o.detach().cpu().numpy() for o in out]
    xs = np64(x)
    for i in range(len(xs)):
        _check_row([o[i] for o in out], xs[i], int(t[i]), k, T)


# One column to rows in pieces; 4 and 8 waves; whole vectors and odd ends.
SHAPES = [(1, 1, 1), (2, 2, 3), (3, 7, 7), (5, 8, 2), (4, 100, 256), (6, 513, 20), (3, 1000, 128),
          (2, 4099, 5), (300, 1023, 9), (1, 32000, 5), (2, 50257, 64), (1, 152064, 256),
          (130, 33003, 20), (5, 70001, 33)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab,k", SHAPES)
def test_forward(rows, vocab, k, dtype):
    for T in (None, 0.7):
        print(f"top {rows} x {vocab} k={k} {dtype} T={T}", flush=True)
        x, t = _logits(rows, vocab, dtype, rows + vocab)
        out = _ko().fused_top_logprobs(x.to(DEV), t.to(DEV), k, T)
        assert [o.dtype for o in out] == [torch.float32] * 3 + [torch.int64] * 2 + [torch.float32]
        assert [o.shape for o in out] == [(rows,)] * 4 + [(rows, k)] * 2
        _check(out, x, t, k, 1.0 if T is None else T)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab", [(1, 152064), (3, 5003), (300, 4104)])
def test_equal_and_clustered_logits(rows, vocab, dtype):
    """Lists that overflow: constant rows, a handful of values, large values
    that few threads hold, rising and falling rows."""
    ko = _ko()
    g = torch.Generator().manual_seed(vocab)
    at = torch.arange(vocab)
    base = torch.randn(vocab, generator=g)
    cases = [torch.zeros(vocab), torch.full((vocab,), -3.0),
             torch.randint(0, 3, (vocab,), generator=g).float(),
             torch.where((at // 8) % 256 < 3, 5 + base, base - 20),
             torch.where((at // 4) % 512 < 2, 9.0, 1.0), at / vocab, -at / vocab,
             torch.where(at >= vocab - 300, 1.0, 0.0),
             torch.where(at % 2 == 0, -0.0, 0.0)]
    for n, row in enumerate(cases):
        x = row.to(dtype).expand(rows, vocab).contiguous()
        t = torch.randint(0, vocab, (rows,), generator=g)
        for k in (1, 20, 256):
            print(f"clustered {n} {rows} x {vocab} k={k} {dtype}", flush=True)
            out = ko.fused_top_logprobs(x.to(DEV), t.to(DEV), k)
            pick = sorted({0, rows // 2, rows - 1})
            _check([o[pick] for o in out], x[pick], t[pick], k)


@pytest.mark.parametrize("rows,vocab", [(2, 3), (2, 700), (1, 140001), (400, 9001)])
def test_masked_logits(rows, vocab):
    ko = _ko()
    g = torch.Generator().manual_seed(3)
    k = 20
    for dtype in DTYPES:
        full = torch.randn(rows, vocab, generator=g).to(dtype)
        for finite in (0, 1, 3, 19, 20, 21, 300):
            if finite > vocab:
                continue
            print(f"masked {rows} x {vocab} {dtype} {finite} finite", flush=True)
            x = torch.full_like(full, -float("inf"))
            keep = torch.randperm(vocab, generator=g)[:finite]
            x[:, keep] = full[:, keep]
            t = torch.randint(0, vocab, (rows,), generator=g)
            if finite and rows > 1:
                t[1] = keep[0]
            out = [o.cpu().numpy() for o in ko.fused_top_logprobs(x.to(DEV), t.to(DEV), k)]
            for i in range(min(rows, 3)):
                got = [o[i] for o in out]
                if finite:
                    _check_row(got, np64(x[i]), int(t[i]), k, 1.0)
                else:
                    assert np.isnan(got[0]) and np.isnan(got[1]) and got[2] == -np.inf
                    assert got[3] == int(t[i]) and (got[4] == -1).all()
                    assert (got[5] == -np.inf).all()


@pytest.mark.parametrize("rows,vocab", [(2, 700), (1, 140001), (300, 9001)])
def test_logits_masked_with_the_types_lowest_value(rows, vocab):
    """Whole rows of it are uniform; in others it is a weight of 0 that is
    listed behind every other."""
    ko = _ko()
    g = torch.Generator().manual_seed(5)
    k = 20
    for dtype in DTYPES:
        low = torch.finfo(dtype).min
        full = torch.randn(rows, vocab, generator=g).to(dtype)
        for keep in (0, 1, 19, 300):
            print(f"lowest {rows} x {vocab} {dtype} {keep} kept", flush=True)
            x = torch.full_like(full, low)
            at = torch.randperm(vocab, generator=g)[:keep]
            x[:, at] = full[:, at]
            t = torch.randint(0, vocab, (rows,), generator=g)
            out = [o.cpu().numpy() for o in ko.fused_top_logprobs(x.to(DEV), t.to(DEV), k)]
            for i in range(min(rows, 3)):
                _check_row([o[i] for o in out], np64(x[i]), int(t[i]), k, 1.0)


def test_rows_without_a_distribution():
    ko = _ko()
    for rows, vocab in ((1, 131072), (300, 9001)):
        for dtype in DTYPES:
            for bad in (float("nan"), float("inf")):
                x, t = _logits(rows, vocab, dtype, 9)
                x[rows // 2, vocab - 1] = bad
                out = ko.fused_top_logprobs(x.to(DEV), t.to(DEV), 7)
                row = [o[rows // 2].cpu() for o in out]
                assert row[3] == -1 and (row[4] == -1).all()
                assert all(r.isnan().all() for r in (*row[:3], row[5]))
                if rows > 1:
                    _check([o[:2] for o in out], x[:2], t[:2], 7)


def test_targets_outside_and_extreme_logits():
    ko = _ko()
    x, t = _logits(6, 1000, torch.float32, 5)
    t[:3] = torch.tensor([-100, 1000, 2 ** 40])
    x[3] *= 1e30
    x[4] = 3e38
    x[5] = -3e38
    x[5, 17] = -1e38
    out = ko.fused_top_logprobs(x.to(DEV), t.to(DEV), 4)
    _check([o[:3] for o in out], x[:3], t[:3], 4)
    assert (out[3][:3] == -1).all()
    assert (out[0][:3] == -out[2][:3]).all()
    for i in (3, 4, 5):
        want = top_oracle.forward_row(np64(x[i]), int(t[i]), 4)
        assert out[3][i] == want[3] and (out[4][i].cpu().numpy() == want[4]).all()
    # Peaked rows: log-probabilities next to 0 keep their precision.
    y = torch.full((1, 5000), -20.0)
    y[0, 11] = 15.0
    lp = ko.fused_top_logprobs(y.to(DEV), torch.tensor([11], device=DEV), 1)
    exact = -np.log1p(4999 * np.exp(-35.0))
    assert abs(float(lp[0]) - exact) <= 2 * U and abs(float(lp[5]) - exact) <= 2 * U


# ------------------------------------------------------------------------ gradients


def _grads(rows, k, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, generator=g), 0.3 * torch.randn(rows, generator=g),
            torch.randn(rows, generator=g), torch.randn(rows, k, generator=g))


def _check_grad(d, x, t, ids, T, g, dtype):
    """p: the saved lse's error and rounding, its exponent's roundings (of |y|
    and lse), the exponential; then the k-term sum and a few products."""
    d, xs, ids = np64(d), np64(x), ids.cpu().numpy()
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    for i in range(len(xs)):
        want, size = top_oracle.backward_row(xs[i], int(t[i]), ids[i], T,
                                             *(np64(v[i]) if v is not None else 0.0
                                               for v in g))
        tt = float(np.float32(T))
        err, _ = _sum_error(xs[i], tt)
        y = xs[i][np.isfinite(xs[i])] / tt
        rel = err + (8 * np.abs(y).max() + 8 * abs(y.max() + np.log(len(y))) + 300) * U
        bound = size * rel
        bound = bound + half * (np.abs(want) + bound) + tiny
        off = np.abs(d[i] - want) - bound
        assert (off <= 0).all(), (i, int(off.argmax()), float(off.max()))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 4), (4, 100, 256), (2, 1000, 20),
                                          (7, 4099, 64), (5, 50257, 33), (2, 152064, 128),
                                          (300, 2001, 20)])
def test_backward(rows, vocab, k, dtype):
    for T in (1.0, 0.7):
        print(f"top backward {rows} x {vocab} k={k} {dtype} T={T}", flush=True)
        x, t = _logits(rows, vocab, dtype, rows * 3 + vocab)
        t[0] = -100 if rows > 1 else t[0]
        leaf = x.to(DEV).requires_grad_()
        out = _ko().fused_top_logprobs(leaf, t.to(DEV), k, T)
        g = _grads(rows, k, vocab)
        of = [out[i] for i in (0, 1, 2, 5)]
        d, = torch.autograd.grad(of, leaf, [v.to(DEV) for v in g])
        assert d.dtype == dtype and d.shape == x.shape
        pick = range(rows) if rows < 10 else (0, 1, rows - 1)
        pick = list(pick)
        _check_grad(d[pick], x[pick], t[pick], out[4][pick], T, [v[pick] for v in g], dtype)


def test_each_gradient_alone_and_masked_rows():
    ko = _ko()
    x, t = _logits(5, 3001, torch.float32, 2)
    x[1, 100:] = -float("inf")       # fewer elements than alternatives
    x[2, ::2] = -float("inf")
    k = 128
    for which in range(4):
        leaf = x.to(DEV).requires_grad_()
        out = ko.fused_top_logprobs(leaf, t.to(DEV), k)
        g = _grads(5, k, which)[which]
        of = out[(0, 1, 2, 5)[which]]
        rows = [0, 1, 2, 3, 4]
        if which == 0:  # a masked target's -inf has a gradient of p alone
            t_ok = [i for i in rows if torch.isfinite(x[i, t[i]])]
        d, = torch.autograd.grad(of, leaf, g.to(DEV))
        gs = [g if i == which else None for i in range(4)]
        _check_grad(d, x, t, out[4], 1.0, gs, torch.float32)
        assert not d[1, 100:].any() or which == 0
    assert t_ok
    # Nothing asked for, nothing given.
    leaf = x.to(DEV)
    assert not any(o.requires_grad for o in ko.fused_top_logprobs(leaf, t.to(DEV), 3))
    out = ko.fused_top_logprobs(leaf.requires_grad_(), t.to(DEV), 3)
    assert [o.requires_grad for o in out] == [True, True, True, False, False, True]


def test_gradient_against_differences():
    """Along random directions, differences of the oracle's outputs in 64
    bits."""
    ko = _ko()
    x, t = _logits(2, 400, torch.float32, 12)
    k, T = 9, 1.3
    g = _grads(2, k, 1)
    leaf = x.to(DEV).requires_grad_()
    out = ko.fused_top_logprobs(leaf, t.to(DEV), k, T)
    d, = torch.autograd.grad([out[i] for i in (0, 1, 2, 5)], leaf, [v.to(DEV) for v in g])
    ids = out[4].cpu().numpy()

    def loss(v):
        total = 0.0
        for i in range(2):
            lp, ent, lse, _, order, top = top_oracle.forward_row(v[i], int(t[i]), k, T)
            assert (order == ids[i]).all()
            total += (lp * float(g[0][i]) + ent * float(g[1][i]) + lse * float(g[2][i])
                      + (top * np64(g[3][i])).sum())
        return total

    rng = np.random.RandomState(0)
    base = np64(x)
    for _ in range(5):
        v = rng.randn(*base.shape)
        e = 1e-5
        num = (loss(base + e * v) - loss(base - e * v)) / (2 * e)
        ana = (np64(d) * v).sum()
        # float32 gradients of at most 400 roundings and terms, and e^2.
        assert abs(num - ana) <= np.abs(np64(d) * v).sum() * 800 * U + 1e-7


def test_layouts():
    """Shifted windows, row strides, odd offsets, leading dims, one row used by
    all, no rows; targets with strides."""
    ko = _ko()
    g = torch.Generator().manual_seed(7)
    for dtype in DTYPES:
        base = torch.randn(3, 6, 5003, generator=g).to(dtype).to(DEV)
        t = torch.randint(0, 4000, (3, 6), generator=g).to(DEV)
        for x, tt in ((base, t), (base[:, :-1], t[:, 1:]), (base[..., 3:4103], t),
                      (base[0], t[0]), (base[1, 2], t[1, 2]), (base[:, 1:2].expand(3, 6, 5003), t)):
            out = ko.fused_top_logprobs(x, tt, 11)
            want = ko.fused_top_logprobs(x.contiguous(), tt.contiguous(), 11)
            assert [o.shape for o in out] == [tt.shape] * 4 + [(*tt.shape, 11)] * 2
            for i in (3, 4):
                assert torch.equal(out[i], want[i])
            # Another alignment adds the same weights in another order.
            for i in (0, 1, 2, 5):
                assert (out[i] - want[i]).abs().max() <= 2e-5
            leaf = x.detach().requires_grad_()
            o = ko.fused_top_logprobs(leaf, tt, 11)
            d, = torch.autograd.grad(o[5].sum() + o[0].sum(), leaf)
            assert d.shape == x.shape
        e = ko.fused_top_logprobs(base[:0], t[:0], 4)
        assert [o.shape for o in e] == [(0, 6)] * 4 + [(0, 6, 4)] * 2
        leaf = base[:0].detach().requires_grad_()
        d, = torch.autograd.grad(ko.fused_top_logprobs(leaf, t[:0], 4)[0].sum(), leaf)
        assert d.shape == (0, 6, 5003)


def test_second_derivative_is_refused():
    from kernel_opt.top import _FusedTopLogprobs
    x, t = _logits(3, 50, torch.float32, 1)
    for f in (_ko().fused_top_logprobs, lambda a, b, k: _FusedTopLogprobs.apply(a, b, k, 1.0)):
        leaf = x.to(DEV).requires_grad_()
        out = f(leaf.tanh(), t.to(DEV), 5)
        d, = torch.autograd.grad(out[0].sum() + out[5].sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="no second derivative"):
            torch.autograd.grad(d.square().sum(), leaf)


def test_statement_streams_threads_and_graphs():
    """The same bits from the compiled function, its Python statement, other
    streams, threads at once, and replays of two graphs captured on one stream."""
    ko = _ko()
    from kernel_opt.top import _FusedTopLogprobs
    for rows, vocab in ((2, 140000), (600, 5000)):
        x, t = _logits(rows, vocab, torch.bfloat16, 4)
        x, t = x.to(DEV), t.to(DEV)
        leaf = x.clone().requires_grad_()
        g = [v.to(DEV) for v in _grads(rows, 20, 6)]

        def step(f=ko.fused_top_logprobs, args=()):
            out = f(leaf, t, 20, *args)
            d, = torch.autograd.grad([out[i] for i in (0, 1, 2, 5)], leaf, g)
            return [o.detach().clone() for o in (*out, d)]

        def same(a, b):
            return all(torch.equal(p, q) for p, q in zip(a, b))

        want = step()
        for _ in range(3):
            assert same(want, step())
        assert same(want, step(_FusedTopLogprobs.apply, (1.0,)))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step()
        torch.cuda.current_stream().wait_stream(s)
        assert same(want, got)
        torch.cuda.synchronize()
        found = [None] * 3

        def work(i):
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    found[i] = [o.clone() for o in ko.fused_top_logprobs(x, t, 20)]
            stream.synchronize()

        threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        assert all(same(want[:6], f) for f in found)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                out = step()
            graphs.append((graph, out))
        for rep in range(3):
            with torch.no_grad():
                leaf.copy_(torch.randn_like(x, dtype=torch.float32))
            a, b = torch.cuda.Stream(), torch.cuda.Stream()
            for st, (graph, _) in zip((a, b), graphs):  # at once
                st.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(st):
                    graph.replay()
            torch.cuda.synchronize()
            now = step()
            assert same(graphs[0][1], now) and same(graphs[1][1], now)


def test_rows_beyond_32_bits():
    ko = _ko()
    rows, vocab = 2 ** 15 + 3, 2 ** 16 + 5
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEV)
    x[-2:] = torch.randn(2, vocab, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    t = torch.full((rows,), 5, device=DEV)
    out = ko.fused_top_logprobs(x, t, 12)
    few = ko.fused_top_logprobs(x[-2:], t[-2:], 12)
    assert torch.equal(out[4][-2:], few[4]) and torch.equal(out[3][-2:], few[3])
    assert (out[5][-2:] - few[5]).abs().max() <= 2e-5
    # A row of 2^25 columns, its largest at the far end.
    v = 2 ** 25 + 3
    y = torch.zeros(1, v, device=DEV)
    y[0, -1], y[0, -5] = 3.0, 2.0
    o = ko.fused_top_logprobs(y, torch.tensor([v - 5], device=DEV), 4)
    assert o[4].tolist() == [[v - 1, v - 5, 0, 1]] and o[3].tolist() == [1]


def test_refusals():
    ko = _ko()
    x = torch.zeros(4, 64, device=DEV)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad, text in ((x.double(), "dtype"), (x[:, :0], "last dim"), (x.t()[:4], "contiguous"),
                      (x.cpu(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=text):
            ko.fused_top_logprobs(bad, t, 3)
    for bad, text in ((t[:3], "targets must be"), (t.int(), "int64"), (t.cpu(), "GPU tensors")):
        with pytest.raises(RuntimeError, match=text):
            ko.fused_top_logprobs(x, bad, 3)
    for k in (0, 257, 2.5, True, -1):
        with pytest.raises(ValueError, match="k must be"):
            ko.fused_top_logprobs(x, t, k)
    for T in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="temperature"):
            ko.fused_top_logprobs(x, t, 3, T)
