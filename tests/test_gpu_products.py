"""Products of a training step on the GPU against their definitions in float64: the
loss over a vocabulary without its logits, the experts' products and the
orthogonalised updates, values and every gradient.

Bars are normwise (max |error| / max |value|) and count roundings of half a step u
(2^-24, 2^-53). A sum of n products of random signs makes n roundings, each of at most u
of a partial sum that grows as the square root: 0.41 sqrt(n) u of its own size in the
mean square, and the largest of many such errors, against the largest of as many
values, keeps that ratio. bar(n) = 4 (sqrt(n) + 8) u is about ten times that. What
follows a sum adds its own: a logit's error counts in the exponential with the logit's
size (below 6 here) and the exponential's argument in base 2 with as much again."""
import math

import numpy as np
import pytest
import torch

from helpers import bits_equal

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64
U = {F32: 2.0 ** -24, F64: 2.0 ** -53}


def _mods():
    from dtmi import autograd as A, device as D
    return A, D


def bar(*sums):
    return 4 * sum(math.sqrt(n) + 8 for n in sums)


def close(got, want, dt, roundings, what):
    got = np.asarray(got.numpy() if hasattr(got, "numpy") else got, np.float64)
    want = want.detach().numpy() if isinstance(want, torch.Tensor) else np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.size:
        return
    assert np.isfinite(got).all(), what
    err, top = np.abs(got - want).max(), np.abs(want).max()
    assert err <= roundings * U[dt] * max(top, 1e-300), (what, err / max(top, 1e-300) / U[dt], roundings)


def t64(a, grad=True):
    return torch.tensor(np.asarray(a, np.float64), requires_grad=grad)


# -------------------------------------------------------------------- loss
LOSS = [  # rows, C, V, bias, tied, ignored targets
    (1, 1, 1, False, False, 0),
    (1, 8, 3, True, False, 0),
    (5, 64, 64, False, False, 0),
    (7, 36, 65, True, True, 0),
    (64, 128, 65, False, False, 9),
    (65, 33, 130, True, False, 64),
    (129, 68, 513, True, True, 5),
    (200, 96, 1000, False, True, 0),
    (333, 51, 777, True, False, 100),
    (130, 132, 4100, True, False, 0),
    (16, 300, 1000, True, True, 0),      # few rows
    (32, 515, 777, True, False, 2),
    (17, 1030, 514, False, True, 0),
    (31, 90, 1029, False, False, 0),
    (2, 129, 3001, True, False, 0),      # few rows and many words
    (17, 40, 9001, False, True, 3),
    (32, 70, 6000, True, False, 0),
]


def loss_inputs(case, dt, seed=0):
    R, C, V, bias, tied, ign = case
    rng = np.random.default_rng(R * 7 + V + seed)
    x = rng.standard_normal((R, C)).astype(dt)
    w = (rng.standard_normal((V, C) if tied else (C, V)) * 1.2 / math.sqrt(C)).astype(dt)
    b = (0.5 * rng.standard_normal(V)).astype(dt) if bias else None
    t = rng.integers(0, V, R)
    if ign:
        t[rng.permutation(R)[:ign]] = -100
    return x, w, b, t


def loss_ref(x, w, b, t, tied, reduction, g=None):
    x, w = t64(x), t64(w)
    leaves = [x, w] + ([t64(b)] if b is not None else [])
    z = x @ (w.T if tied else w) + (leaves[2] if b is not None else 0.0)
    ok = torch.tensor(t >= 0)
    l = torch.logsumexp(z, 1) - z[torch.arange(len(t)), torch.tensor(np.maximum(t, 0))]
    l = torch.where(ok, l, torch.zeros_like(l))
    y = l.sum() / max(1, int(ok.sum())) if reduction == "mean" else l
    gr = torch.autograd.grad(y, leaves, torch.tensor(np.asarray(g, np.float64)) if g is not None else None)
    return y, gr


def loss_bars(C, R, V):
    z = 6 * (math.sqrt(C) + 8) + 24   # of the exponential
    return 4 * (z + math.sqrt(V)), 4 * (z + math.sqrt(V)), 4 * (z + math.sqrt(R))


def loss_run(case, dt, reduction, g, hide=True, ignore=-100):
    A, D = _mods()
    R, C, V, bias, tied, ign = case
    x, w, b, t = loss_inputs(case, dt)
    xh = x.copy()
    if hide:
        xh[t < 0] = np.nan   # what lies there is not read
    X = A.Tensor(D.from_numpy(xh), requires_grad=True)
    W = A.Tensor(D.from_numpy(w), requires_grad=True)
    Bt = A.Tensor(D.from_numpy(b), requires_grad=True) if bias else None
    y = A.linear_cross_entropy(X, W.transpose(1, 0) if tied else W, t, Bt, ignore=ignore if ign else None,
                               reduction=reduction)
    y.backward(D.from_numpy(np.asarray(g, dt)) if g is not None else None)
    return (x, w, b, t), y, [X.grad, W.grad] + ([Bt.grad] if bias else [])


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("case", LOSS, ids=lambda c: "-".join(str(int(v)) for v in c))
def test_loss(dev, dt, reduction, case):
    R, C, V, bias, tied, ign = case
    g = None if reduction == "mean" else np.random.default_rng(1).standard_normal(R).astype(dt)
    (x, w, b, t), y, grads = loss_run(case, dt, reduction, g)
    ry, rg = loss_ref(x, w, b, t, tied, reduction, g)
    by, bx, bw = loss_bars(C, R, V)
    # a loss of nearly 0 is the difference of two logits
    top = float(ry.detach().abs().max())
    close(y, ry, dt, by * max(1.0, 6.0 / top if top else 1.0), "loss")
    for got, want, n, name in zip(grads, rg, (bx, bw, bw), ("dx", "dw", "db")):
        # what p - 1 cancels: the largest gradients have p far from 1, but for V = 1
        if V == 1:
            assert np.abs(got.numpy()).max() <= 8 * U[dt], name
        else:
            close(got, want, dt, n, name)
    if ign:
        assert not grads[0].numpy()[t < 0].any()


@pytest.mark.parametrize("case", [
    (3000, 12, 50001, True, False, 300),   # float64: three pieces of logits
    (1100, 9, 130003, False, True, 0),     # a vocabulary of which a piece is the fewest rows
], ids=["three", "fewest"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_over_pieces_of_rows(dev, case, reduction):
    """More logits than a piece holds (1 GiB, 1024 rows at least)."""
    g = None if reduction == "mean" else np.random.default_rng(1).standard_normal(case[0])
    (x, w, b, t), y, grads = loss_run(case, F64, reduction, g)
    ry, rg = loss_ref(x, w, b, t, case[4], reduction, g)
    by, bx, bw = loss_bars(case[1], case[0], case[2])
    close(y, ry, F64, by, "loss")
    for got, want, n, name in zip(grads, rg, (bx, bw, bw), ("dx", "dw", "db")):
        close(got, want, F64, n, name)


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("C,V", [(37, 131), (36, 131), (37, 132)])
def test_loss_of_odd_sizes_and_many_rows(dev, dt, tied, C, V):
    case = (1030, C, V, True, tied, 13)
    for reduction in ("mean", "none"):
        g = None if reduction == "mean" else np.random.default_rng(1).standard_normal(case[0]).astype(dt)
        (x, w, b, t), y, grads = loss_run(case, dt, reduction, g)
        ry, rg = loss_ref(x, w, b, t, tied, reduction, g)
        by, bx, bw = loss_bars(C, 1030, V)
        close(y, ry, dt, by, "loss")
        for got, want, n, name in zip(grads, rg, (bx, bw, bw), ("dx", "dw", "db")):
            close(got, want, dt, n, (reduction, name))


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("tied", [False, True])
def test_loss_whose_gradients_are_grouped_products(dev, dt, tied):
    """Odd sizes of 1e9 operations and more: all gradients, and each by itself."""
    A, D = _mods()
    case = (1030, 259, 2001, True, tied, 7)
    (x, w, b, t), y, grads = loss_run(case, dt, "mean", None)
    ry, rg = loss_ref(x, w, b, t, tied, "mean")
    by, bx, bw = loss_bars(*case[1:2], case[0], case[2])
    close(y, ry, dt, by, "loss")
    for got, want, n, name in zip(grads, rg, (bx, bw, bw), ("dx", "dw", "db")):
        close(got, want, dt, n, name)
    for i in range(3):
        X, W, B = (A.Tensor(D.from_numpy(v), requires_grad=i == j) for j, v in enumerate((x, w, b)))
        A.linear_cross_entropy(X, W.transpose(1, 0) if tied else W, t, B, ignore=-100).backward()
        assert [p.grad is None for p in (X, W, B)] == [i != j for j in range(3)]
        close((X, W, B)[i].grad, rg[i], dt, (bx, bw, bw)[i], i)


@pytest.mark.parametrize("dt", [F32, F64])
def test_loss_on_wide_tiles(dev, dt):
    """Enough rows and columns for 128-wide tiles, with edges in both."""
    case = (2100, 72, 2500, False, False, 0)
    (x, w, b, t), y, grads = loss_run(case, dt, "mean", None)
    ry, rg = loss_ref(x, w, b, t, False, "mean")
    by, bx, bw = loss_bars(case[1], case[0], case[2])
    close(y, ry, dt, by, "loss")
    close(grads[0], rg[0], dt, bx, "dx")
    close(grads[1], rg[1], dt, bw, "dw")
    again = loss_run(case, dt, "mean", None)[2]
    assert all(bits_equal(a.numpy(), c.numpy()) for a, c in zip(grads, again))


def test_losses_without_gradients_are_the_same(dev):
    A, D = _mods()
    case = (37, 96, 1001, True, False, 4)
    (x, w, b, t), y, _ = loss_run(case, F32, "none", np.ones(37))
    with A.no_grad():
        z = A.linear_cross_entropy(A.Tensor(x), A.Tensor(w), A.Indices(t), A.Tensor(b), ignore=-100, reduction="none")
    assert bits_equal(y.numpy(), z.numpy())
    assert z._backward is None


@pytest.mark.parametrize("case", [
    (70, 64, 130, True, False, 41),       # ignored rows gone through with the others
    (700, 256, 8000, False, True, 500),   # left out: 2 * 500 * 256 * 8000 operations
], ids=["few", "many"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("ignore", [-100, 2 ** 40, 3])
def test_losses_alone_beside_ignored_rows(dev, case, reduction, ignore):
    A, D = _mods()
    x, w, b, t = loss_inputs(case, F32)
    out = t < 0
    t[~out & (t == ignore)] = 4
    ry, _ = loss_ref(x, w, b, t, case[4], reduction, None if reduction == "mean" else np.ones(len(t)))
    t[out], x[out] = ignore, np.nan
    W = A.Tensor(w).transpose(1, 0) if case[4] else A.Tensor(w)
    with A.no_grad():
        y = A.linear_cross_entropy(A.Tensor(x), W, A.Indices(t), A.Tensor(b) if case[3] else None, ignore=ignore,
                                   reduction=reduction)
    close(y, ry, F32, loss_bars(case[1], case[0], case[2])[0], "loss")
    if reduction == "none":
        assert not y.numpy()[out].any()


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("ign", [1, 4000, 9999])
def test_loss_leaves_rows_out_of_many(dev, dt, reduction, ign):
    case = (10000, 5, 7, True, False, ign)
    g = None if reduction == "mean" else np.random.default_rng(1).standard_normal(case[0]).astype(dt)
    (x, w, b, t), y, grads = loss_run(case, dt, reduction, g)
    ry, rg = loss_ref(x, w, b, t, False, reduction, g)
    by, bx, bw = loss_bars(5, 10000, 7)
    close(y, ry, dt, by, "loss")
    for got, want, n, name in zip(grads, rg, (bx, bw, bw), ("dx", "dw", "db")):
        close(got, want, dt, n, name)
    assert not grads[0].numpy()[t < 0].any()


def test_ones_are_written_when_they_are_asked_for(dev):
    """backward()'s own gradient: what reads it finds ones, also in a view and twice over."""
    A, D = _mods()
    for dt in (F32, F64):
        g = D.ones_later((2, 3), dt)
        v = g.reshape(6)[1:]
        assert D.known_ones(g) and D.known_ones(v)
        assert (v.numpy() == 1).all() and not D.known_ones(g) and not D.known_ones(v)
        v.assign(2.0)
        assert g.numpy().tolist() == [[1, 2, 2], [2, 2, 2]]
        x = A.Tensor(np.asarray(3.0, dt), requires_grad=True)
        x.backward()
        x.backward()
        assert float(x.grad) == 2.0


@pytest.mark.parametrize("dest", [False, True])
def test_gradients_of_a_mean_by_itself_and_scaled(dev, dest):
    """backward() leaves them as the forward pass made them, backward(g) scales them."""
    A, D = _mods()
    x, w, b, t = loss_inputs((40, 24, 130, True, False, 0), F32)
    got = []
    for g in (None, 1.0, 0.5):
        X, W, B = (A.Tensor(D.from_numpy(v), requires_grad=True) for v in (x, w, b))
        if dest:
            W.grad_dest = D.zeros(w.shape, F32)
        A.linear_cross_entropy(X, W, t, B).backward(g)
        assert not dest or W.grad.ptr == W.grad_dest.ptr
        got.append([p.grad.numpy() for p in (X, W, B)])
    for one, same, half in zip(*got):
        assert bits_equal(one, same) and bits_equal(0.5 * one, half)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_loss_with_every_target_ignored(dev, reduction):
    A, D = _mods()
    X = A.Tensor(np.full((3, 8), np.nan, F32), requires_grad=True)
    W = A.Tensor(np.ones((8, 5), F32), requires_grad=True)
    b = A.Tensor(np.ones(5, F32), requires_grad=True)
    y = A.linear_cross_entropy(X, W, [7, 7, 7], b, ignore=7, reduction=reduction)
    assert not np.any(y.numpy()) and y.shape == (() if reduction == "mean" else (3,))
    y.backward(D.from_numpy(np.ones(y.shape, F32)))
    assert all(not np.any(p.grad.numpy()) and p.grad.shape == p.shape for p in (X, W, b))


def test_loss_without_rows(dev):
    A, D = _mods()
    X, W = A.Tensor(np.ones((0, 8)), requires_grad=True), A.Tensor(np.ones((8, 5)), requires_grad=True)
    y = A.linear_cross_entropy(X, W, np.zeros(0, np.int64))
    y.backward()
    assert float(y.numpy()) == 0 and not W.grad.numpy().any() and X.grad.shape == (0, 8)
    assert A.linear_cross_entropy(X, W, np.zeros(0, np.int64), reduction="none").shape == (0,)


def test_loss_without_inputs(dev):
    """C = 0: the bias alone."""
    A, D = _mods()
    b = np.array([0.0, 1.0, -2.0])
    X, W, B = (A.Tensor(v, requires_grad=True) for v in (np.ones((4, 0)), np.ones((0, 3)), b))
    y = A.linear_cross_entropy(X, W, [0, 1, 2, 1], B)
    y.backward()
    p = np.exp(b) / np.exp(b).sum()
    close(y, -(np.log(p)[[0, 1, 2, 1]]).mean(), F64, 64, "loss")
    close(B.grad, p - np.array([0.25, 0.5, 0.25]), F64, 64, "db")
    assert X.grad.shape == (4, 0) and W.grad.shape == (0, 3)


def test_loss_masked_vocabulary(dev):
    """Entries that a bias of -inf or of the type's lowest value takes out (a padded
    vocabulary): no probability, no gradient; whole tiles of them too."""
    A, D = _mods()
    R, C, V, real = 70, 32, 600, 130
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((R, C)).astype(F32), (rng.standard_normal((C, V)) * 0.2).astype(F32)
    t = rng.integers(0, real, R)
    ry, (rx, rw) = loss_ref(x, w[:, :real], None, t, False, "mean")
    for low in (-np.inf, float(np.finfo(F32).min)):
        b = np.zeros(V, F32)
        b[real:] = low
        X, W = A.Tensor(x, requires_grad=True), A.Tensor(w, requires_grad=True)
        y = A.linear_cross_entropy(X, W, t, A.Tensor(b))
        y.backward()
        by, bx, bw = loss_bars(C, R, V)
        close(y, ry, F32, by, "loss")
        close(X.grad, rx, F32, bx, "dx")
        close(W.grad.numpy()[:, :real], rw, F32, bw, "dw")
        assert not W.grad.numpy()[:, real:].any()


def test_loss_of_large_logits(dev):
    """Logits of thousands: differences count, neither overflow nor a lost row."""
    A, D = _mods()
    x = np.array([[3000.0, 1.0], [-3000.0, 1.0], [1.0, 0.0]])
    w = np.array([[1.0, 0.999, -1.0], [0.0, 0.5, 0.25]])
    t = [1, 2, 0]
    for dt in (F32, F64):
        l = A.linear_cross_entropy(A.Tensor(x.astype(dt)), A.Tensor(w.astype(dt)), t, reduction="none")
        z = x.astype(dt).astype(F64) @ w.astype(dt).astype(F64)
        want = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1) - z[np.arange(3), t]
        # the logits' own rounding, 3000 u a product
        assert np.abs(l.numpy() - want).max() <= 8 * 3000 * U[dt]


def test_loss_nan_and_infinity_show(dev):
    A, D = _mods()
    x = np.ones((3, 4), F32)
    x[1, 2] = np.nan
    x[2, 1] = np.inf
    l = A.linear_cross_entropy(A.Tensor(x), A.Tensor(np.ones((4, 70), F32)), [0, 1, 2], reduction="none").numpy()
    assert np.isfinite(l[0]) and not np.isfinite(l[1:]).any()


def test_loss_gradients_are_scaled_shared_and_taken_twice(dev):
    """An upstream gradient that is not 1, w in two places, a second backward through the
    same node, gradients not asked for, and a destination for w's."""
    A, D = _mods()
    case = (50, 48, 99, True, False, 6)
    x, w, b, t = loss_inputs(case, F64)
    _, (rx, rw, rb) = loss_ref(x, w, b, t, False, "mean")
    X, W, B = (A.Tensor(v, requires_grad=True) for v in (x, w, b))
    y = A.linear_cross_entropy(X, W, t, B, ignore=-100)
    (y * 0.25).backward()
    _, bx, bw = loss_bars(48, 50, 99)
    for p, r, n in ((X, rx, bx), (W, rw, bw), (B, rb, bw)):
        close(p.grad, 0.25 * r, F64, n, "scaled")
        p.grad = None
    y.backward()
    for p, r, n in ((X, rx, bx), (W, rw, bw), (B, rb, bw)):
        close(p.grad, r, F64, n, "second")
        p.grad = None
    W.grad_dest = D.full(w.shape, 7.0, F64)
    B.grad_dest = D.full(b.shape, 7.0, F64)
    (A.linear_cross_entropy(X, W, t, B, ignore=-100) * 0.5).backward()
    assert W.grad.ptr == W.grad_dest.ptr and B.grad.ptr == B.grad_dest.ptr
    close(W.grad, 0.5 * rw, F64, bw, "destination")
    W2, X2 = A.Tensor(w, requires_grad=True), A.Tensor(x)
    (A.linear_cross_entropy(X2, W2, t, A.Tensor(b), ignore=-100) +
     A.linear_cross_entropy(X2, W2, t, A.Tensor(b), ignore=-100)).backward()
    close(W2.grad, 2 * rw, F64, bw, "two uses")
    assert X2.grad is None


def test_loss_with_split_bf16_products(dev):
    """Its gradient products follow the GEMM arithmetic that is set."""
    from dtmi import _lib
    case = (260, 64, 512, False, False, 0)
    want = loss_ref(*loss_inputs(case, F32), False, "mean")
    with _lib.use_gemm_math("bf16x6"):
        _, y, grads = loss_run(case, F32, "mean", None)
    by, bx, bw = loss_bars(64, 260, 512)
    close(y, want[0], F32, by, "loss")
    close(grads[0], want[1][0], F32, bx, "dx")
    close(grads[1], want[1][1], F32, bw, "dw")


def test_loss_of_one_position(dev):
    """x without leading axes, a target without any."""
    A, D = _mods()
    x, w = np.linspace(-1, 1, 6), np.linspace(0, 2, 24).reshape(6, 4)
    for reduction in ("mean", "none"):
        X = A.Tensor(x, requires_grad=True)
        y = A.linear_cross_entropy(X, A.Tensor(w), 2, reduction=reduction)
        y.backward()
        z = x @ w
        p = np.exp(z - z.max()) / np.exp(z - z.max()).sum()
        assert y.shape == () and X.grad.shape == (6,)
        close(y, -np.log(p[2]), F64, 64, "loss")
        close(X.grad, w @ (p - np.eye(4)[2]), F64, 64, "dx")


def test_loss_matches_its_differences(dev):
    A, D = _mods()
    case = (20, 12, 33, True, False, 3)
    x, w, b, t = loss_inputs(case, F64)
    g = np.random.default_rng(2).standard_normal(20)
    _, _, grads = loss_run(case, F64, "none", g, hide=False)
    rng = np.random.default_rng(4)
    for i, (v, d) in enumerate(zip((x, w, b), grads)):
        e = rng.standard_normal(v.shape)
        h = 1e-5

        def f(s):
            a = [x, w, b]
            a[i] = v + s * h * e
            with A.no_grad():
                l = A.linear_cross_entropy(*[A.Tensor(q) for q in a[:2]], t, A.Tensor(a[2]), ignore=-100,
                                           reduction="none")
            return float((l.numpy() * g).sum())
        # h^2 of the third derivative and rounding / h, both near 1e-10
        assert abs((f(1) - f(-1)) / (2 * h) - float((d.numpy() * e).sum())) <= 1e-7


def test_gpt_loss_is_the_forward_loss(dev):
    from dtmi import nn as N
    cfg = N.GPTConfig(vocab=65, ctx=16, dim=32, heads=4, layers=2, dtype="float64")
    m = N.GPT(cfg, seed=1)
    rng = np.random.default_rng(0)
    x, y = rng.integers(0, 65, (3, 16)), rng.integers(0, 65, (3, 16))
    _, a = m(x, y)
    a.backward()
    want = [p.grad.numpy() for p in m.parameters()]
    m.zero_grad()
    b = m.loss(x, y)
    b.backward()
    assert abs(float(a.numpy()) - float(b.numpy())) <= 1e-13 * abs(float(a.numpy()))
    for (name, p), r in zip(m.named_parameters(), want):
        assert np.abs(p.grad.numpy() - r).max() <= 1e-12 * max(np.abs(r).max(), 1e-300), name
    assert m.loss(x, y, reduction="none").shape == (3, 16)


# ----------------------------------------------------------------- experts
EXPERTS = [  # R, K, N, sizes, bias
    (1, 1, 1, [1], True),
    (5, 8, 12, [2, 0, 3], True),
    (40, 33, 65, [40], False),
    (70, 36, 64, [0, 1, 64, 5], True),
    (200, 64, 132, [3, 130, 0, 0, 50], True),
    (300, 100, 30, [0, 0], True),
    (515, 68, 257, [128, 129, 0, 255, 1], True),
    (600, 48, 20, [4] * 70 + [1, 100, 219], False),   # more experts than a launch holds
    (20, 515, 201, [16, 0, 4], True),                 # few rows each
    (41, 770, 131, [32, 7, 1], False),
    (9, 36, 1000, [1, 8], True),
    (24, 5003, 70, [16, 0, 5], True),                 # and long rows, split over blocks
    (33, 60, 4100, [1, 32], False),
    (5000, 24, 40, [4000, 999], True),                # sums over rows long enough to be split
]


def experts_ref(x, w, b, g, sizes):
    x, w = t64(x), t64(w)
    leaves = [x, w] + ([t64(b)] if b is not None else [])
    at, parts = 0, []
    for e, n in enumerate(sizes):
        parts.append(x[at:at + n] @ w[e] + (leaves[2][e] if b is not None else 0.0))
        at += n
    y = torch.cat(parts + [torch.zeros(x.shape[0] - at, w.shape[2], dtype=torch.float64) + 0 * w.sum()])
    return y, torch.autograd.grad(y, leaves, t64(g, False))


def experts_run(x, w, b, g, sizes, hide=True):
    A, D = _mods()
    used = sum(sizes)
    x, g = x.copy(), g.copy()
    if hide:
        x[used:], g[used:] = np.nan, np.nan
    X, W = A.Tensor(x, requires_grad=True), A.Tensor(w, requires_grad=True)
    B = A.Tensor(b, requires_grad=True) if b is not None else None
    y = A.expert_linear(X, W, sizes, B)
    y.backward(D.from_numpy(g))
    return y, [X.grad, W.grad] + ([B.grad] if b is not None else [])


def experts_inputs(R, K, N, E, bias, dt):
    rng = np.random.default_rng(R + K * 3 + N)
    return ((rng.standard_normal((R, K))).astype(dt), (rng.standard_normal((E, K, N)) / math.sqrt(K)).astype(dt),
            rng.standard_normal((E, N)).astype(dt) if bias else None, rng.standard_normal((R, N)).astype(dt))


def experts_check(R, K, N, sizes, bias, dt):
    x, w, b, g = experts_inputs(R, K, N, len(sizes), bias, dt)
    y, grads = experts_run(x, w, b, g, sizes)
    ry, rg = experts_ref(x, w, b, g, sizes)
    close(y, ry, dt, bar(K), "y")
    for got, want, n, name in zip(grads, rg, (N, max(sizes), max(sizes)), ("dx", "dw", "db")):
        close(got, want, dt, bar(n), name)
    used = sum(sizes)
    assert not y.numpy()[used:].any() and not grads[0].numpy()[used:].any()
    return y, grads


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", EXPERTS, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{len(c[3])}")
def test_experts(dev, dt, case):
    experts_check(*case, dt)


@pytest.mark.parametrize("dt", [F32, F64])
def test_experts_on_wide_tiles(dev, dt):
    first = experts_check(3000, 392, 516, [900, 1, 700, 0, 1300], True, dt)
    again = experts_check(3000, 392, 516, [900, 1, 700, 0, 1300], True, dt)
    assert bits_equal(first[0].numpy(), again[0].numpy())
    assert all(bits_equal(a.numpy(), c.numpy()) for a, c in zip(first[1], again[1]))


def test_experts_without_rows_inputs_outputs_or_experts(dev):
    A, D = _mods()
    for R, K, N, sizes in ((0, 4, 3, [0, 0]), (4, 0, 3, [1, 2]), (4, 3, 0, [1, 2]), (4, 3, 5, [])):
        x, w, b, g = experts_inputs(R, max(K, 1), max(N, 1), len(sizes), True, F64)
        x, w, b, g = x[:, :K], w[:, :K, :N], b[:, :N], g[:, :N]
        y, grads = experts_run(x, w, b, g, sizes)
        assert y.shape == (R, N) and [d.shape for d in grads] == [(R, K), (len(sizes), K, N), (len(sizes), N)]
        at, want, db = 0, np.zeros((R, N)), np.zeros((len(sizes), N))
        for e, n in enumerate(sizes):
            want[at:at + n] = b[e]
            db[e] = g[at:at + n].sum(0)
            at += n
        if K == 0:
            close(y, want, F64, 2, "y")
            close(grads[2], db, F64, 4, "db")


def test_experts_strided_operands_and_destinations(dev):
    """x a transposed view, sizes as Indices, gradients into their destinations, an
    expert's weights used twice."""
    A, D = _mods()
    sizes = [5, 0, 7]
    x, w, b, g = experts_inputs(13, 8, 6, 3, True, F64)
    X0 = A.Tensor(np.ascontiguousarray(x.T), requires_grad=True)
    W, B = A.Tensor(w, requires_grad=True), A.Tensor(b, requires_grad=True)
    W.grad_dest, B.grad_dest = D.full(w.shape, 7.0, F64), D.full(b.shape, 7.0, F64)
    y = A.expert_linear(X0.transpose(1, 0), W, A.Indices(sizes), B)
    y.backward(D.from_numpy(np.ascontiguousarray(g.T)).transpose(1, 0))
    ry, (rx, rw, rb) = experts_ref(x, w, b, g, sizes)
    close(y, ry, F64, bar(8), "y")
    close(X0.grad, rx.T, F64, bar(6), "dx")
    close(W.grad, rw, F64, bar(7), "dw")
    assert W.grad.ptr == W.grad_dest.ptr and B.grad.ptr == B.grad_dest.ptr
    W2, X2 = A.Tensor(w, requires_grad=True), A.Tensor(x)
    (A.expert_linear(X2, W2, sizes) + A.expert_linear(X2, W2, sizes)).backward(D.from_numpy(g))
    close(W2.grad, 2 * rw, F64, bar(7), "two uses")
    assert X2.grad is None


def test_experts_match_their_differences(dev):
    A, D = _mods()
    sizes = [3, 0, 9, 2]
    x, w, b, g = experts_inputs(15, 10, 7, 4, True, F64)
    _, grads = experts_run(x, w, b, g, sizes, hide=False)
    rng = np.random.default_rng(5)
    for i, (v, d) in enumerate(zip((x, w, b), grads)):
        e = rng.standard_normal(v.shape)

        def f(s):
            a = [x, w, b]
            a[i] = v + s * 1e-3 * e
            return float((A.expert_linear(A.Tensor(a[0]), A.Tensor(a[1]), sizes, A.Tensor(a[2])).numpy() * g).sum())
        # bilinear: the difference is exact but for rounding, 1e-15 * 1e2 / 1e-3
        assert abs((f(1) - f(-1)) / 2e-3 - float((d.numpy() * e).sum())) <= 1e-9


# ----------------------------------------------------------------- updates
COEF = (3.4445, -4.7750, 2.0315)


def ns_ref(g, steps, coef, eps):
    """Through the singular values, in float64: U f(s) V^T."""
    u, s, vt = np.linalg.svd(np.asarray(g, np.float64), full_matrices=False)
    s = s / (np.sqrt((s * s).sum()) + eps)
    slope, v = np.ones_like(s), s.copy()
    for _ in range(steps):
        a, b, c = coef
        slope = slope * (a + 3 * b * v ** 2 + 5 * c * v ** 4)
        v = a * v + b * v ** 3 + c * v ** 5
    # what noise in X grows by: along a singular direction, and across two
    grow = max(np.abs(slope).max(), (np.abs(v) / np.maximum(s, 1e-300)).max(), 1.0) if s.size else 1.0
    return (u * v) @ vt, grow


def ns_bar(g, ref, grow, steps, dt):
    """steps + 1 roundings of X (and of the sums that make it) each grow by `grow` at
    most: relative to the result's largest entry."""
    m, n = g.shape
    g = np.asarray(g, np.float64)
    top = np.abs(g).max() / np.linalg.norm(g)
    return 4 * (steps + 1) * (0.5 * math.sqrt(max(m, n)) + 8) * grow * max(top / np.abs(ref).max(), 1.0 / grow)


def check_ns(got, g, dt, steps=5, coef=COEF, eps=1e-7, what=""):
    ref, grow = ns_ref(g, steps, coef, eps)
    close(got, ref, dt, ns_bar(g, ref, grow, steps, dt), what)


SHAPES = [(1, 1), (1, 9), (9, 1), (3, 5), (64, 64), (65, 63), (36, 132), (200, 68), (130, 257), (129, 400), (33, 2000)]


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}")
def test_orthogonalize(dev, dt, shape):
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    g = (np.random.default_rng(shape[0] * 3 + shape[1]).standard_normal(shape) * 1e-3).astype(dt)
    got = orthogonalize(D.from_numpy(g))
    check_ns(got, g, dt)
    assert bits_equal(got.numpy(), orthogonalize(D.from_numpy(g)).numpy())


# blocks of 16 rows, 2, 4 and 6 of them; columns that 8 or 16 waves share or go through in
# turn; as much as a block holds (float32) and more; a square that only the groups take
SMALL = [(15, 17), (16, 16), (17, 16), (5, 130), (31, 33), (32, 1000), (16, 2200), (48, 49), (50, 20), (33, 270),
         (34, 608), (64, 65), (64, 400), (80, 96), (96, 96), (97, 97), (96, 130),
         (64, 1000), (21, 1089), (3, 5000), (32, 1025), (33, 2049), (65, 900)]  # thin, in pieces of 64 columns


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("shape", SMALL, ids=lambda s: f"{s[0]}x{s[1]}")
def test_orthogonalize_small_ones_alone_and_beside_a_large_one(dev, dt, shape):
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    rng = np.random.default_rng(shape[0] + shape[1])
    for s in {shape, shape[::-1]}:
        g = rng.standard_normal(s).astype(dt)
        alone = orthogonalize(D.from_numpy(g))
        check_ns(alone, g, dt, what="alone")
        assert bits_equal(alone.numpy(), orthogonalize(D.from_numpy(g)).numpy())
        # (how a grouped product's sums are split goes by the whole call: no bits to compare)
        check_ns(orthogonalize([D.from_numpy(g), D.from_numpy(g)])[1], g, dt, what="twice")
        big = rng.standard_normal((130, 140)).astype(dt)
        outs = orthogonalize([D.from_numpy(big), D.from_numpy(g)])
        check_ns(outs[0], big, dt, what="large")
        check_ns(outs[1], g, dt, what="beside")


@pytest.mark.parametrize("dt", [F32, F64])
def test_orthogonalize_more_small_ones_than_a_launch_holds(dev, dt):
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    rng = np.random.default_rng(0)
    gs = [rng.standard_normal(s).astype(dt) for s in [(40, 24), (3, 17, 5), (24, 40)] + [(12, 8)] * 70 + [(1, 1)]]
    for o, g in zip(orthogonalize([D.from_numpy(g) for g in gs]), gs):
        for at in np.ndindex(*g.shape[:-2]):
            check_ns(o.numpy()[at], g[at], dt)


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("steps", [1, 2, 5])
def test_orthogonalize_thin_ones(dev, dt, steps):
    """Wide and tall, stacked, more than a launch holds, by odd numbers of steps."""
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    rng = np.random.default_rng(0)
    gs = [rng.standard_normal(s).astype(dt) for s in [(24, 2000), (1900, 17), (3, 30, 1300), (1, 3000)] + [(2, 70)] * 62]
    outs = orthogonalize([D.from_numpy(g) for g in gs], steps)
    for o, g in zip(outs, gs):
        for at in np.ndindex(*g.shape[:-2]):
            check_ns(o.numpy()[at], g[at], dt, steps)
    again = orthogonalize([D.from_numpy(g) for g in gs], steps)
    assert all(bits_equal(a.numpy(), b.numpy()) for a, b in zip(outs, again))


@pytest.mark.parametrize("dt", [F32, F64])
def test_orthogonalize_many_at_once(dev, dt):
    """Wide, tall, square and stacked matrices and more of them than a launch holds: each
    as by itself."""
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    rng = np.random.default_rng(0)
    gs = [rng.standard_normal(s).astype(dt) for s in
          [(40, 24), (24, 40), (3, 17, 5), (2, 2, 12, 30), (0, 4), (0, 3, 4)] + [(12, 8)] * 70]
    outs = orthogonalize([D.from_numpy(g) for g in gs])
    for i, (o, g) in enumerate(zip(outs, gs)):
        assert o.shape == g.shape
        for at in np.ndindex(*g.shape[:-2]):
            if g[at].size:
                check_ns(o.numpy()[at], g[at], dt, what=i)
    assert orthogonalize([]) == []


@pytest.mark.parametrize("dt", [F32, F64])
def test_orthogonalize_on_wide_tiles(dev, dt):
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    rng = np.random.default_rng(0)
    gs = [rng.standard_normal(s).astype(dt) for s in [(516, 1028), (1030, 515)] + [(512, 640)] * 3]
    for o, g in zip(orthogonalize([D.from_numpy(g) for g in gs]), gs):
        check_ns(o, g, dt)


def test_orthogonalize_coefficients_steps_and_scale(dev):
    from dtmi import device as D
    from dtmi.optim import orthogonalize
    g = np.random.default_rng(1).standard_normal((20, 30))
    for steps, coef in ((1, COEF), (2, (1.5, -0.5, 0.0)), (12, (1.875, -1.25, 0.375))):
        check_ns(orthogonalize(D.from_numpy(g), steps, coef), g, F64, steps, coef, what=(steps, coef))
    # convergent coefficients: orthonormal rows
    o = orthogonalize(D.from_numpy(g), 30, (1.875, -1.25, 0.375)).numpy()
    assert np.abs(o @ o.T - np.eye(20)).max() <= 1e-12
    for scale in (1e-25, 1e25):   # float32 squares of these leave its range
        g32 = (g * scale).astype(F32)
        check_ns(orthogonalize(D.from_numpy(g32), eps=0.0), g32, F32, eps=0.0, what=scale)
    assert not orthogonalize(D.from_numpy(np.zeros((5, 7), F32))).numpy().any()
    assert np.isnan(orthogonalize(D.from_numpy(np.full((5, 7), np.nan, F32))).numpy()).all()
    from dtmi._lib import DtmiError
    for steps in (0, 65, -1):
        with pytest.raises(DtmiError, match="steps"):
            orthogonalize(D.from_numpy(g), steps)


def muon_ref(p, m, g, scale, lr, mu, nesterov, wd, dt):
    m = mu * m + scale * g.astype(F64)
    u = scale * g.astype(F64) + mu * m if nesterov else m
    o, grow = ns_ref(u, 5, COEF, 1e-7)
    k, n = p.shape
    rate = lr * math.sqrt(max(1.0, n / k))
    # u itself carries 3 roundings
    tol = (rate * (ns_bar(u, o, grow, 5, dt) + 8 * grow) * np.abs(o).max() + 4 * np.abs(p).max()) * U[dt]
    return (1 - lr * wd) * p - rate * o, m, tol


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("large", [None, (150, 101), (1700, 30)], ids=["small", "groups", "thin"])
def test_muon(dev, dt, nesterov, large):
    """Three steps, with a device-side gradient factor, a changed rate, a parameter
    without a gradient, a stack of matrices and a saved state."""
    from dtmi import device as D
    from dtmi.optim import Muon
    rng = np.random.default_rng(2)
    shapes = [(16, 48), (48, 16), (33, 33), (3, 20, 12), (7, 9)] + [large] * (large is not None)
    P = [(0.1 * rng.standard_normal(s)).astype(dt) for s in shapes]
    ps = [D.from_numpy(p) for p in P]
    opt = Muon(ps, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1)
    ref = [p.astype(F64) for p in P]
    mom = [np.zeros(s) for s in shapes]
    assert opt.state_bytes() == sum(p.nbytes for p in P)
    for step, (lr, scale) in enumerate(((0.02, 1.0), (0.02, 0.37), (0.005, 2.5))):
        G = [rng.standard_normal(s).astype(dt) for s in shapes]
        skip = 4 if step == 1 else None
        opt.lr = lr
        f = scale if step != 1 else D.from_numpy(np.array([scale]))
        opt.step([None if i == skip else D.from_numpy(g) for i, g in enumerate(G)], grad_scale=f)
        for i in range(len(P)):
            if i == skip:
                continue
            s = np.float64(dt(scale))
            got, gm = ps[i].numpy(), opt.m[i].numpy()
            for at in np.ndindex(*shapes[i][:-2]):
                want, m, tol = muon_ref(ref[i][at], mom[i][at], G[i][at], s, lr, 0.9, nesterov, 0.1, dt)
                assert np.abs(got[at] - want).max() <= tol * (step + 1) * 4, (step, i)
                assert np.abs(gm[at] - m).max() <= 8 * (step + 1) * U[dt] * np.abs(m).max(), (step, i)
                mom[i][at] = gm[at]
                ref[i][at] = got[at]
        if step == 0:
            state = opt.state_dict()
            other = Muon(ps)
            other.load_state_dict(state)
            assert all(bits_equal(a.numpy(), b.numpy()) for a, b in zip(opt.m, other.m))


def test_muon_keeps_to_its_matrices(dev):
    """Matrices back to back in one buffer: the neighbours of one that has no gradient, and
    what lies before and behind, stay as they are."""
    from dtmi import device as D
    from dtmi.optim import Muon
    flat = D.full((13 * 17 * 3 + 8,), 5.0, F32)
    ps = [flat[4 + 221 * i:4 + 221 * (i + 1)].reshape(13, 17) for i in range(3)]
    opt = Muon(ps, lr=0.1)
    rng = np.random.default_rng(0)
    opt.step([D.from_numpy(rng.standard_normal((13, 17)).astype(F32)), None,
              D.from_numpy(rng.standard_normal((13, 17)).astype(F32))])
    f = flat.numpy()
    assert (f[:4] == 5).all() and (f[-4:] == 5).all() and (f[4 + 221:4 + 442] == 5).all()
    assert (f[4:4 + 221] != 5).all() and (f[4 + 442:-4] != 5).all()
    with pytest.raises(ValueError, match="gradients for"):
        opt.step([None])
    g = D.from_numpy(rng.standard_normal((13, 17)).astype(F32))
    for scale in (D.full((1,), 1.0, F32), D.full((2,), 1.0, F64)):
        with pytest.raises(ValueError, match="float64"):
            opt.step([g, None, None], grad_scale=scale)


def test_a_training_step_of_a_model_with_experts(dev):
    """The operators together: tokens gathered by expert, two products with a GELU
    between them, the loss without logits, and an update of the stacked weights."""
    from dtmi import autograd as A, device as D
    from dtmi.optim import Muon
    rng = np.random.default_rng(7)
    T, C, H, E, V = 50, 24, 40, 3, 77
    x, t = rng.standard_normal((T, C)), rng.integers(0, V, T)
    t[:5] = -1
    w1, w2, wv = (rng.standard_normal(s) * 0.2 for s in ((E, C, H), (E, H, C), (C, V)))
    b1 = 0.1 * rng.standard_normal((E, H))
    expert = rng.integers(0, E, T)
    order = np.argsort(expert, kind="stable")
    sizes = np.bincount(expert, minlength=E)
    L = [A.Tensor(v, requires_grad=True) for v in (x, w1, b1, w2, wv)]
    h = A.expert_linear(A.embedding(L[0], order), L[1], sizes, L[2]).gelu()
    y = A.embedding(A.expert_linear(h, L[3], sizes), np.argsort(order))
    loss = A.linear_cross_entropy(y + L[0], L[4], t, ignore=-1)
    loss.backward()
    R = [t64(v) for v in (x, w1, b1, w2, wv)]
    xe = R[0][torch.tensor(order)]
    e = torch.tensor(expert[order])
    hr = torch.nn.functional.gelu(torch.bmm(xe[:, None], R[1][e].contiguous())[:, 0] + R[2][e], approximate="tanh")
    yr = torch.bmm(hr[:, None], R[3][e].contiguous())[:, 0][torch.tensor(np.argsort(order))] + R[0]
    lr = torch.nn.functional.cross_entropy(yr @ R[4], torch.tensor(t), ignore_index=-1)
    want = torch.autograd.grad(lr, R)
    close(loss, lr, F64, 512, "loss")
    for got, r, name in zip(L, want, ("x", "w1", "b1", "w2", "wv")):
        close(got.grad, r, F64, 2048, name)
    before = [p.numpy() for p in (L[1], L[3])]
    opt = Muon([L[1].data, L[3].data], lr=0.02)
    opt.step([L[1].grad, L[3].grad])
    for p, b, g in zip((L[1], L[3]), before, (L[1].grad, L[3].grad)):
        got, g = p.numpy(), g.numpy()
        for i in range(E):
            w, _, tol = muon_ref(b[i], 0 * b[i], g[i], 1.0, 0.02, 0.95, True, 0.0, F64)
            assert np.abs(got[i] - w).max() <= tol
