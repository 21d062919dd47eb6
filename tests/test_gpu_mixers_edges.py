"""Sequence mixers on the GPU at the edges of their ranges, against their
definitions in float64: memories of one key, scores and decays that leave the
types' range on the way to a finite value, operands without elements, states
moved on between the passes. Bars count roundings of half a step u as in
test_gpu_mixers; a bar that differs has its own count beside it."""
import numpy as np
import pytest
import torch

from helpers import bits_equal
from test_gpu_mixers import F32, F64, U, _mods, bthd, close, conv_ref, cross_ref, scan_ref, t64

pytestmark = pytest.mark.gpu


def cross_grads(q, k, v, g, lengths=None, scale=None, strided=False, kept=True):
    """o, dq, dk, dv of cross_attention, dS kept for the dQ pass or formed twice."""
    from dtmi import kernels as K
    A, _ = _mods()
    L = [A.Tensor(bthd(x, strided), requires_grad=True) for x in (q, k, v)]
    before = K.attn_set_ds_limit(0 if not kept else 1 << 32)
    try:
        o = A.cross_attention(*L, lengths=lengths, scale=scale)
        o.backward(bthd(g, strided))
    finally:
        K.attn_set_ds_limit(before)
    return [o.numpy()] + [x.grad.numpy() for x in L]


ONE_KEY = [  # B, H, Hk, Tq, Tk, D, lengths
    (1, 1, 1, 1, 1, 64, None),
    (2, 4, 2, 9, 1, 32, None),
    (2, 3, 3, 70, 1, 72, None),
    (1, 2, 1, 40, 1, 128, None),
    (3, 2, 2, 33, 40, 64, [1, 1, 1]),
    (2, 4, 1, 5, 300, 96, [1, 1]),
    (4, 2, 1, 50, 700, 40, [1, 700, 0, 1]),
]


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", ONE_KEY, ids=lambda c: "-".join(str(v) for v in c[:6]))
def test_cross_attention_of_one_key(dev, dt, case, kept):
    """With one key the probability is 1 whatever the score: o is its value, and
    dQ and dK are 0, not what rounding leaves of a difference. Each sequence is
    judged by itself."""
    B, H, Hk, Tq, Tk, Dh, lengths = case
    rng = np.random.default_rng(Tq + Tk + Dh)
    q, g = (rng.standard_normal((B, H, Tq, Dh)).astype(dt) for _ in range(2))
    k, v = (rng.standard_normal((B, Hk, Tk, Dh)).astype(dt) for _ in range(2))
    o, dq, dk, dv = cross_grads(q, k, v, g, lengths, kept=kept)
    R = [t64(x) for x in (q, k, v)]
    ro = cross_ref(*R, lengths, Dh ** -.5)
    want = torch.autograd.grad(ro, R, t64(g, False))
    for i in range(B):
        n = Tk if lengths is None else lengths[i]
        close(o[i], ro[i], dt, 4 if n == 1 else 512, f"o {i}")
        if n > 1:
            for got, w, name in zip((dq, dk, dv), want, ("dq", "dk", "dv")):
                close(got[i], w[i], dt, 512, f"{name} {i}")
            continue
        assert not dq[i].any() and not dk[i].any(), i
        # a sum over the group's rows, each term with its probability's roundings
        close(dv[i], want[2][i], dt, H // Hk * Tq + 8, f"dv {i}")


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", [(1, 1, 1, 3, 40, 8), (1, 2, 2, 40, 300, 16), (1, 2, 1, 130, 20, 64), (2, 2, 2, 1, 900, 32)],
                         ids=lambda c: "-".join(str(v) for v in c))
def test_cross_attention_of_scores_whose_rounding_is_large(dev, dt, case):
    """Scores of 1e11 (float64: 1e25), finite: a step of them is far above 1, and
    the largest takes all the weight. o is its value to the bit."""
    B, H, Hk, Tq, Tk, Dh = case
    rng = np.random.default_rng(Tk)
    size = 1e5 if dt is F32 else 1e12
    q, g = (rng.standard_normal((B, H, Tq, Dh)).astype(dt) for _ in range(2))
    k, v = (rng.standard_normal((B, Hk, Tk, Dh)).astype(dt) for _ in range(2))
    q, k = q * dt(size), k * dt(size)
    s = np.repeat(k, H // Hk, 1).astype(F64) @ np.swapaxes(q, 2, 3).astype(F64)  # [B, H, Tk, Tq]
    top = np.sort(s, 2)
    # the winner is clear of every score's rounding (D of them, and one of the scaling)
    assert (top[:, :, -1] - top[:, :, -2] > 4 * (Dh + 2) * U[dt] * np.abs(s).max()).all()
    best = s.argmax(2)  # [B, H, Tq]
    want = np.take_along_axis(np.repeat(v, H // Hk, 1), best[..., None], 2)
    o, dq, dk, dv = cross_grads(q, k, v, g, scale=1.0)
    assert bits_equal(o, want)
    assert np.isfinite(dq).all() and np.isfinite(dk).all()
    sums = np.zeros((B, H, Tk, Dh))
    for b in range(B):
        for h in range(H):
            np.add.at(sums[b, h], best[b, h], g[b, h].astype(F64))
    close(dv, sums.reshape(B, Hk, H // Hk, Tk, Dh).sum(2), dt, H // Hk * Tq + 8, "dv")


@pytest.mark.parametrize("kept", [True, False])
@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", [(1, 1, 1, 3, 40, 1), (1, 2, 2, 70, 300, 20), (2, 4, 2, 40, 33, 64), (1, 2, 1, 5, 2000, 72),
                                  (1, 12, 12, 200, 160, 40)],
                         ids=lambda c: "-".join(str(v) for v in c))
def test_rows_without_a_finite_score_pass_no_gradient(dev, dt, case, kept):
    """Scores of -inf from infinite keys or from infinite queries: such a row is 0,
    its dq is 0 and it adds nothing to dk and dv."""
    B, H, Hk, Tq, Tk, Dh = case
    rng = np.random.default_rng(Tk)
    q, k = (np.abs(rng.standard_normal(s)).astype(dt) + dt(.1) for s in ((B, H, Tq, Dh), (B, Hk, Tk, Dh)))
    v, g = (rng.standard_normal(s).astype(dt) for s in ((B, Hk, Tk, Dh), (B, H, Tq, Dh)))
    beyond = v.copy()
    beyond[..., 0, 0] = np.inf
    for values in (v, beyond):
        for got in cross_grads(q, np.full_like(k, -np.inf), values, g, kept=kept):
            assert (got == 0).all()
    dead = (0, H - 1, Tq // 2)
    qi = q.copy()
    qi[dead] = -np.inf
    o, dq, dk, dv = cross_grads(qi, k, v, g, kept=kept)
    assert (o[dead] == 0).all() and (dq[dead] == 0).all()
    R, live = [t64(x) for x in (q, k, v)], np.ones((B, H, Tq, 1))
    live[dead] = 0
    ro = cross_ref(*R, None, Dh ** -.5) * torch.tensor(live)
    want = torch.autograd.grad(ro, R, t64(g, False))
    close(o, ro, dt, 512, "o")
    # dS sums to 0 along the keys, whose elements have a mean of 1.5 times their spread: of
    # dq's terms less than half is left
    for got, w, name, bar in zip((dq, dk, dv), want, ("dq", "dk", "dv"), (1024, 512, 512)):
        close(got, w, dt, bar, name)


def scan_all(v, dt, lengths=None, softplus=True, steps=False):
    """out, state and gradients of ssm_scan for arrays by name, and the reference's."""
    A, D = _mods()
    names = [n for n in ("u", "dt", "A", "B", "C", "D", "z", "bias", "h") if n in v]
    L = {n: A.Tensor(D.from_numpy(v[n].astype(dt)), requires_grad=True) for n in names}
    y, state = A.ssm_scan(*(L[n] for n in ("u", "dt", "A", "B", "C")), D=L.get("D"), z=L.get("z"), dt_bias=L.get("bias"),
                          state=L.get("h"), lengths=lengths, return_state=True, softplus=softplus)
    y.backward(D.from_numpy(v["g"].astype(dt)))
    # where A has no finite value the reference takes one whose decay is 0 all the same
    R = {n: t64(np.maximum(v[n].astype(dt).astype(F64), -1e30)) for n in names}
    B, T, C = v["u"].shape
    N = v["A"].shape[1]
    zero = {n: torch.zeros(s, dtype=torch.float64) for n, s in (("D", C), ("bias", C), ("h", (B, C, N)))}
    Bm, Cm = (R[n] if R[n].ndim == 4 else R[n][:, :, None] for n in "BC")
    ry, rs = scan_ref(R["u"], R["dt"], R["A"], Bm, Cm, R.get("D", zero["D"]), R.get("z"), R.get("bias", zero["bias"]),
                      R.get("h", zero["h"]), lengths, softplus)
    want = torch.autograd.grad(ry, [R[n] for n in names], t64(v["g"].astype(dt), False))
    return y, state, {n: L[n].grad for n in names}, ry, rs, dict(zip(names, want))


@pytest.mark.parametrize("dt", [F32, F64])
def test_scan_growth_of_a_zero_state(dev, dt):
    """Steps of a negative size make states grow; a state of 0, and a gradient of
    0, stay 0 over any growth, also where a segment's decay alone leaves the type's range."""
    rng = np.random.default_rng(6)
    B, T, C, N = 1, 300, 3, 4
    v = {n: rng.standard_normal((B, T, C)) for n in ("u", "g")}
    v.update(A=np.full((C, N), -1.0), B=rng.standard_normal((B, T, N)), C=rng.standard_normal((B, T, N)),
             D=rng.standard_normal(C), h=rng.standard_normal((B, C, N)), dt=.1 + rng.random((B, T, C)) * .1)
    v["u"][:, 40:200] = v["g"][:, 40:200] = 0
    v["dt"][:, 41:199] = -3 if dt is F32 else -60
    v["dt"][:, [40, 199]] = 20000  # exp(-20000) leaves nothing that exp(158 x 60) could bring back
    y, state, got, ry, rs, want = scan_all(v, dt, softplus=False)
    # decays of 0.1 and more: 10 steps' worth of 4 roundings, and the products around them, as in test_scan
    close(y, ry, dt, 256, "y")
    close(state, rs, dt, 256, "state")
    for n in got:
        close(got[n], want[n], dt, 512, "d" + n)


@pytest.mark.parametrize("dt,size,rate,n,bar", [
    (F32, 1e-30, 2.0, 48, 512),     # e^96 times 1e-30
    (F64, 1e-300, 48.0, 16, 4096),  # e^768 times 1e-300
])
def test_scan_growth_of_a_small_state(dev, dt, size, rate, n, bar):
    """A state whose product with a segment's growth is in range where the growth
    is not. The exponent's relative roundings count by its size: 96 and 768, two of
    them in one product over the segment, and as much again step by step."""
    A, D = _mods()
    T, C, N = 300, 2, 3
    rng = np.random.default_rng(7)
    h = (1 + rng.random((1, C, N))) * size
    step, u = np.full((1, T, C), .1), np.zeros((1, T, C))
    step[:, :n], step[:, n] = -rate, 800
    step[:, n + 1:] = .1 + rng.random((1, T - n - 1, C)) * .1
    u[:, n + 1:] = rng.standard_normal((1, T - n - 1, C))
    Bm, Cm = rng.standard_normal((2, 1, T, N)).astype(dt)
    a = [x.astype(dt) for x in (u, step, -np.ones((C, N)), Bm, Cm)]
    with A.no_grad():
        y, state = A.ssm_scan(*(A.Tensor(D.from_numpy(x)) for x in a), state=D.from_numpy(h.astype(dt)), return_state=True,
                              softplus=False)
    z = torch.zeros((), dtype=torch.float64)
    r = [t64(x, False) for x in a]
    ry, rs = scan_ref(r[0], r[1], r[2], r[3][:, :, None], r[4][:, :, None], z, None, z, t64(h.astype(dt), False), None, False)
    close(y.numpy()[:, :n], ry[:, :n], dt, bar, "y while it grows")
    close(y.numpy()[:, n:], ry[:, n:], dt, 256, "y after")
    close(state, rs, dt, 256, "state")


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("B,T,C,N,lengths", [(1, 19, 5, 4, None), (2, 40, 70, 16, [40, 13]), (1, 700, 33, 5, None),
                                             (3, 33, 20, 33, [0, 1, 33])],
                         ids=lambda v: str(v) if isinstance(v, int) else "")
def test_scan_of_states_that_are_forgotten_at_once(dev, dt, B, T, C, N, lengths):
    """A of -inf, as -exp(log rate) gives when it overflows (or a finite one that
    does in base 2): the decay is 0 at every position and 1 where there is none."""
    rng = np.random.default_rng(T)
    v = {n: rng.standard_normal((B, T, C)) for n in ("u", "g", "z")}
    v.update(A=-0.5 - rng.random((C, N)) * 8, B=rng.standard_normal((B, T, N)), C=rng.standard_normal((B, T, N)),
             D=rng.standard_normal(C), h=rng.standard_normal((B, C, N)), dt=rng.standard_normal((B, T, C)) * .5)
    v["A"][rng.random((C, N)) < .3] = -np.inf
    v["A"][0, 0], v["A"][-1, -1] = -np.inf, -.9 * float(np.finfo(dt).max)
    y, state, got, ry, rs, want = scan_all(v, dt, lengths)
    close(y, ry, dt, 256, "y")
    close(state, rs, dt, 256, "state")
    for n in got:
        close(got[n], want[n], dt, 512, "d" + n)


def leave_sevens():
    """Sevens in the memory that the next arrays of up to 512 bytes are made of."""
    _, D = _mods()
    held = [D.full((n,), 7.0, F32) for n in (64, 128) for _ in range(64)]
    del held


def test_scan_without_channels_has_zero_map_gradients(dev):
    A, D = _mods()
    for G in (1, 2):
        L = [A.Tensor(D.full(s, 1.0, F32), requires_grad=True)
             for s in ((2, 3, 0), (2, 3, 0), (0, 5), (2, 3, G, 5), (2, 3, G, 5))]
        y = A.ssm_scan(*L)
        leave_sevens()
        y.backward(D.full(y.shape, 1.0, F32))
        for x in L:
            assert x.grad.shape == x.shape and (x.grad.numpy() == 0).all()


def test_cross_attention_without_heads_has_zero_memory_gradients(dev):
    A, D = _mods()
    L = [A.Tensor(D.full(s, 1.0, F32), requires_grad=True) for s in ((2, 0, 3, 8), (2, 2, 4, 8), (2, 2, 4, 8))]
    o = A.cross_attention(*L)
    leave_sevens()
    o.backward(D.full(o.shape, 1.0, F32))
    for x in L:
        assert x.grad.shape == x.shape and (x.grad.numpy() == 0).all()


@pytest.mark.parametrize("grad", [False, True])
def test_conv_gradient_after_its_state_moved_on(dev, grad):
    """The state handed to causal_conv may be moved on in place before backward."""
    A, D = _mods()
    rng = np.random.default_rng(9)
    B, T, C, K = 2, 6, 20, 4
    x, g = rng.standard_normal((2, B, T, C))
    w, st = rng.standard_normal((K, C)), rng.standard_normal((B, K - 1, C))
    X, W = (A.Tensor(D.from_numpy(a), requires_grad=True) for a in (x, w))
    state = D.from_numpy(st)
    y = A.causal_conv(X, W, state=A.Tensor(state, requires_grad=True) if grad else state)
    with A.no_grad():
        A.causal_conv_step(A.Tensor(D.from_numpy(x[:, 0])), W, None, state)
    y.backward(D.from_numpy(g))
    rx, rw = t64(x), t64(w)
    ry, _ = conv_ref(rx, rw, torch.zeros(C, dtype=torch.float64), t64(st, False), None, True)
    want = torch.autograd.grad(ry, (rx, rw), t64(g, False))
    close(y, ry, F64, K + 16, "y")
    close(X.grad, want[0], F64, 2 * K + 32, "dx")
    close(W.grad, want[1], F64, 2 * K + 160, "dw")


# ------------------------------------------------ configurations without a fault
JOIN = [  # more than 2048 rows of a split loop, B, H, Hk, Tq, Tk, D, lengths
    (2, 4, 2, 300, 1500, 40, None),
    (1, 12, 12, 200, 1500, 128, None),
    (2, 2, 1, 520, 700, 20, None),
    (1, 3, 3, 700, 900, 90, None),
    (5, 2, 1, 210, 1500, 72, [1500, 0, 97, 1024, 1025]),
    (4, 4, 2, 140, 800, 128, [1, 800, 65, 0]),
    (3, 2, 2, 350, 600, 48, [33, 600, 577]),
]


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", JOIN, ids=lambda c: "-".join(str(v) for v in c[:6]))
def test_cross_attention_joins_many_rows(dev, dt, case):
    B, H, Hk, Tq, Tk, Dh, lengths = case
    rng = np.random.default_rng(Tq + Dh)
    q, g = (rng.standard_normal((B, H, Tq, Dh)).astype(dt) for _ in range(2))
    k, v = (rng.standard_normal((B, Hk, Tk, Dh)).astype(dt) for _ in range(2))
    got = cross_grads(q, k, v, g, lengths, strided=Tq % 4 == 0)
    R = [t64(x) for x in (q, k, v)]
    ro = cross_ref(*R, lengths, Dh ** -.5)
    for i in range(B):  # each sequence by itself
        close(got[0][i], ro[i], dt, 512, f"o {i}")
    for x, w, name in zip(got[1:], torch.autograd.grad(ro, R, t64(g, False)), ("dq", "dk", "dv")):
        close(x, w, dt, 512, name)


@pytest.mark.parametrize("dt", [F32, F64])
def test_step_sizes_keep_their_relative_accuracy(dev, dt):
    """One position, one state, operands of 1: the state is softplus(dt) and the
    gradient of dt its sigmoid, each judged by itself from 1e-35 to 80. float32
    takes exp(x) as a power of two whose exponent carries two roundings of its size,
    2 |x| u of the value; beside that exponential, reciprocal, series and sums: 16."""
    A, D = _mods()
    x = np.concatenate([np.linspace(-80, 80, 3201), np.linspace(-9, -3, 801), [0.0]]).astype(dt)
    C = len(x)
    one = lambda *s: A.Tensor(D.full(s, 1.0, dt), requires_grad=True)  # noqa: E731
    X = A.Tensor(D.from_numpy(x[None, None]), requires_grad=True)
    y, state = A.ssm_scan(one(1, 1, C), X, A.Tensor(D.full((C, 1), -1.0, dt)), one(1, 1, 1), one(1, 1, 1), return_state=True)
    y.backward(D.full((1, 1, C), 1.0, dt))
    x = x.astype(F64)
    bar = (16 + (2 * np.abs(x) if dt is F32 else 0)) * U[dt]
    for got, want, what in ((state, np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x))), "softplus"),
                            (X.grad, 1 / (1 + np.exp(-x)), "sigmoid")):
        off = np.abs(got.numpy().reshape(-1).astype(F64) - want) / want / bar
        assert off.max() <= 1, (what, x[off.argmax()], off.max())


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("B,T,C,N,lengths", [(1, 300, 70, 16, None), (2, 260, 40, 4, [260, 131]), (1, 200, 24, 40, None),
                                             (100, 80, 130, 4, None), (130, 70, 130, 7, None),  # more blocks than CUs, cut
                                             (130, 70, 65, 13, None), (140, 70, 20, 20, None)],   # in one piece
                         ids=lambda v: str(v) if isinstance(v, int) else "")
def test_scan_of_slow_decays(dev, dt, B, T, C, N, lengths):
    """Rates of 1..N and steps of 1e-3 to 1e-1, as such layers start with: a
    segment leaves most of the state that enters it. A value carries 4 roundings a
    step over up to T steps, its gradients those of both ways: 4 T and 8 T, and 512."""
    rng = np.random.default_rng(T)
    v = {n: rng.standard_normal((B, T, C)) for n in ("u", "g", "z")}
    size = np.exp(rng.random(C) * np.log(100) + np.log(1e-3))
    v.update(A=-np.broadcast_to(np.arange(1, N + 1), (C, N)) * np.exp(.1 * rng.standard_normal((C, N))),
             B=rng.standard_normal((B, T, N)), C=rng.standard_normal((B, T, N)), D=1 + .1 * rng.standard_normal(C),
             bias=size + np.log(-np.expm1(-size)), h=rng.standard_normal((B, C, N)), dt=rng.standard_normal((B, T, C)) * .5)
    y, state, got, ry, rs, want = scan_all(v, dt, lengths)
    close(y, ry, dt, 4 * T, "y")
    close(state, rs, dt, 4 * T, "state")
    for n in got:
        close(got[n], want[n], dt, 8 * T + 512, "d" + n)


@pytest.mark.parametrize("dt", [F32, F64])
def test_steps_take_views(dev, dt):
    """Single positions out of fused projections: the bits of contiguous operands."""
    A, D = _mods()
    rng = np.random.default_rng(3)
    B, C, N, G, K = 3, 36, 8, 2, 4

    def fused(a):
        """a [B, ...] as the second of two arrays that one projection leaves side by side."""
        both = np.full((B, 2) + a.shape[1:], np.nan, dt)
        both[:, 1] = a
        return A.Tensor(D.from_numpy(both).transpose(1, 0, *range(2, a.ndim + 1))[1])

    def whole(a):
        return A.Tensor(D.from_numpy(a))
    x, step, z = rng.standard_normal((3, B, C)).astype(dt)
    Bm, Cm = rng.standard_normal((2, B, G, N)).astype(dt)
    w, b, Am, Dm, bias = (whole(rng.standard_normal(s).astype(dt)) for s in ((K, C), C, (C, N), C, C))
    cs, hs = rng.standard_normal((B, K - 1, C)).astype(dt), rng.standard_normal((B, C, N)).astype(dt)
    out = []
    for of in (whole, fused):
        c, h = D.from_numpy(cs), D.from_numpy(hs)
        y = A.causal_conv_step(of(x), w, b, c)
        s = A.ssm_scan_step(of(x), of(step), Am, of(Bm), of(Cm), Dm, of(z), bias, h)
        out.append([t.numpy() for t in (y, s, c, h)])
    for a, b_ in zip(*out):
        assert np.isfinite(a).all() and bits_equal(a, b_)


@pytest.mark.parametrize("D_", [64, 45])
def test_cross_attention_results_in_views(dev, D_):
    """Output and gradients written into parts of larger arrays, nothing beside them."""
    from dtmi import kernels as K
    _, D = _mods()
    rng = np.random.default_rng(D_)
    B, H, Hk, Tq, Tk = 2, 4, 2, 37, 50
    q, g = (D.from_numpy(rng.standard_normal((B, H, Tq, D_)).astype(F32)) for _ in range(2))
    k, v = (D.from_numpy(rng.standard_normal((B, Hk, Tk, D_)).astype(F32)) for _ in range(2))

    def room(T, heads):
        """Three arrays [B, T, 3, heads, D] in one of sevens; the view is the middle one."""
        a = D.full((B, T, 3, heads, D_), 7.0, F32)
        return a, a.transpose(2, 0, 3, 1, 4)[1]
    o, m, l = K.xattn_fwd(q, k, v)
    grads = K.xattn_bwd(q, k, v, o, g, m, l)
    rooms = [room(Tq, H), room(Tq, H), room(Tk, Hk), room(Tk, Hk)]
    o2, m2, l2 = K.xattn_fwd(q, k, v, out=rooms[0][1])
    K.xattn_bwd(q, k, v, o2, g, m2, l2, dq=rooms[1][1], dk=rooms[2][1], dv=rooms[3][1])
    for want, (whole, view) in zip((o,) + tuple(grads), rooms):
        assert bits_equal(view.numpy(), want.numpy())
        rest = whole.numpy()
        assert (rest[:, :, [0, 2]] == 7).all()
