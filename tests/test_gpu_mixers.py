"""Sequence mixers on the GPU against their definitions in float64: the short
causal convolution, the selective scan and cross attention, forward and every
gradient, whole sequences and single positions.

Bars are normwise (max |error| / max |value|) and count roundings of half a step
u (2^-24, 2^-53) on the way to a value: a convolution's K products, bias,
sigmoid and gate (K + 16); sums over positions add pairwise parts of at most 64
positions in a row and their partial sums (64 + 64 more). A scan's state passes
through 4 roundings a step, each weighed by the decay since: with the decays
used here (rates of 0.5 and more times steps of 0.3 and more) at most 1 / (1 -
exp(-0.15)) = 7 steps' worth, times the products around it, and the gradients
go through it twice: 256. A softmax's scores of up to 2^4 in base 2 carry D + 2
roundings of their size, which the exponential makes relative ones: 2^4 (D + 2)
in the worst case, of which the sum's average leaves a small part: 512."""
import numpy as np
import pytest
import torch

from helpers import bits_equal

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
F32, F64 = np.float32, np.float64


def _mods():
    from dtmi import autograd as A, device as D
    return A, D


def close(got, want, dt, roundings, what):
    got = np.asarray(got.numpy() if hasattr(got, "numpy") else got, np.float64)
    want = want.detach().numpy() if isinstance(want, torch.Tensor) else np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.size:
        return
    assert np.isfinite(got).all(), what
    err, top = np.abs(got - want).max(), np.abs(want).max()
    assert err <= roundings * U[dt] * max(top, 1e-300), (what, err / max(top, 1e-300) / U[dt])


def put(a, fused, seed=0):
    """a [B, T, ...] on the device, whole or as one of two interleaved arrays."""
    _, D = _mods()
    if not fused:
        return D.from_numpy(a)
    both = np.full(a.shape[:2] + (2,) + a.shape[2:], np.nan, a.dtype)
    both[:, :, 1] = a
    order = (2, 0, 1) + tuple(range(3, a.ndim + 1))
    return D.from_numpy(both).transpose(*order)[1]


def hide(a, lengths, axis=1):
    """NaN where a padded batch holds nothing."""
    if lengths is None:
        return a
    a = a.copy()
    for i, n in enumerate(lengths):
        ix = [slice(None)] * a.ndim
        ix[0], ix[axis] = i, slice(n, None)
        a[tuple(ix)] = np.nan
    return a


def t64(a, grad=True):
    return torch.tensor(np.asarray(a, np.float64), requires_grad=grad)


# ------------------------------------------------------------- convolution
def conv_ref(x, w, b, state, lengths, silu):
    B, T, C = x.shape
    K = w.shape[0]
    full = torch.cat([state, x], 1)
    pre = sum(w[k] * full[:, k:k + T] for k in range(K)) + b
    y = pre * torch.sigmoid(pre) if silu else pre
    n = torch.tensor([T] * B if lengths is None else lengths)
    y = torch.where((torch.arange(T)[None] < n[:, None])[..., None], y, torch.zeros((), dtype=y.dtype))
    return y, torch.stack([full[i, n[i]:n[i] + K - 1] for i in range(B)])


CONV = [  # B, T, C, K, lengths, fused, silu, bias, state
    (1, 1, 1, 4, None, False, True, True, False),
    (2, 3, 5, 4, None, False, True, False, True),
    (3, 17, 64, 1, [17, 0, 4], False, True, True, False),
    (4, 33, 36, 2, [33, 1, 0, 32], True, True, True, True),
    (2, 130, 96, 3, [130, 65], False, False, True, True),
    (1, 700, 260, 4, None, True, True, True, False),
    (3, 64, 37, 5, [2, 64, 63], True, True, True, True),
    (2, 9, 128, 8, [9, 3], False, True, True, True),
    (2, 40, 12, 7, None, False, True, False, False),
    (2, 40, 12, 6, None, False, False, False, False),
]


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", CONV, ids=lambda c: "-".join(str(v) for v in c[:4]))
def test_conv(dev, dt, case):
    A, D = _mods()
    B, T, C, K, lengths, fused, silu, bias, with_state = case
    rng = np.random.default_rng(T * 31 + C)
    x, g = (rng.standard_normal((B, T, C)).astype(dt) for _ in range(2))
    w, b = (rng.standard_normal((K, C)) * K ** -.5).astype(dt), rng.standard_normal(C).astype(dt)
    st = rng.standard_normal((B, K - 1, C)).astype(dt)
    X, W = (A.Tensor(v, requires_grad=True) for v in (put(hide(x, lengths), fused), D.from_numpy(w)))
    Bt = A.Tensor(D.from_numpy(b), requires_grad=True) if bias else None
    S = A.Tensor(D.from_numpy(st), requires_grad=True) if with_state else None
    y, new = A.causal_conv(X, W, Bt, silu=silu, state=S, lengths=lengths, return_state=True)
    y.backward(put(hide(g, lengths), fused))
    rx, rw = t64(x), t64(w)
    rb, rs = t64(b if bias else 0 * b), t64(st if with_state else 0 * st)
    ry, rnew = conv_ref(rx, rw, rb, rs, lengths, silu)
    grads = torch.autograd.grad(ry, [rx, rw, rb, rs], t64(g, False))
    close(y, ry, dt, K + 16, "y")
    close(new, rnew, dt, 0, "state")
    close(X.grad, grads[0], dt, 2 * K + 32, "dx")
    close(W.grad, grads[1], dt, 2 * K + 160, "dw")
    if bias:
        close(Bt.grad, grads[2], dt, 2 * K + 160, "db")
    if with_state:
        close(S.grad, grads[3], dt, 2 * K + 32, "dstate")


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("B,C,K", [(1, 1, 2), (3, 130, 4), (5, 64, 1), (2, 37, 8)])
def test_conv_in_pieces(dev, dt, B, C, K):
    """A sequence in two calls and then position by position, the state handed
    on, gives the whole sequence's bits."""
    A, D = _mods()
    rng = np.random.default_rng(C)
    T = 12
    x = rng.standard_normal((B, T, C)).astype(dt)
    w, b = A.Tensor(D.from_numpy(rng.standard_normal((K, C)).astype(dt))), A.Tensor(D.zeros((C,), dt))
    with A.no_grad():
        whole, end = A.causal_conv(A.Tensor(D.from_numpy(x)), w, b, return_state=True)
        y1, s = A.causal_conv(A.Tensor(D.from_numpy(x[:, :2])), w, b, return_state=True)
        y2, s = A.causal_conv(A.Tensor(D.from_numpy(x[:, 2:9])), w, b, state=s, return_state=True)
        steps = [A.causal_conv_step(A.Tensor(D.from_numpy(x[:, t])), w, b, s).numpy() for t in range(9, T)]
    got = np.concatenate([y1.numpy(), y2.numpy(), np.stack(steps, 1)], 1)
    assert bits_equal(got, whole.numpy())
    assert bits_equal(s.numpy(), end.numpy())


# -------------------------------------------------------------------- scan
def scan_ref(u, dt, Am, Bm, Cm, D, z, bias, h, lengths, softplus):
    B, T, C = u.shape
    G = Bm.shape[2]
    raw = dt + bias
    d = torch.nn.functional.softplus(raw, threshold=500) if softplus else raw
    n = torch.tensor([T] * B if lengths is None else lengths)
    Bm, Cm = (m.repeat_interleave(C // G, 2) for m in (Bm, Cm))
    out = []
    for t in range(T):
        on = (t < n)[:, None]
        new = torch.exp(d[:, t, :, None] * Am) * h + (d[:, t] * u[:, t])[..., None] * Bm[:, t]
        h = torch.where(on[..., None], new, h)
        y = (h * Cm[:, t]).sum(-1) + D * u[:, t]
        if z is not None:
            y = y * torch.nn.functional.silu(z[:, t])
        out.append(torch.where(on, y, torch.zeros((), dtype=y.dtype)))
    return torch.stack(out, 1), h


SCAN = [  # B, T, C, N, G, lengths, fused, has (D, z, bias, state, softplus)
    (1, 1, 1, 1, 1, None, False, (1, 1, 1, 0, 1)),
    (2, 2, 3, 4, 1, None, False, (0, 0, 0, 0, 0)),
    (3, 15, 64, 16, 1, [15, 0, 7], False, (1, 1, 1, 1, 1)),
    (2, 16, 65, 5, 1, None, True, (1, 0, 1, 1, 1)),
    (4, 17, 70, 8, 2, [17, 16, 1, 0], True, (1, 1, 1, 1, 1)),
    (1, 100, 130, 13, 1, None, False, (1, 1, 0, 0, 1)),
    (2, 33, 40, 17, 4, [33, 20], False, (0, 1, 1, 1, 0)),
    (2, 40, 66, 32, 1, [24, 40], True, (1, 1, 1, 1, 1)),
    (1, 37, 96, 33, 3, None, False, (1, 0, 0, 1, 1)),
    (2, 50, 20, 64, 1, [50, 31], False, (1, 1, 1, 1, 1)),
    (1, 700, 66, 16, 1, None, True, (1, 1, 1, 1, 1)),     # segments of the sequence
    (3, 410, 16, 3, 1, [0, 410, 130], False, (1, 1, 1, 1, 1)),  # with ends inside and before them
    (2, 300, 70, 48, 2, [300, 129], True, (1, 1, 1, 1, 1)),
    (1, 230, 200, 8, 1, None, False, (1, 1, 1, 0, 1)),
    (300, 20, 64, 2, 1, None, False, (1, 1, 1, 1, 1)),    # enough blocks for one segment
    (257, 19, 8, 40, 1, None, False, (1, 1, 1, 1, 1)),    # of sixteen waves
]


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", SCAN, ids=lambda c: "-".join(str(v) for v in c[:5]))
def test_scan(dev, dt, case):
    A, D = _mods()
    B, T, C, N, G, lengths, fused, (hasD, hasz, hasb, hash_, softplus) = case
    rng = np.random.default_rng(T * 7 + N)

    def normal(*s, std=1.0):
        return (rng.standard_normal(s) * std).astype(dt)
    v = dict(u=normal(B, T, C), z=normal(B, T, C), g=normal(B, T, C), B=normal(B, T, G, N), C=normal(B, T, G, N),
             A=(-0.5 - rng.random((C, N)) * 8).astype(dt), D=normal(C), bias=normal(C, std=.2), h=normal(B, C, N))
    v["dt"] = normal(B, T, C, std=.5) if softplus else (0.3 + rng.random((B, T, C))).astype(dt)
    if not softplus:
        v["bias"] = (rng.random(C) * .2).astype(dt)
    along = ("u", "dt", "z", "B", "C", "g")
    dev_ = {n: put(hide(a, lengths), fused) if n in along else D.from_numpy(a) for n, a in v.items()}
    names = ["u", "dt", "A", "B", "C"] + [n for n, on in zip(("D", "z", "bias", "h"), (hasD, hasz, hasb, hash_)) if on]
    L = {n: A.Tensor(dev_[n], requires_grad=True) for n in names}
    y, state = A.ssm_scan(*(L[n] for n in ("u", "dt", "A", "B", "C")), D=L.get("D"), z=L.get("z"), dt_bias=L.get("bias"),
                          state=L.get("h"), lengths=lengths, return_state=True, softplus=bool(softplus))
    y.backward(dev_["g"])
    R = {n: t64(v[n]) for n in names}
    zero = {n: torch.zeros(v[n].shape, dtype=torch.float64) for n in ("D", "bias", "h")}
    ry, rstate = scan_ref(R["u"], R["dt"], R["A"], R["B"], R["C"], R.get("D", zero["D"]), R.get("z"),
                          R.get("bias", zero["bias"]), R.get("h", zero["h"]), lengths, softplus)
    grads = torch.autograd.grad(ry, [R[n] for n in names], t64(v["g"], False))
    close(y, ry, dt, 256, "y")
    close(state, rstate, dt, 256, "state")
    for n, want in zip(names, grads):
        close(L[n].grad, want, dt, 512 if n in ("A", "D", "bias", "B", "C") else 256, "d" + n)
    with A.no_grad():  # without what the backward needs, the same bits
        y2 = A.ssm_scan(*(L[n] for n in ("u", "dt", "A", "B", "C")), D=L.get("D"), z=L.get("z"), dt_bias=L.get("bias"),
                        state=L.get("h"), lengths=lengths, softplus=bool(softplus))
    assert bits_equal(y2.numpy(), y.numpy())


def test_scan_gradients_against_differences(dev):
    A, D = _mods()
    rng = np.random.default_rng(5)
    B, T, C, N = 2, 19, 3, 5
    v = [rng.standard_normal((B, T, C)), rng.standard_normal((B, T, C)), -0.5 - rng.random((C, N)),
         rng.standard_normal((B, T, N)), rng.standard_normal((B, T, N)), rng.standard_normal(C),
         rng.standard_normal((B, T, C)), rng.standard_normal(C), rng.standard_normal((B, C, N))]
    g = rng.standard_normal((B, T, C))

    def loss(vals):
        with A.no_grad():
            L = [A.Tensor(D.from_numpy(a)) for a in vals]
            return float((A.ssm_scan(*L[:8], state=L[8], lengths=[19, 12]).numpy() * g).sum())
    L = [A.Tensor(D.from_numpy(a), requires_grad=True) for a in v]
    A.ssm_scan(*L[:8], state=L[8], lengths=[19, 12]).backward(D.from_numpy(g))
    for i, x in enumerate(L):
        r = rng.standard_normal(v[i].shape)
        e = 1e-5
        up, down = (loss(v[:i] + [v[i] + s * e * r] + v[i + 1:]) for s in (1, -1))
        want = float((x.grad.numpy() * r).sum())
        # a central difference is off by e^2 / 6 of a third derivative and 2^-53 |loss| / e
        assert abs((up - down) / (2 * e) - want) <= 1e-6 * max(1.0, abs(want)), i


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("B,C,N,G", [(1, 1, 1, 1), (3, 70, 16, 2), (2, 33, 13, 1), (2, 65, 64, 1), (1, 24, 20, 3)])
def test_scan_in_pieces(dev, dt, B, C, N, G):
    """A sequence in two calls and then position by position gives the whole sequence's values."""
    A, D = _mods()
    rng = np.random.default_rng(N)
    T = 25

    def normal(*s):
        return rng.standard_normal(s).astype(dt)
    u, d, z = normal(B, T, C), normal(B, T, C) * dt(.5), normal(B, T, C)
    Bm, Cm = normal(B, T, G, N), normal(B, T, G, N)
    Am, Dm, bias = (-0.5 - rng.random((C, N))).astype(dt), normal(C), normal(C)
    w = [A.Tensor(D.from_numpy(a)) for a in (Am, Dm, bias)]

    def part(sl, state=None):
        a = [A.Tensor(D.from_numpy(np.ascontiguousarray(x[:, sl]))) for x in (u, d, Bm, Cm, z)]
        if isinstance(sl, int):
            return A.ssm_scan_step(a[0], a[1], w[0], a[2], a[3], w[1], a[4], w[2], state), state
        return A.ssm_scan(a[0], a[1], w[0], a[2], a[3], w[1], a[4], w[2], state=state, return_state=True)
    with A.no_grad():
        whole, end = part(slice(0, T))
        y1, s = part(slice(0, 7))
        y2, s = part(slice(7, 20), s)
        steps = [part(t, s)[0].numpy() for t in range(20, T)]
    got = np.concatenate([y1.numpy(), y2.numpy(), np.stack(steps, 1)], 1)
    close(got, whole.numpy(), dt, 64, "y")
    close(s, end.numpy(), dt, 64, "state")


# --------------------------------------------------------- cross attention
def cross_ref(q, k, v, lengths, scale):
    H, Hk = q.shape[1], k.shape[1]
    outs = []
    for i in range(q.shape[0]):
        n = k.shape[2] if lengths is None else lengths[i]
        kr, vr = (x[i, :, :n].repeat_interleave(H // Hk, 0) for x in (k, v))
        s = q[i] @ kr.transpose(1, 2) * scale
        outs.append(torch.softmax(s, -1) @ vr if n else 0 * q[i])
    return torch.stack(outs)


CROSS = [  # B, H, Hk, Tq, Tk, D, lengths, strided
    (1, 1, 1, 1, 1, 1, None, False),
    (2, 2, 2, 1, 300, 64, [300, 0], True),
    (2, 8, 2, 1, 77, 32, [1, 77], False),
    (1, 2, 1, 17, 33, 5, None, False),
    (3, 4, 2, 5, 63, 31, [0, 63, 32], True),
    (2, 3, 3, 70, 65, 64, [65, 64], True),
    (1, 6, 2, 40, 129, 72, [97], False),
    (2, 2, 1, 130, 40, 96, None, True),
    (1, 4, 4, 33, 200, 100, None, False),
    (2, 4, 1, 50, 70, 128, [70, 13], True),
    (1, 1, 1, 600, 3, 40, None, False),
    (1, 1, 1, 3, 3000, 48, None, True),
    (1, 12, 12, 200, 160, 64, None, True),
    (2, 4, 1, 1, 900, 128, [900, 130], True),   # up to 16 rows per key/value head
    (1, 6, 2, 5, 210, 100, None, False),
    (4, 16, 1, 1, 70, 96, [1, 0, 70, 16], False),
    (2, 4, 2, 3, 150, 80, [150, 20], True),     # widths between the powers of two
    (1, 4, 1, 60, 90, 80, None, True),
    (2, 2, 2, 40, 70, 44, None, False),
    (1, 4, 2, 5, 70, 76, None, False),
    (1, 2, 2, 30, 60, 77, None, False),
    (1, 2, 1, 8, 130, 37, [120], True),
    (1, 3, 3, 45, 40, 120, None, True),
    (9, 1, 1, 90, 1100, 40, [0, 1, 1100, 64, 65, 600, 1099, 33, 2], False),  # parts by the lengths' sum
]


def bthd(a, strided):
    """(B, H, T, D) on the device, or as heads out of a [B, T, H, D] buffer."""
    _, D = _mods()
    if not strided:
        return D.from_numpy(a)
    return D.from_numpy(np.ascontiguousarray(a.transpose(0, 2, 1, 3))).transpose(0, 2, 1, 3)


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", CROSS, ids=lambda c: "-".join(str(v) for v in c[:6]))
def test_cross_attention(dev, dt, case):
    A, D = _mods()
    B, H, Hk, Tq, Tk, Dh, lengths, strided = case
    rng = np.random.default_rng(Tq * 13 + Tk)
    q, g = (rng.standard_normal((B, H, Tq, Dh)).astype(dt) for _ in range(2))
    k, v = (rng.standard_normal((B, Hk, Tk, Dh)).astype(dt) for _ in range(2))
    Q, Kt, V = (A.Tensor(bthd(x, strided), requires_grad=True) for x in (q, hide(k, lengths, 2), hide(v, lengths, 2)))
    o = A.cross_attention(Q, Kt, V, lengths=lengths)
    o.backward(bthd(g, strided))
    rq, rk, rv = t64(q), t64(k), t64(v)
    ro = cross_ref(rq, rk, rv, lengths, Dh ** -.5)
    grads = torch.autograd.grad(ro, (rq, rk, rv), t64(g, False))
    close(o, ro, dt, 512, "o")
    for x, want, n in zip((Q, Kt, V), grads, "qkv"):
        close(x.grad, want, dt, 512, "d" + n)
    with A.no_grad():
        assert bits_equal(A.cross_attention(Q, Kt, V, lengths=lengths).numpy(), o.numpy())


@pytest.mark.parametrize("dt", [F32, F64])
@pytest.mark.parametrize("case", [(2, 3, 3, 70, 65, 64, [65, 64]), (1, 4, 2, 90, 700, 96, None), (2, 2, 1, 40, 33, 128, [7, 33]),
                                  (2, 3, 1, 50, 47, 20, [3, 47]), (1, 2, 1, 40, 50, 72, None),
                                  (1, 2, 2, 33, 40, 45, [31])],
                         ids=lambda c: "-".join(str(v) for v in c[:6]))
def test_cross_attention_backward_without_kept_ds(dev, dt, case):
    """dS formed twice where its workspace is refused: the same dK and dV bits,
    and dQ to the same bar."""
    from dtmi import kernels as K
    A, D = _mods()
    B, H, Hk, Tq, Tk, Dh, lengths = case
    rng = np.random.default_rng(Tq + Tk)
    v = [rng.standard_normal(s).astype(dt) for s in ((B, H, Tq, Dh), (B, Hk, Tk, Dh), (B, Hk, Tk, Dh), (B, H, Tq, Dh))]

    def grads():
        L = [A.Tensor(D.from_numpy(x), requires_grad=True) for x in v[:3]]
        A.cross_attention(*L, lengths=lengths).backward(D.from_numpy(v[3]))
        return [x.grad.numpy() for x in L]
    kept = grads()
    before = K.attn_set_ds_limit(0)
    try:
        again = grads()
    finally:
        K.attn_set_ds_limit(before)
    assert bits_equal(kept[1], again[1]) and bits_equal(kept[2], again[2])
    R = [t64(x) for x in v[:3]]
    want = torch.autograd.grad(cross_ref(*R, lengths, Dh ** -.5), R, t64(v[3], False))
    close(kept[0], want[0], dt, 512, "dq, dS kept")
    close(again[0], want[0], dt, 512, "dq, dS formed twice")


def test_cross_attention_scale_and_large_scores(dev):
    """Scores far from zero, falling and rising along the keys: the running
    reference moves in every part and the sums stay finite."""
    A, D = _mods()
    rng = np.random.default_rng(3)
    for sign in (1.0, -1.0):
        q = np.abs(rng.standard_normal((1, 2, 20, 16))).astype(F32)
        ramp = np.linspace(0, 30, 500)[:, None] * sign
        k = (np.abs(rng.standard_normal((1, 2, 500, 16))) * 0.1 + ramp).astype(F32)
        v = rng.standard_normal((1, 2, 500, 16)).astype(F32)
        with A.no_grad():
            o = A.cross_attention(*(A.Tensor(D.from_numpy(x)) for x in (q, k, v)), scale=0.5)
        ro = cross_ref(t64(q, False), t64(k, False), t64(v, False), None, 0.5)
        # scores reach 250 (360 in base 2, 2^8.5): 17 products and a scaling round them by up to 18 x 2^8.5 u
        close(o, ro, F32, 18 * 363, "o")


def test_cross_attention_without_a_finite_score_is_zero(dev):
    A, D = _mods()
    q = np.ones((1, 1, 3, 1), F32)
    k = np.full((1, 1, 40, 1), -np.inf, F32)
    k[0, 0, 20:] = -np.inf
    v = np.ones((1, 1, 40, 1), F32)
    Q, Kt, V = (A.Tensor(D.from_numpy(x), requires_grad=True) for x in (q, k, v))
    o = A.cross_attention(Q, Kt, V)
    assert (o.numpy() == 0).all()
    k[0, 0, 7] = 2.0
    v[0, 0, 7] = 5.0
    with A.no_grad():
        o = A.cross_attention(A.Tensor(D.from_numpy(q)), A.Tensor(D.from_numpy(k)), A.Tensor(D.from_numpy(v)))
    assert (o.numpy() == 5).all()


@pytest.mark.parametrize("what", ["conv", "scan", "cross"])
def test_nothing_to_do(dev, what):
    """Empty batches, sequences and memories: empty or zero results, zero gradients."""
    A, D = _mods()

    def leaf(*s):
        return A.Tensor(D.full(s, 1.0, F32), requires_grad=True)
    for B, T in ((0, 5), (2, 0), (2, 3)):
        if what == "conv":
            x, w, b, s = leaf(B, T, 8), leaf(4, 8), leaf(8), leaf(B, 3, 8)
            y, st = A.causal_conv(x, w, b, state=s, lengths=[0] * B, return_state=True)
            leaves = (x, w, b, s)
            assert (st.numpy() == 1).all()
        elif what == "scan":
            u, dt, Am, Bm, Cm, s = leaf(B, T, 8), leaf(B, T, 8), leaf(8, 5), leaf(B, T, 5), leaf(B, T, 5), leaf(B, 8, 5)
            y, st = A.ssm_scan(u, dt, Am, Bm, Cm, state=s, lengths=[0] * B, return_state=True)
            leaves = (u, dt, Am, Bm, Cm, s)
            assert (st.numpy() == 1).all()
        else:
            q, k, v = leaf(B, 2, T, 8), leaf(B, 2, 4, 8), leaf(B, 2, 4, 8)
            y = A.cross_attention(q, k, v, lengths=[0] * B)
            leaves = (q, k, v)
        assert (y.numpy() == 0).all()
        y.backward(D.full(y.shape, 1.0, F32))
        for x in leaves:
            assert x.grad.shape == x.shape and (x.grad.numpy() == 0).all()
    if what == "cross":
        q, k, v = leaf(2, 2, 3, 8), leaf(2, 2, 0, 8), leaf(2, 2, 0, 8)
        y = A.cross_attention(q, k, v)
        y.backward(D.full(y.shape, 1.0, F32))
        assert (y.numpy() == 0).all() and (q.grad.numpy() == 0).all() and k.grad.shape == k.shape


def test_lengths_are_checked(dev):
    A, D = _mods()
    x, w = A.Tensor(D.zeros((2, 5, 8))), A.Tensor(D.zeros((4, 8)))
    for bad, err in (([5, 6], IndexError), ([-1, 2], IndexError), ([1], ValueError), ([1.0, 2.0], TypeError)):
        with pytest.raises(err):
            A.causal_conv(x, w, lengths=bad)
    q, k = A.Tensor(D.zeros((2, 1, 3, 8))), A.Tensor(D.zeros((2, 1, 4, 8)))
    with pytest.raises(IndexError):
        A.cross_attention(q, k, k, lengths=[5, 0])


def test_entry_points_refuse_shapes(dev):
    import ctypes as C
    L = dev
    n = C.c_int64()
    assert L.dtmi_scan_kept(0, 1, 1, 8, 65, C.byref(n)) == 1 and b"64 states" in L.dtmi_last_error()
    assert L.dtmi_conv_step(0, 1, 8, 9, None, 8, None, None, None, 1, None, 8) == 1
    assert b"taps" in L.dtmi_last_error()
    assert L.dtmi_conv_step(0, 1, 8, 4, None, 8, None, None, None, 1, None, 8) == 1
    st = (C.c_int64 * 3)(1, 1, 1)
    a = [None, st, None, st, None, st, None, None, st, None, None]
    assert L.dtmi_xattn_fwd(0, 1, 3, 2, 1, 1, 8, 1.0, *a) == 1 and b"share" in L.dtmi_last_error()
    assert L.dtmi_xattn_fwd(0, 1, 2, 2, 1, 1, 129, 1.0, *a) == 1 and b"head dimension" in L.dtmi_last_error()
    assert L.dtmi_xattn_fwd(2, 1, 2, 2, 1, 1, 8, 1.0, *a) == 1 and b"dtype" in L.dtmi_last_error()


def test_rows_far_apart(dev):
    """Element offsets past 2^31 along the positions of a sequence."""
    A, D = _mods()
    rng = np.random.default_rng(1)
    T, step = 40, 56_000_000
    big = D.empty((step * (T - 1) + 256,), F32)
    rows = rng.standard_normal((T, 2, 64)).astype(F32)
    for t in range(T):
        big[t * step:t * step + 128].assign(rows[t].reshape(-1))

    def view(i):
        return D.DeviceArray(big.block, (1, 1, T, 64), F32, 64 * i * 4, (0, 0, step, 1))
    q = rng.standard_normal((1, 1, 5, 64)).astype(F32)
    with A.no_grad():
        o = A.cross_attention(A.Tensor(D.from_numpy(q)), A.Tensor(view(0)), A.Tensor(view(1)))
        want = cross_ref(t64(q, False), t64(rows[None, None, :, 0], False), t64(rows[None, None, :, 1], False), None, .125)
        close(o, want, F32, 512, "cross")
        x = D.DeviceArray(big.block, (1, T, 64), F32, 0, (0, step, 1))
        w = rng.standard_normal((3, 64)).astype(F32)
        y = A.causal_conv(A.Tensor(x), A.Tensor(D.from_numpy(w)))
        zero = torch.zeros(1, 2, 64, dtype=torch.float64)
        close(y, conv_ref(t64(rows[None, :, 0], False), t64(w, False), torch.zeros(64), zero, None, True)[0], F32, 19,
              "conv")
        Am = -np.ones((64, 4), F32)
        Bm = rng.standard_normal((1, T, 4)).astype(F32)
        y = A.ssm_scan(A.Tensor(x), A.Tensor(x), *(A.Tensor(D.from_numpy(a)) for a in (Am, Bm, Bm)))
        u = t64(rows[None, :, 0], False)
        z = torch.zeros((), dtype=torch.float64)
        close(y, scan_ref(u, u, t64(Am, False), t64(Bm[:, :, None], False), t64(Bm[:, :, None], False), z, None, z,
                          torch.zeros(1, 64, 4, dtype=torch.float64), None, True)[0], F32, 256, "scan")


def test_results_repeat(dev):
    """The same bits on every run: no sum depends on timing."""
    A, D = _mods()
    rng = np.random.default_rng(2)
    B, T, C, N = 2, 300, 200, 16

    def t(*s):
        return D.from_numpy(rng.standard_normal(s).astype(F32))
    v = [t(B, T, C), t(B, T, C), D.from_numpy((-rng.random((C, N))).astype(F32)), t(B, T, N), t(B, T, N), t(C), t(B, T, C),
         t(C)]
    q, k, g, gq = t(B, 4, T, 64), t(B, 2, 333, 64), t(B, T, C), t(B, 4, T, 64)
    w, b = t(4, C), t(C)

    def once():
        L = [A.Tensor(a, requires_grad=True) for a in v]
        y = A.ssm_scan(*L)
        y.backward(g)
        M = [A.Tensor(a, requires_grad=True) for a in (q, k, k)]
        o = A.cross_attention(*M, lengths=[333, 100])
        o.backward(gq)
        P = [A.Tensor(a, requires_grad=True) for a in (v[0], w, b)]
        c = A.causal_conv(*P)
        c.backward(g)
        return [x.numpy() for x in (y, o, c)] + [x.grad.numpy() for x in L + M + P]
    first = once()
    for a, b_ in zip(first, once()):
        assert bits_equal(a, b_)


def test_gradients_land_and_accumulate(dev):
    """Parameters with a place for their gradient get it written there; a second
    backward adds; an upstream gradient may be a transposed view; one tensor may
    be several operands; two graphs may be alive at once."""
    A, D = _mods()
    rng = np.random.default_rng(8)
    B, T, C, N = 2, 30, 40, 6

    def t(*s):
        return rng.standard_normal(s)
    x, w, b, Am, Dm, Bm = t(B, T, C), t(4, C), t(C), -rng.random((C, N)) - .5, t(C), t(B, T, N)
    g = t(B, C, T)
    flat = D.zeros((4 * C + C + C * N + C,), F64)
    leaves = [A.Tensor(D.from_numpy(a), requires_grad=True) for a in (w, b, Am, Dm)]
    off = 0
    for p in leaves:
        n = p.data.size
        p.grad_dest = flat[off:off + n].reshape(p.shape)
        off += n
    W, bias, At, Dt = leaves
    X, M = A.Tensor(D.from_numpy(x), requires_grad=True), A.Tensor(D.from_numpy(Bm), requires_grad=True)

    def graph():
        c = A.causal_conv(X, W, bias)
        return A.ssm_scan(c, c, At, M, M, Dt, z=X)  # the maps one tensor, the convolution's output twice
    y1, y2 = graph(), graph()
    up = D.from_numpy(g).transpose(0, 2, 1)  # (B, T, C), C not contiguous
    y1.backward(up)
    once = flat.numpy()
    for p in leaves:
        assert p.grad.ptr == p.grad_dest.ptr
    y2.backward(up)
    assert bits_equal(flat.numpy(), once + once)
    R = [t64(a) for a in (x, w, b, Am, Dm, Bm)]
    zero = torch.zeros(B, 3, C, dtype=torch.float64)
    rc, _ = conv_ref(R[0], R[1], R[2], zero, None, True)
    m = R[5][:, :, None]
    ry, _ = scan_ref(rc, rc, R[3], m, m, R[4], R[0], torch.zeros(C, dtype=torch.float64),
                     torch.zeros(B, C, N, dtype=torch.float64), None, True)
    want = torch.autograd.grad(ry, R, t64(g.transpose(0, 2, 1), False))
    for p, r, n in zip([X] + leaves + [M], want, ("x", "w", "b", "A", "D", "B and C")):
        close(p.grad.numpy() / 2, r, F64, 1024, "d" + n)


@pytest.mark.parametrize("what", ["conv", "scan"])
def test_lengths_uploaded_once_and_padding_left_out(dev, what):
    """An Indices serves as lengths for several calls; every sequence of a padded
    batch gives the bits it gives alone."""
    A, D = _mods()
    rng = np.random.default_rng(4)
    B, T, C, N = 5, 70, 48, 16
    ln = [70, 1, 0, 33, 64]
    ix = A.Indices(ln)
    x, m = rng.standard_normal((B, T, C)).astype(F32), rng.standard_normal((B, T, N)).astype(F32)
    w, Am = rng.standard_normal((4, C)).astype(F32), (-rng.random((C, N))).astype(F32)

    def run(x, m, ln):
        X, M = A.Tensor(D.from_numpy(x)), A.Tensor(D.from_numpy(m))
        if what == "conv":
            return A.causal_conv(X, A.Tensor(D.from_numpy(w)), lengths=ln, return_state=True)
        return A.ssm_scan(X, X, A.Tensor(D.from_numpy(Am)), M, M, lengths=ln, return_state=True)
    with A.no_grad():
        for _ in range(2):
            y, s = run(hide(x, ln), hide(m, ln), ix)
        for i, n in enumerate(ln):
            y1, s1 = run(x[i:i + 1, :n], m[i:i + 1, :n], None)
            assert (y.numpy()[i, n:] == 0).all()
            if what == "conv":
                assert bits_equal(y.numpy()[i, :n], y1.numpy()[0]) and bits_equal(s.numpy()[i], s1.numpy()[0])
            else:  # a sequence alone may be split differently
                close(y.numpy()[i, :n], y1.numpy()[0], F32, 64, "y")
                close(s.numpy()[i], s1.numpy()[0], F32, 64, "state")


@pytest.mark.parametrize("dt", [F32, F64])
def test_a_decoder_block(dev, dt):
    """The operators as a decoder uses them together: a projection into input
    and gate, the convolution and the scan over it, the result's queries reading
    an encoder's padded states; every parameter's gradient from one backward, and
    the same block one token at a time."""
    from dtmi import nn as N
    A, D = _mods()
    rng = np.random.default_rng(11)
    B, T, M, C, S, H, Kt = 2, 21, 13, 32, 4, 2, 3
    mem_len = [13, 6]

    def normal(*s, std=.3):
        return (rng.standard_normal(s) * std).astype(dt)
    P = dict(inp=normal(C, 2 * C), cw=normal(Kt, C), cb=normal(C), xp=normal(C, C + 2 * S), A=(-.5 - rng.random((C, S))).astype(dt),
             D=normal(C), bias=normal(C), wq=normal(C, C), wk=normal(C, C), wv=normal(C, C), out=normal(C, C))
    x, enc, g = normal(B, T, C, std=1.0), normal(B, M, C, std=1.0), normal(B, T, C, std=1.0)

    def split(t, sizes):
        """Column ranges of a projection, as products with selecting matrices."""
        outs, at = [], 0
        for n in sizes:
            sel = np.zeros((sum(sizes), n), dt)
            sel[at:at + n] = np.eye(n)
            outs.append(t @ A.Tensor(D.from_numpy(sel)))
            at += n
        return outs

    def heads(t, n):
        return t.reshape(B, n, H, C // H).transpose(0, 2, 1, 3)

    L = {n: A.Tensor(D.from_numpy(a), requires_grad=True) for n, a in P.items()}
    X, E = A.Tensor(D.from_numpy(x), requires_grad=True), A.Tensor(D.from_numpy(enc), requires_grad=True)

    def run(X, states=None):
        n = X.shape[1]
        u, z = split(N.linear(X, L["inp"], None), (C, C))
        c = A.causal_conv(u, L["cw"], L["cb"])
        d, Bm, Cm = split(N.linear(c, L["xp"], None), (C, S, S))
        y = A.ssm_scan(c, d, L["A"], Bm, Cm, L["D"], z, L["bias"])
        o = A.cross_attention(heads(N.linear(y, L["wq"], None), n), heads(N.linear(E, L["wk"], None), M),
                              heads(N.linear(E, L["wv"], None), M), lengths=mem_len)
        return N.linear(o.transpose(0, 2, 1, 3).reshape(B, n, C), L["out"], None)
    y = run(X)
    y.backward(D.from_numpy(g))

    R = {n: t64(a) for n, a in P.items()}
    rx, re = t64(x), t64(enc)

    def ref(rx):
        n = rx.shape[1]
        hd = lambda t, n: t.reshape(B, n, H, C // H).transpose(1, 2)  # noqa: E731
        u, z = (rx @ R["inp"]).split(C, -1)
        c, _ = conv_ref(u, R["cw"], R["cb"], torch.zeros(B, Kt - 1, C, dtype=torch.float64), None, True)
        d, Bm, Cm = (c @ R["xp"]).split((C, S, S), -1)
        yy, _ = scan_ref(c, d, R["A"], Bm[:, :, None], Cm[:, :, None], R["D"], z, R["bias"],
                         torch.zeros(B, C, S, dtype=torch.float64), None, True)
        o = cross_ref(hd(yy @ R["wq"], n), hd(re @ R["wk"], M), hd(re @ R["wv"], M), mem_len, (C // H) ** -.5)
        return o.transpose(1, 2).reshape(B, n, C) @ R["out"]
    ry = ref(rx)
    grads = torch.autograd.grad(ry, [rx, re] + [R[n] for n in P], t64(g, False))
    # eight operators in a row of the bars above
    close(y, ry, dt, 2048, "y")
    for t, want, n in zip([X, E] + [L[n] for n in P], grads, ["x", "enc"] + list(P)):
        close(t.grad, want, dt, 2048, "d" + n)

    # one token at a time, the states handed on
    with A.no_grad():
        cs, hs = D.zeros((B, Kt - 1, C), dt), D.zeros((B, C, S), dt)
        k, v = heads(N.linear(E, L["wk"], None), M), heads(N.linear(E, L["wv"], None), M)
        for t in range(T):
            u, z = split(N.linear(A.Tensor(D.from_numpy(np.ascontiguousarray(x[:, t]))), L["inp"], None), (C, C))
            c = A.causal_conv_step(u, L["cw"], L["cb"], cs)
            d, Bm, Cm = split(N.linear(c, L["xp"], None), (C, S, S))
            s = A.ssm_scan_step(c, d, L["A"], Bm, Cm, L["D"], z, L["bias"], hs)
            o = A.cross_attention(heads(N.linear(s, L["wq"], None), 1), k, v, lengths=mem_len)
            got = N.linear(o.reshape(B, C), L["out"], None)
            close(got, ry.detach().numpy()[:, t], dt, 2048 * 4, f"token {t}")
