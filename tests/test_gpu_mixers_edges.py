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
