"""Sequence mixers (CPU): arguments that the operators refuse, before any
device work. Operands are views onto no memory: a check that let one through
would fail at the first device call instead of with the error expected here."""
import numpy as np
import pytest

from dtmi import kernels as K
from dtmi.autograd import Tensor, causal_conv, causal_conv_step, cross_attention, ssm_scan, ssm_scan_step
from dtmi.device import DeviceArray


class _Nowhere:
    ptr = None
    nbytes = 0


def arr(*shape, dt=np.float32, strides=None):
    return DeviceArray(_Nowhere(), shape, dt, 0, strides)


def ten(*shape, **kw):
    return Tensor(arr(*shape, **kw))


@pytest.mark.parametrize("x,w,b,state,what", [
    ((2, 5, 8), (9, 8), None, None, "taps"),
    ((2, 5, 8), (0, 8), None, None, "taps"),
    ((2, 5, 8), (4, 7), None, None, "w must be"),
    ((2, 5, 8), (4, 8), (7,), None, "b must be"),
    ((2, 5, 8), (4, 8), (8,), (2, 4, 8), "state must be"),
    ((2, 5, 8), (4, 8), (8,), (1, 3, 8), "state must be"),
    ((5, 8), (4, 8), None, None, "x must be"),
])
def test_conv_refuses(x, w, b, state, what):
    with pytest.raises(ValueError, match=what):
        causal_conv(ten(*x), ten(*w), ten(*b) if b else None, state=arr(*state) if state else None)


def test_conv_refuses_types():
    with pytest.raises(ValueError, match="w must be"):
        causal_conv(ten(2, 5, 8), ten(4, 8, dt=np.float64))
    with pytest.raises(TypeError):
        causal_conv(ten(2, 5, 8, dt=np.int32), ten(4, 8, dt=np.int32))


@pytest.mark.parametrize("state", [(2, 3, 7), (3, 3, 8), (2, 2, 8)])
def test_conv_step_refuses_a_state_that_does_not_fit(state):
    with pytest.raises(ValueError, match="state must be"):
        causal_conv_step(ten(2, 8), ten(4, 8), None, arr(*state))


def test_step_states_are_contiguous():
    with pytest.raises(ValueError, match="contiguous"):
        causal_conv_step(ten(2, 8), ten(4, 8), None, arr(2, 3, 8, strides=(24, 1, 3)))
    with pytest.raises(ValueError, match="contiguous"):
        ssm_scan_step(ten(2, 8), ten(2, 8), ten(8, 4), ten(2, 4), ten(2, 4), None, None, None,
                      arr(2, 8, 4, strides=(64, 8, 1)))


def scan_args(**kw):
    a = dict(u=(2, 5, 8), dt=(2, 5, 8), A=(8, 4), B=(2, 5, 4), C=(2, 5, 4), D=(8,), z=(2, 5, 8), dt_bias=(8,))
    a.update(kw)
    return [ten(*a[n]) for n in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")]


@pytest.mark.parametrize("bad,what", [
    (dict(u=(5, 8)), "u must be"),
    (dict(dt=(2, 5, 7)), "dt must be"),
    (dict(A=(7, 4)), "A must be"),
    (dict(A=(8, 65), B=(2, 5, 65), C=(2, 5, 65)), "1 to 64 states"),
    (dict(A=(8, 0), B=(2, 5, 0), C=(2, 5, 0)), "1 to 64 states"),
    (dict(B=(2, 5, 3)), "B must be"),
    (dict(C=(2, 4, 4)), "C must be"),
    (dict(B=(2, 5, 3, 4), C=(2, 5, 3, 4)), "groups dividing"),
    (dict(B=(2, 5, 2, 4)), "C must be"),
    (dict(D=(7,)), "D must be"),
    (dict(z=(2, 6, 8)), "z must be"),
    (dict(dt_bias=(1,)), "dt_bias must be"),
])
def test_scan_refuses(bad, what):
    with pytest.raises(ValueError, match=what):
        ssm_scan(*scan_args(**bad))


def test_scan_refuses_a_state_that_does_not_fit():
    with pytest.raises(ValueError, match="state must be"):
        ssm_scan(*scan_args(), state=arr(2, 8, 5))
    with pytest.raises(ValueError, match="state must be"):
        ssm_scan_step(ten(2, 8), ten(2, 8), ten(8, 4), ten(2, 4), ten(2, 4), None, None, None, arr(1, 8, 4))


@pytest.mark.parametrize("q,k,v,what", [
    ((2, 4, 5, 8), (2, 3, 7, 8), (2, 3, 7, 8), "share"),
    ((2, 4, 5, 8), (1, 4, 7, 8), (1, 4, 7, 8), "match"),
    ((2, 4, 5, 8), (2, 4, 7, 9), (2, 4, 7, 9), "match"),
    ((2, 4, 5, 8), (2, 4, 7, 8), (2, 4, 6, 8), "one shape"),
    ((2, 4, 5, 129), (2, 4, 7, 129), (2, 4, 7, 129), "1 to 128"),
    ((4, 5, 8), (2, 4, 7, 8), (2, 4, 7, 8), "must be"),
])
def test_cross_attention_refuses(q, k, v, what):
    with pytest.raises(ValueError, match=what):
        cross_attention(ten(*q), ten(*k), ten(*v))


def test_kernel_wrappers_refuse_rows_that_are_not_contiguous():
    with pytest.raises(ValueError, match="contiguous"):
        K.conv_fwd(arr(2, 5, 8, strides=(40, 1, 5)), arr(4, 8))
    with pytest.raises(ValueError, match="contiguous"):
        K.xattn_fwd(arr(2, 4, 5, 8, strides=(160, 40, 1, 5)), arr(2, 4, 7, 8), arr(2, 4, 7, 8))
