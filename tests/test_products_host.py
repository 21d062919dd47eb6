"""Products of a training step (CPU): arguments that they refuse, before any device
work. Operands are views onto no memory: a check that let one through would fail at
the first device call instead of with the error expected here."""
import numpy as np
import pytest

from dtmi import kernels as K
from dtmi.autograd import Tensor, expert_linear, linear_cross_entropy
from dtmi.device import DeviceArray
from dtmi.optim import Muon, orthogonalize


class _Nowhere:
    ptr = 0
    nbytes = 0


def arr(*shape, dt=np.float32, strides=None):
    return DeviceArray(_Nowhere(), shape, dt, 0, strides)


def ten(*shape, **kw):
    return Tensor(arr(*shape, **kw))


@pytest.mark.parametrize("x,w,t,what", [
    ((3, 8), (7, 5), [0, 1, 2], "do not match"),
    ((3, 8), (8,), [0, 1, 2], "do not match"),
    ((3, 8), (8, 0), [0, 1, 2], "do not match"),
    ((3, 8), (8, 5), [0, 1], "targets of shape"),
    ((3, 1, 8), (8, 5), [0, 1, 2], "targets of shape"),
])
def test_loss_refuses_shapes(x, w, t, what):
    with pytest.raises(ValueError, match=what):
        linear_cross_entropy(ten(*x), ten(*w), t)


@pytest.mark.parametrize("t,ignore", [([0, 5, 1], None), ([0, -1, 1], None), ([2 ** 40, 0, 1], None)])
def test_loss_refuses_targets_outside_the_vocabulary(t, ignore):
    with pytest.raises(IndexError, match="out of bounds"):
        linear_cross_entropy(ten(3, 8), ten(8, 5), t, ignore=ignore)


def test_loss_refuses_types_and_options():
    with pytest.raises(TypeError, match="integers"):
        linear_cross_entropy(ten(3, 8), ten(8, 5), [0.0, 1.0, 2.0])
    with pytest.raises(TypeError, match="dtype mismatch"):
        linear_cross_entropy(ten(3, 8), ten(8, 5, dt=np.float64), [0, 1, 2])
    with pytest.raises(TypeError):
        linear_cross_entropy(ten(3, 8, dt=np.int32), ten(8, 5, dt=np.int32), [0, 1, 2])
    with pytest.raises(ValueError, match="b must be"):
        linear_cross_entropy(ten(3, 8), ten(8, 5), [0, 1, 2], ten(8))
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(ten(3, 8), ten(8, 5), [0, 1, 2], reduction="sum")


@pytest.mark.parametrize("x,w,sizes,b,what", [
    ((6, 8), (2, 7, 5), [3, 3], None, "w must be"),
    ((6, 8), (8, 5), [6], None, "w must be"),
    ((6, 8), (2, 8, 5), [3, 4], None, "more than the 6 rows"),
    ((6, 8), (2, 8, 5), [3, -1], None, "negative"),
    ((6, 8), (2, 8, 5), [2 ** 62, 2 ** 62], None, "more than the 6 rows"),
    ((6, 8), (2, 8, 5), [6], None, "one entry for each of the 2"),
    ((6, 8), (2, 8, 5), [[3, 3]], None, "one entry for each of the 2"),
    ((6, 8), (2, 8, 5), [3, 3], (5,), "b must be"),
    ((2, 3, 8), (2, 8, 5), [3, 3], None, "x must be"),
])
def test_experts_refuse(x, w, sizes, b, what):
    with pytest.raises(ValueError, match=what):
        expert_linear(ten(*x), ten(*w), sizes, ten(*b) if b else None)


def test_experts_refuse_types():
    with pytest.raises(TypeError, match="integers"):
        expert_linear(ten(6, 8), ten(2, 8, 5), [3.0, 3.0])
    with pytest.raises(TypeError, match="dtype mismatch"):
        expert_linear(ten(6, 8), ten(2, 8, 5, dt=np.float64), [3, 3])


def test_updates_refuse():
    with pytest.raises(ValueError, match="matrices are needed"):
        orthogonalize(arr(8))
    with pytest.raises(ValueError, match="contiguous"):
        orthogonalize([arr(8, 4, strides=(1, 8))])
    with pytest.raises(TypeError, match="dtype mismatch"):
        orthogonalize([arr(8, 4), arr(8, 4, dt=np.float64)])
    with pytest.raises(TypeError):
        orthogonalize(arr(8, 4, dt=np.int32))
    with pytest.raises(ValueError, match="matrices are needed"):
        Muon([arr(8, 4), arr(8)])
    ps = K.Matrices([arr(8, 4)], "Muon")
    for bad in (arr(4, 8), arr(8, 4, dt=np.float64)):
        with pytest.raises(ValueError, match="gradient must be"):
            K.muon(ps, [bad], ps.pointers([arr(8, 4)]), [1.0], 1.0, 0.9, True, 5, (1.0, 1.0, 1.0), 0.0)
    a = arr(8, 4)
    with pytest.raises(ValueError, match="overlap"):
        Muon([a, a])
    with pytest.raises(ValueError, match="overlap"):
        Muon([arr(2, 8, 4), DeviceArray(_Nowhere(), (4, 4), np.float32, 4 * 60)])
