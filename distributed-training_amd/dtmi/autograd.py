"""Reverse-mode autograd over device arrays, with dtrain's Tensor API.

Mirrors dtrain/autograd.py: `Tensor(data, requires_grad, name)`, `.grad`,
`.backward(grad=None)`, `.register_grad_ready_hook(fn)`, the operators
`+ - * @`, `.sum .mean .reshape .transpose .gelu .relu`, and the functional ops
`embedding`, `layer_norm`, `causal_attention`, `cross_entropy`, `no_grad`.
Without a counterpart there: beside causal_attention, `causal_conv`, `ssm_scan`,
`cross_attention` and the single-token `causal_conv_step`, `ssm_scan_step`; beside
cross_entropy and linear, `linear_cross_entropy` and `expert_linear`.

Differences from dtrain are in where the numbers live, not in semantics:
`.data` and `.grad` are DeviceArrays (HBM buffers owned by libdtmi; `.numpy()`
and `np.asarray` copy to the host), and every op's forward and backward is a
libdtmi kernel launch. `backward()` is dtrain's algorithm (autograd.py:151-195):
a topological order, a reverse walk, leaf accumulation `grad = g` or
`grad + g`, and grad-ready hooks called once per leaf with its final gradient.
"""
from __future__ import annotations

import numpy as np

from . import device as dev
from . import kernels as K
from .device import DeviceArray

_grad_enabled = True


class no_grad:
    """dtrain/autograd.py:19-26."""

    def __enter__(self):
        global _grad_enabled
        self.prev, _grad_enabled = _grad_enabled, False

    def __exit__(self, *a):
        global _grad_enabled
        _grad_enabled = self.prev


def _contig(x: DeviceArray) -> DeviceArray:
    return x if x.is_contiguous else x.contiguous()


def _unbroadcast(g: DeviceArray, shape: tuple) -> DeviceArray:
    """dtrain/autograd.py:29-36: sum g over the axes broadcast from `shape`."""
    shape = tuple(shape)
    if g.shape == shape:
        return g
    lead = g.ndim - len(shape)
    if lead > 0:
        g = _contig(g)
        rest = g.shape[lead:]
        if len(rest) == 1:  # [.., N] -> [N]: deterministic two-stage column sum
            g = K.colsum(g.reshape(-1, rest[0]))
        else:
            g = K.reduce_sum(g, list(range(lead)))
    axes = [i for i, s in enumerate(shape) if s == 1 and g.shape[i] != 1]
    if axes:
        g = K.reduce_sum(g, axes, keepdims=True)
    return g


def _broadcast_to(g: DeviceArray, shape) -> DeviceArray:
    """np.broadcast_to(g, shape).copy() on the device."""
    shape = tuple(shape)
    out = dev.empty(shape, g.dtype)
    if out.size == 0:
        return out
    nd = len(shape)
    pad = nd - g.ndim
    st = [0] * pad + [0 if (s == 1 and shape[pad + i] != 1) else g.strides[i] for i, s in enumerate(g.shape)]
    view = DeviceArray(g.block, shape, g.dtype, g.offset, st)
    K.copy_into(out, view)
    return out


class Tensor:
    __slots__ = ("data", "grad", "requires_grad", "_parents", "_backward", "_hooks", "name", "grad_dest",
                 "_dest_live", "_ln_pre", "_rowdot", "_ln_out", "__weakref__")

    def __init__(self, data, requires_grad=False, _parents=(), _backward=None, name=None):
        self.data = data if isinstance(data, DeviceArray) else dev.asarray(np.asarray(data))
        self.grad = None
        self.requires_grad = requires_grad
        self._parents = _parents
        self._backward = _backward
        self._hooks = []
        self.name = name
        # Optional preallocated home for this leaf's gradient (same shape and
        # dtype), e.g. its slot in a gradient bucket: the kernel producing
        # the gradient writes straight into it, so the bucket needs no copy.
        self.grad_dest = None
        self._dest_live = None
        # A LayerNorm of this tensor computed by the kernel that produced it
        # (w, b, eps, y, mean, rstd); layer_norm(self, w, b, eps) takes it once.
        self._ln_pre = None
        self._rowdot = None
        # the output of layer_norm: the backward of the product that reads it
        # may hand its gradient over as split-K partials (kernels.SplitSum),
        # which the LayerNorm backward adds as it loads them
        self._ln_out = False

    # ------------------------------------------------------------ utilities
    @property
    def shape(self):
        return self.data.shape

    @property
    def dtype(self):
        return self.data.dtype

    def numpy(self):
        return self.data.numpy()

    def register_grad_ready_hook(self, fn):
        """fn(tensor) is called once this leaf's gradient is complete."""
        self._hooks.append(fn)

    def __repr__(self):
        return f"Tensor(shape={self.shape}, dtype={self.dtype}, requires_grad={self.requires_grad})"

    @staticmethod
    def _make(data, parents, backward):
        rg = _grad_enabled and any(p.requires_grad for p in parents)
        return Tensor(data, rg, parents if rg else (), backward if rg else None)

    def _wrap(self, o):
        return o if isinstance(o, Tensor) else Tensor(np.asarray(o, dtype=self.dtype))

    # ---------------------------------------------------------------- ops
    def __add__(self, o):
        a, b = self, self._wrap(o)

        def bw(g):
            return _unbroadcast(g, a.shape), _unbroadcast(g, b.shape)
        return Tensor._make(K.binary("add", a.data, b.data), (a, b), bw)

    __radd__ = __add__

    def __neg__(self):
        return Tensor._make(K.neg(self.data), (self,), lambda g: (K.neg(g),))

    def __sub__(self, o):
        return self + (-self._wrap(o))

    def __mul__(self, o):
        a, b = self, self._wrap(o)

        def bw(g):
            return (_unbroadcast(K.binary("mul", g, b.data), a.shape),
                    _unbroadcast(K.binary("mul", g, a.data), b.shape))
        return Tensor._make(K.binary("mul", a.data, b.data), (a, b), bw)

    __rmul__ = __mul__

    def __matmul__(self, o):
        a, b = self, o
        A, B = _contig(a.data), _contig(b.data)
        if A.ndim >= 2 and B.ndim == 2:
            lead = A.shape[:-1]
            y = K.gemm(A.reshape(-1, A.shape[-1]), B).reshape(*lead, B.shape[1])

            def bw(g):
                g2 = _contig(g).reshape(-1, B.shape[1])
                A2 = A.reshape(-1, A.shape[-1])
                ga = K.gemm(g2, B, a_kcontig=True, b_kcontig=True).reshape(A.shape)  # g @ b^T
                gb = K.gemm(A2, g2, a_kcontig=False, b_kcontig=False)               # sum_batch a^T @ g
                return ga, gb
        elif A.ndim == 3 and B.ndim == 3 and A.shape[0] == B.shape[0]:
            y = K.gemm(A, B)

            def bw(g):
                gc = _contig(g)
                return K.gemm(gc, B, a_kcontig=True, b_kcontig=True), K.gemm(A, gc, a_kcontig=False, b_kcontig=False)
        else:
            raise NotImplementedError(f"matmul of shapes {A.shape} @ {B.shape}")
        return Tensor._make(y, (a, b), bw)

    def sum(self, axis=None, keepdims=False):
        a = self
        nd = a.data.ndim
        axes = list(range(nd)) if axis is None else [axis] if isinstance(axis, int) else list(axis)
        axes = [x % nd for x in axes] if nd else []
        out = K.reduce_sum(_contig(a.data), axes, keepdims=keepdims)

        def bw(g):
            if axis is not None and not keepdims:
                g = _contig(g).reshape(tuple(1 if d in axes else s for d, s in enumerate(a.shape)))
            return (_broadcast_to(g, a.shape),)
        return Tensor._make(out, (a,), bw)

    def mean(self, axis=None, keepdims=False):
        n = self.data.size if axis is None else self.data.shape[axis]
        return self.sum(axis, keepdims) * (1.0 / n)

    def reshape(self, *shape):
        a = self
        return Tensor._make(a.data.reshape(*shape), (a,), lambda g: (g.reshape(a.shape),))

    def transpose(self, *axes):
        a = self
        inv = tuple(np.argsort(axes))
        return Tensor._make(a.data.transpose(*axes), (a,), lambda g: (g.transpose(*inv),))

    def gelu(self):
        x = _contig(self.data)

        def bw(g):
            return (K.gelu_bwd(x, _contig(g)),)
        return Tensor._make(K.gelu_fwd(x), (self,), bw)

    def relu(self):
        x = _contig(self.data)
        return Tensor._make(K.relu_fwd(x), (self,), lambda g: (K.relu_bwd(x, _contig(g)),))

    # ------------------------------------------------------------ backward
    def backward(self, grad=None):
        """dtrain/autograd.py:151-195 over device gradients."""
        if grad is None:
            if self.data.size != 1:
                raise ValueError("backward() without a gradient needs a scalar output")
            grad = dev.ones_later(self.data.shape, self.data.dtype)
        elif not isinstance(grad, DeviceArray):
            grad = dev.asarray(np.asarray(grad, dtype=self.dtype))
        order, seen, users = [], set(), {}
        stack = [(self, False)]
        while stack:
            node, done = stack.pop()
            if done:
                order.append(node)
                continue
            if id(node) in seen:
                continue
            seen.add(id(node))
            stack.append((node, True))
            for p in node._parents:
                users[id(p)] = users.get(id(p), 0) + 1
                if id(p) not in seen:
                    stack.append((p, False))
        # A leaf with a grad_dest, no gradient yet and exactly one incoming
        # edge lets its producing node write the gradient straight into the
        # destination (grad_out); any other case goes through a new array.
        live = []
        for node in order:
            if node._backward is None and node.grad_dest is not None and node.requires_grad:
                if node.grad is None and users.get(id(node), 0) == 1:
                    node._dest_live = node.grad_dest
                    live.append(node)
        try:
            grads = {id(self): grad}
            for node in reversed(order):
                g = grads.pop(id(node), None)
                if g is None:
                    continue
                if node._backward is None:
                    if isinstance(g, K.SplitSum):
                        g = g.value()
                    if node.requires_grad:
                        node._dest_live = None
                        if node.grad is None:
                            node.grad = g
                        elif node.grad_dest is not None and node.grad.ptr == node.grad_dest.ptr:
                            node.grad = K.binary("add", node.grad, g, out=node.grad)  # accumulate in place
                        else:
                            node.grad = K.binary("add", node.grad, g)
                        for h in node._hooks:
                            h(node)
                    continue
                self._backprop(node, g, grads)
        finally:
            for node in live:
                node._dest_live = None
        return None

    @staticmethod
    def _backprop(node, g, grads):
        # A backward function may offer `with_addend = (i, f)`: when parent i
        # already has a pending gradient P, f(g, P) returns the parents'
        # gradients with P already added into parent i's (P + its own, the
        # order of the sum below), or None to decline.
        # a gradient left as split-K partials goes on as it is only to a
        # backward that takes it (the LayerNorm's); any other gets its value
        if isinstance(g, K.SplitSum) and not getattr(node._backward, "takes_split_sum", False):
            g = g.value()
        outs, summed = None, -1
        fuse = getattr(node._backward, "with_addend", None)
        if fuse is not None:
            i, f = fuse
            p = node._parents[i]
            if p.requires_grad and id(p) in grads:
                outs = f(g, grads[id(p)])
                summed = i if outs is not None else -1
        if outs is None:
            outs = node._backward(g)
        for j, (p, pg) in enumerate(zip(node._parents, outs)):
            if not p.requires_grad or pg is None:
                continue
            if tuple(pg.shape) != tuple(p.shape):
                raise RuntimeError(f"gradient shape {pg.shape} != {p.shape}")
            k = id(p)
            if j == summed or k not in grads:
                grads[k] = pg
            else:
                a = grads[k].value() if isinstance(grads[k], K.SplitSum) else grads[k]
                grads[k] = K.binary("add", a, pg.value() if isinstance(pg, K.SplitSum) else pg)


def grad_out(t: Tensor):
    """Where a backward function should write the gradient of `t`: its live
    grad_dest during backward() (see Tensor.grad_dest), else None."""
    return t._dest_live


# ------------------------------------------------------------ functional ops
class Indices:
    """Integer ids (token ids, positions, targets) mirrored once in HBM.

    dtrain passes index arrays as NumPy arrays (autograd.py:199, 250); every
    op accepting one also accepts an Indices, so a batch can be uploaded once
    and reused with no host-to-device copy inside a step. The embedding
    backward's stable segment order (the order np.add.at adds rows in) is
    computed on first use and kept with it.
    """

    __slots__ = ("host", "dev", "shape", "_segs", "_rows", "_lo", "_hi")

    def __init__(self, idx):
        self.host = np.asarray(idx)
        if not np.issubdtype(self.host.dtype, np.integer):
            raise TypeError("indices must be integers")
        self.shape = self.host.shape
        self._lo = int(self.host.min()) if self.host.size else 0
        self._hi = int(self.host.max()) if self.host.size else -1
        self.dev = dev.from_numpy(self.host.reshape(-1).astype(np.int64))
        self._segs = self._rows = None

    def check(self, n: int, what: str, allow_negative: bool):
        lo = -n if allow_negative else 0
        if self.host.size and (self._lo < lo or self._hi >= n):
            raise IndexError(f"{what} out of bounds for size {n}")

    def wrapped(self, n: int) -> "Indices":
        """Negative ids taken modulo n (NumPy indexing)."""
        if self._lo >= 0:
            return self
        return Indices(np.where(self.host < 0, self.host + n, self.host))

    def segments(self):
        """The stable sort of the indices by row, built on the device from
        the uploaded ids once (kernels.embedding_segments)."""
        if self._segs is None:
            self._segs = K.embedding_segments(self.dev)
        return self._segs

    def expert_rows(self):
        """The host values as the rows of expert_linear's experts, checked once."""
        if self._rows is None:
            self._rows = K.ExpertRows(self.host)
        return self._rows


def as_indices(idx) -> Indices:
    return idx if isinstance(idx, Indices) else Indices(idx)


def embedding(weight: Tensor, idx) -> Tensor:
    """dtrain/autograd.py:199-204. `idx`: a host integer array or an Indices."""
    V = weight.shape[0]
    ix = as_indices(idx)
    ix.check(V, "index", allow_negative=True)
    ix = ix.wrapped(V)
    w = weight.data if weight.data.is_contiguous else weight.data.contiguous()
    out = K.embedding_fwd(w, ix.dev, ix.shape)

    def bw(g):
        return (K.embedding_bwd(_contig(g).reshape(-1, weight.shape[1]), V, ix.segments(), out=grad_out(weight)),)
    return Tensor._make(out, (weight,), bw)


def layer_norm(x: Tensor, w: Tensor, b: Tensor, eps=1e-5) -> Tensor:
    """dtrain/autograd.py:207-223. When the kernel that produced x already
    computed this LayerNorm of it (nn.linear(..., ln=...)), its result is used
    (the same bits)."""
    xd = _contig(x.data)
    pre, x._ln_pre = x._ln_pre, None
    if pre is not None and pre[0] is w and pre[1] is b and pre[2] == eps:
        y, mean, rstd = pre[3:]
    else:
        y, mean, rstd = K.layernorm_fwd(xd, _contig(w.data), _contig(b.data), eps)

    def bw(g, dx_addend=None):
        # g may be a kernels.SplitSum (the producer's split-K partials)
        return K.layernorm_bwd(g if isinstance(g, K.SplitSum) else _contig(g), xd, _contig(w.data), mean, rstd,
                               dw_out=grad_out(w), db_out=grad_out(b), dx_addend=dx_addend)

    def bw_add(g, pending):
        # x already has a pending gradient (the residual path): the kernel
        # writes pending + dx, the engine's own sum, in the same pass
        if isinstance(pending, K.SplitSum) or not pending.is_contiguous or pending.dtype != xd.dtype or \
                pending.shape != xd.shape:
            return None
        return bw(g, dx_addend=pending)
    bw.with_addend = (0, bw_add)
    bw.takes_split_sum = True
    t = Tensor._make(y, (x, w, b), bw)
    t._ln_out = True
    return t


def causal_attention(q: Tensor, k: Tensor, v: Tensor) -> Tensor:
    """dtrain/autograd.py:226-247 for (B, H, T, D) inputs (any strides with a
    contiguous last axis). Keeps row max/sum instead of the probabilities."""
    o, rmax, rsum = K.attn_fwd(q.data, k.data, v.data)

    def bw(g):
        gq = dev.empty(q.shape, q.dtype)
        gk = dev.empty(q.shape, q.dtype)
        gv = dev.empty(q.shape, q.dtype)
        K.attn_bwd(q.data, k.data, v.data, o, _contig(g), rmax, rsum, dq=gq, dk=gk, dv=gv)
        return gq, gk, gv
    return Tensor._make(o, (q, k, v), bw)


def cross_entropy(logits: Tensor, targets) -> Tensor:
    """dtrain/autograd.py:250-266: mean cross-entropy; `targets`: a host integer
    array or an Indices.

    With gradients enabled the logits' gradient ([rows, V], as large as the
    logits) is computed by the forward pass and held until backward runs or
    the returned loss tensor is dropped. Evaluate under `no_grad()` to skip
    it: a validation loss taken with gradients on keeps that array alive for
    as long as its loss tensor lives."""
    z = _contig(logits.data)
    V = z.shape[-1]
    t = as_indices(targets)
    t.check(V, "target", allow_negative=False)
    if not (_grad_enabled and logits.requires_grad):
        loss, rmax, rsum = K.xent_fwd(z, t.dev)
        return Tensor._make(loss, (logits,), None)
    # training: the gradient for an upstream gradient of 1 comes out of the
    # forward pass (one read of the logits); the backward rescales it in place
    # when the upstream gradient differs, and a second backward through this
    # node recomputes it from the logits and the saved row statistics
    loss, rmax, rsum, dz = K.xent_fused(z, t.dev)
    pending = [dz]

    def bw(g):
        g1 = _contig(g).reshape(1)
        if pending:
            return (K.xent_grad_scale(pending.pop(), g1),)
        return (K.xent_bwd(z, t.dev, rmax, rsum, g=g1),)
    return Tensor._make(loss, (logits,), bw)


# --------------------------------------------- products of a training step
# Beside linear and cross_entropy. dtrain has no counterpart.
def linear_cross_entropy(x: Tensor, w: Tensor, targets, b: Tensor | None = None, ignore: int | None = None,
                         reduction: str = "mean") -> Tensor:
    """cross_entropy(x @ w + b, targets) without the logits: x [..., C], w [C, V] (a
    transposed embedding table [V, C] is read as it lies), b [V], `targets` a host
    integer array or an Indices of x's leading shape.

    Rows whose target is `ignore` do not count: their loss and gradients are 0, whatever
    x holds there. `reduction` "mean" gives the mean over the others (0 if there are
    none), "none" the loss of every row, which without gradients (`no_grad()`) is minus
    the log probability of its target: no logit is written then. The gradients of a mean
    are computed by the forward pass, as cross_entropy's are, from about 1 GiB of logits
    at a time; those of single losses by backward, which forms the logits again."""
    if reduction not in ("mean", "none"):
        raise ValueError(f"linear_cross_entropy: reduction must be 'mean' or 'none', not {reduction!r}")
    X = _contig(x.data)
    if X.ndim < 1 or len(w.shape) != 2 or w.shape[0] != X.shape[-1] or w.shape[1] < 1:
        raise ValueError(f"linear_cross_entropy: x {x.shape} and w {w.shape} do not match")
    lead, (C, V) = X.shape[:-1], w.shape
    K.same_dtype(X, w.data)
    if b is not None and (b.shape != (V,) or b.dtype != X.dtype):
        raise ValueError(f"linear_cross_entropy: b must be {X.dtype} of shape {(V,)}, not {b.dtype} {b.shape}")
    tied = not w.data.is_contiguous and w.data.transpose(1, 0).is_contiguous
    W = w.data.transpose(1, 0) if tied else _contig(w.data)
    bd = _contig(b.data) if b is not None else None
    ix = targets if isinstance(targets, Indices) else None
    host = ix.host if ix is not None else np.asarray(targets)
    if host.size and not np.issubdtype(host.dtype, np.integer):
        raise TypeError("indices must be integers")
    if host.shape != lead:
        raise ValueError(f"linear_cross_entropy: targets of shape {host.shape} for x {x.shape}")
    rows = host.size
    lo, hi = (ix._lo, ix._hi) if ix is not None else (host.min(), host.max()) if rows else (0, -1)
    n = rows
    if ignore is not None and lo <= ignore <= hi:
        keep = host != ignore
        n = int(np.count_nonzero(keep))
        if not 0 <= ignore < V and n < rows:
            lo, hi = (host[keep].min(), host[keep].max()) if n else (0, -1)
    if lo < 0 or hi >= V:
        raise IndexError(f"target out of bounds for size {V}")
    X2 = X if X.ndim == 2 else X.reshape(rows, C)
    t = ix.dev if ix is not None else dev.from_numpy(host.reshape(-1).astype(np.int64))
    mean = reduction == "mean"
    need = [_grad_enabled and p is not None and p.requires_grad for p in (x, w, b)]
    grads = dict(need_dx=need[0], need_dw=need[1], need_db=need[2])
    rest = dict(tied=tied, coef=1.0 / n if mean and n else 1.0, counted=n, ignore=int(ignore or 0))
    ls, total, *made = K.linear_xent(X2, W, bd, t, losses=not mean, mean=mean, **rest, **(grads if mean else {}))
    pending = [made] if mean and any(need) else []

    def bw(g):
        if pending:
            # into their destinations, or in place
            made, dests = list(pending.pop()), (None, None if tied else grad_out(w),
                                                grad_out(b) if b is not None else None)
            if not dev.known_ones(g):
                K.grad_scale_multi([d for d, o in zip(made, dests) if o is None], _contig(g).reshape(1))
            dx, dw, db = [d if o is None or d is None else K.scale(d, alpha_dev=_contig(g).reshape(1), out=o)
                          for d, o in zip(made, dests)]
        else:
            dx, dw, db = K.linear_xent(X2, W, bd, t, g=_contig(g).reshape(-1), **rest, **grads)[2:]
        if dx is not None and dx.shape != x.shape:
            dx = dx.reshape(x.shape)
        dw = dw.transpose(1, 0) if dw is not None and tied else dw
        return (dx, dw) if b is None else (dx, dw, db)
    out = total if mean else ls.reshape(lead)
    return Tensor._make(out, (x, w) if b is None else (x, w, b), bw)


def expert_linear(x: Tensor, w: Tensor, sizes, b: Tensor | None = None) -> Tensor:
    """Products of experts that each take some of the rows: x [R, K] sorted by expert, the
    first sizes[0] rows expert 0's, the next sizes[1] expert 1's, ...; y = x @ w[e] +
    b[e] with w [E, K, N], b [E, N]. `sizes`: one whole number for each expert (a host
    array or an Indices), adding up to R at most. Rows past the last expert's give 0 and
    get no gradient, and are not read; an expert may have none (embedding() gathers rows
    by expert, with a gradient)."""
    X, W = _contig(x.data), _contig(w.data)
    if X.ndim != 2:
        raise ValueError(f"expert_linear: x must be [rows, {w.shape[1] if len(w.shape) == 3 else 'K'}], not {x.shape}")
    if isinstance(sizes, Indices):
        n = sizes.expert_rows()
    else:
        n = K.ExpertRows(sizes)
    y = K.expert_linear_fwd(X, W, n, _contig(b.data) if b is not None else None)

    def bw(g):
        dx, dw, db = K.expert_linear_bwd(X, W, _contig(g), n, x.requires_grad, w.requires_grad,
                                         b is not None and b.requires_grad, dw_out=grad_out(w),
                                         db_out=grad_out(b) if b is not None else None)
        return (dx, dw) if b is None else (dx, dw, db)
    return Tensor._make(y, (x, w) if b is None else (x, w, b), bw)


# --------------------------------------------------------- sequence mixers
# Beside causal_attention, for decoders whose own state does not grow and that
# read an encoder. dtrain has no counterpart.
def _rows(x: DeviceArray) -> DeviceArray:
    """x itself where its last axis is contiguous, else a copy."""
    return x if x.ndim == 0 or x.shape[-1] <= 1 or x.strides[-1] == 1 else x.contiguous()


def _lengths_of(lengths, B: int, T: int):
    """The lengths of a padded batch on the device, checked on the host: one
    whole number of 0..T per sequence (a host array or an Indices)."""
    if lengths is None:
        return None
    if not isinstance(lengths, Indices) and np.size(lengths) == 0:
        lengths = np.zeros(np.shape(lengths), np.int64)
    ix = as_indices(lengths)
    if ix.shape != (B,):
        raise ValueError(f"lengths must have one entry for each of the {B} sequences, not shape {ix.shape}")
    ix.check(T + 1, "length", allow_negative=False)
    return ix.dev


def _state_of(state):
    return state if state is None or isinstance(state, Tensor) else Tensor(state)


def causal_conv(x: Tensor, w: Tensor, b: Tensor | None = None, silu: bool = True, state=None, lengths=None,
                return_state: bool = False):
    """Short causal convolution over time of x [B, T, C], each channel by itself:
    y[t] = act(b + sum_k w[k] x[t - K + 1 + k]) with w [K, C], K of 1 to 8, and act
    SiLU (silu=False: none).

    `state` [B, K - 1, C] (a Tensor or DeviceArray) holds the inputs before the
    first position, zeros without one; it may be moved on in place once the call
    returns. `lengths` (one per sequence, a host array
    or an Indices) marks a padded batch: y and the gradients are zero from a
    sequence's length on, and what lies there is not read. With `return_state`,
    returns (y, state): the last K - 1 inputs of every sequence as a DeviceArray,
    which carries no gradient."""
    X = _rows(x.data)
    if X.ndim != 3:
        raise ValueError(f"causal_conv: x must be [B, T, C], not {x.shape}")
    ln = _lengths_of(lengths, X.shape[0], X.shape[1])
    st = _state_of(state)
    W, bd, S = _contig(w.data), _contig(b.data) if b is not None else None, _contig(st.data) if st is not None else None
    if S is not None and S is st.data and _grad_enabled and any(p is not None and p.requires_grad for p in (x, w, b, st)):
        S = S.copy()  # the backward reads it again; causal_conv_step may have moved the caller's on by then
    y, new = K.conv_fwd(X, W, bd, S, ln, silu, return_state)

    def bw(g):
        dx, dw, db, ds = K.conv_bwd(X, W, bd, _rows(g), S, ln, silu, need_dstate=st is not None and st.requires_grad,
                                    dw_out=grad_out(w), db_out=grad_out(b) if b is not None else None)
        return tuple([dx, dw] + ([db] if b is not None else []) + ([ds] if st is not None else []))
    t = Tensor._make(y, tuple([x, w] + ([b] if b is not None else []) + ([st] if st is not None else [])), bw)
    return (t, new) if return_state else t


def causal_conv_step(x: Tensor, w: Tensor, b: Tensor | None, state: DeviceArray, silu: bool = True) -> Tensor:
    """causal_conv for one new position per sequence: x [B, C]. `state`
    [B, K - 1, C], contiguous, moves on in place. No gradient."""
    y = K.conv_step(_rows(x.data), _contig(w.data), _contig(b.data) if b is not None else None, state, silu)
    return Tensor(y)


def _maps(m: Tensor, lead: int) -> DeviceArray:
    """B or C of a scan as [..., G, N]: one group where the axis is left out."""
    d = _rows(m.data)
    if d.ndim == lead + 1:
        d = DeviceArray(d.block, d.shape[:-1] + (1,) + d.shape[-1:], d.dtype, d.offset,
                        tuple(d.strides[:-1]) + (0,) + tuple(d.strides[-1:]))
    return d


def ssm_scan(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None = None, z: Tensor | None = None,
             dt_bias: Tensor | None = None, state=None, lengths=None, return_state: bool = False,
             softplus: bool = True):
    """Selective state space scan of u [B, T, C]: with d = softplus(dt + dt_bias)
    (softplus=False: dt + dt_bias; an A of -inf forgets its state at every position),
        h[c, n] = exp(d A[c, n]) h[c, n] + d u B[t, n],   y = sum_n C[t, n] h[c, n] + D u
    and the result y silu(z), or y without z. dt and z are [B, T, C], A is [C, N]
    (N up to 64), B and C are [B, T, N], or [B, T, G, N] for G groups of channels.

    `state` [B, C, N] (a Tensor or DeviceArray) is h before the first position,
    zeros without one. `lengths` and `return_state` as in causal_conv; the state
    returned is h at each sequence's length."""
    U = _rows(u.data)
    if U.ndim != 3:
        raise ValueError(f"ssm_scan: u must be [B, T, C], not {u.shape}")
    ln = _lengths_of(lengths, U.shape[0], U.shape[1])
    st = _state_of(state)
    opt = [D, z, dt_bias, st]
    args = [_rows(dt.data), _contig(A.data), _maps(B, 2), _maps(C, 2), _contig(D.data) if D is not None else None,
            _rows(z.data) if z is not None else None, _contig(dt_bias.data) if dt_bias is not None else None]
    train = _grad_enabled and any(p is not None and p.requires_grad for p in [u, dt, A, B, C] + opt)
    out, new, kept = K.scan_fwd(U, *args, state=_contig(st.data) if st is not None else None, lengths=ln,
                                softplus=softplus, return_state=return_state, keep=train)

    def bw(g):
        du, ddt, dA, dB, dC, dD, dz, dbias, ds = K.scan_bwd(
            U, *args, kept, _rows(g), ln, softplus, need_dstate=st is not None and st.requires_grad,
            dA_out=grad_out(A), dD_out=grad_out(D) if D is not None else None,
            dbias_out=grad_out(dt_bias) if dt_bias is not None else None)
        grads = [du, ddt, dA, dB.reshape(B.shape), dC.reshape(C.shape)]
        return tuple(grads + [x for p, x in zip(opt, (dD, dz, dbias, ds)) if p is not None])
    t = Tensor._make(out, tuple([u, dt, A, B, C] + [p for p in opt if p is not None]), bw)
    return (t, new) if return_state else t


def ssm_scan_step(u: Tensor, dt: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Tensor | None, z: Tensor | None,
                  dt_bias: Tensor | None, state: DeviceArray, softplus: bool = True) -> Tensor:
    """ssm_scan for one new position per sequence: u, dt and z [B, C], the maps
    [B, N] or [B, G, N]. `state` [B, C, N], contiguous, is updated in place. No
    gradient."""
    y = K.scan_step(_rows(u.data), _rows(dt.data), _contig(A.data), _maps(B, 1), _maps(C, 1),
                    _contig(D.data) if D is not None else None, _rows(z.data) if z is not None else None,
                    _contig(dt_bias.data) if dt_bias is not None else None, state, softplus)
    return Tensor(y)


def cross_attention(q: Tensor, k: Tensor, v: Tensor, lengths=None, scale: float | None = None) -> Tensor:
    """Attention of q [B, H, Tq, D] to another sequence's k, v [B, Hk, Tk, D]: no
    causal mask, any two lengths (one query token included), D up to 128, any
    strides with a contiguous last axis. H is a multiple of Hk; head h reads
    key/value head h // (H // Hk). `lengths` (one per sequence, a host array or an
    Indices) masks the keys from there on, which are not read; a query without
    keys gives 0. `scale` defaults to 1 / sqrt(D)."""
    Q, Kd, V = _rows(q.data), _rows(k.data), _rows(v.data)
    if Q.ndim != 4 or Kd.ndim != 4:
        raise ValueError(f"cross_attention: q and k must be (B, heads, T, D), not {q.shape} and {k.shape}")
    ln = _lengths_of(lengths, Q.shape[0], Kd.shape[2])
    train = _grad_enabled and (q.requires_grad or k.requires_grad or v.requires_grad)
    o, rmax, rsum = K.xattn_fwd(Q, Kd, V, ln, scale, stats=train)

    def bw(g):
        return K.xattn_bwd(Q, Kd, V, o, _rows(g), rmax, rsum, ln, scale)
    return Tensor._make(o, (q, k, v), bw)
