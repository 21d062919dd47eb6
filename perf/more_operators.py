"""Products of a training step that a plain matrix product does not serve, as cases
that can be timed and compared.

Three operators: the loss over a large vocabulary without its logits, with its
gradients; the products of experts that each take some of the rows, with their
gradients; and the orthogonalised update of a set of matrices by Newton-Schulz
steps.

With `own` false, `run` is the plain form: elementary torch operations, the whole
logits, a loop over the experts and over the matrices. With `own` true it makes the
calls a program makes of `dtmi.autograd` and `dtmi.optim`. `exact` is the operators'
definition in float64 by other means (torch's own gradients over pieces of rows, and
the Newton-Schulz steps as a polynomial of the Gram matrix).
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

# the quintic of a Newton-Schulz step: a, b, c of a X + b (X X^T) X + c (X X^T)^2 X
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


# ------------------------------------------------------------------- cases
def listed():
    return [
        # a character model's training step in the type its gradients are checked
        # with: the smallest loss, latency only
        dict(name="loss_char_f64", op="loss", form="train", dtype="float64", rows=512, dim=128, vocab=65),
        # GPT-2-small's head over 8 sequences of its context
        dict(name="loss_gpt2", op="loss", form="train", dtype="float32", rows=8192, dim=768, vocab=50304),
        # padded sequences (no target there), an unpadded vocabulary with a bias, an
        # odd width
        dict(name="loss_padded_odd", op="loss", form="train", dtype="float32", rows=1511, dim=515, vocab=50257,
             ignored=0.3, bias=True),
        # a few continuations scored by their next token, the head being the
        # transposed embedding table: no gradient, a loss for each
        dict(name="loss_score_tied", op="loss", form="score", dtype="float32", rows=5, dim=768, vocab=50304, tied=True),
        # one token each of a serving batch, through two of eight experts
        dict(name="experts_step", op="experts", form="forward", dtype="float32", rows=32, experts=8, dim=768, out=1536),
        # the first product of an experts' layer in training, uneven experts
        dict(name="experts_train", op="experts", form="train", dtype="float32", rows=8192, experts=8, dim=768, out=1536),
        # many small experts of an odd width, some without rows, rows that were
        # dropped at the end
        dict(name="experts_many_odd", op="experts", form="train", dtype="float32", rows=4099, experts=64, dim=384,
             out=501, bias=True, unused=101),
        # few rows in float64
        dict(name="experts_train_f64", op="experts", form="train", dtype="float64", rows=777, experts=5, dim=128,
             out=256, bias=True),
        # the matrices of a 4-layer character model's blocks, as one step updates them
        dict(name="update_char", op="update", dtype="float32", shapes="128x384,128x128,128x512,512x128", layers=4),
        # GPT-2-small's attention projections
        dict(name="update_gpt2", op="update", dtype="float32", shapes="768x2304,768x768", layers=12),
        # one large matrix
        dict(name="ortho_large", op="ortho", dtype="float32", shapes="2048x8192", layers=1),
        # stacked tall matrices of odd sizes, float64
        dict(name="ortho_tall_f64", op="ortho", dtype="float64", shapes="333x201", layers=6, stacked=True),
    ]


def _between(rng, lo, hi):
    """A whole number, spread evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _steps_flops(m, n):
    m, n = min(m, n), max(m, n)
    return 5 * (3 * m * m * n + m ** 3)


def draw(rng):
    op = rng.choice(["loss", "loss", "experts", "experts", "update", "ortho"])
    f64 = rng.random() < 0.25
    c = dict(op=op, dtype="float64" if f64 else "float32")
    most = 60_000_000_000 if f64 else 1_500_000_000_000  # operations
    if op == "loss":
        c["form"] = rng.choice(["train", "train", "score"])
        c.update(dim=_between(rng, 48, 1536), vocab=_between(rng, 65, 60000))
        c["rows"] = _between(rng, 1, max(1, min(8192, most // (6 * c["dim"] * c["vocab"]))))
        c.update(ignored=rng.choice([0.0, 0.0, 0.3]), bias=rng.random() < 0.3, tied=rng.random() < 0.3)
    elif op == "experts":
        c["form"] = rng.choice(["forward", "train", "train"])
        c.update(dim=_between(rng, 48, 1536), out=_between(rng, 48, 2048), experts=_between(rng, 1, 64))
        c["rows"] = _between(rng, 1, max(1, min(16384, most // (6 * c["dim"] * c["out"]))))
        c.update(bias=rng.random() < 0.4, unused=rng.choice([0, 0, c["rows"] // 5]))
    else:
        shapes = []
        for _ in range(1 if op == "ortho" else rng.choice([1, 2, 3])):
            shapes.append((_between(rng, 16, 1600), _between(rng, 16, 1600)))
        total = sum(_steps_flops(m, n) for m, n in shapes)
        c["shapes"] = ",".join(f"{m}x{n}" for m, n in shapes)
        c["layers"] = _between(rng, 1, max(1, min(16, most // total)))
        if op == "ortho":
            c["stacked"] = rng.random() < 0.5
    return c


# ------------------------------------------------------------------ inputs
def _shapes(case):
    one = [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split(",")]
    return [s for _ in range(case["layers"]) for s in one]


def _sizes(case, seed):
    """Rows of each expert: uneven as a router leaves them, one in eight without any."""
    r = random.Random(seed * 7919 + 17)
    E, left = case["experts"], case["rows"] - case.get("unused", 0)
    w = [0.0 if E > 1 and r.random() < 0.125 else r.expovariate(1.0) + 0.2 for _ in range(E)]
    if not sum(w):
        w[0] = 1.0
    edges = [int(left * sum(w[:i + 1]) / sum(w)) for i in range(E)]
    edges[-1] = left
    return [b - a for a, b in zip([0] + edges[:-1], edges)]


def _inputs(case, seed):
    """The case's inputs as torch tensors on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = torch.float64 if case["dtype"] == "float64" else torch.float32

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=dt) * std

    if case["op"] == "loss":
        R, C, V = case["rows"], case["dim"], case["vocab"]
        # normalised activations, weights that spread the logits by about 1.5, frequent
        # and rare targets
        t = {"x": normal(R, C)}
        w = normal(V, C, std=1.5 * C ** -0.5) if case.get("tied") else normal(C, V, std=1.5 * C ** -0.5)
        t["w"] = w.T if case.get("tied") else w
        t["b"] = normal(V, std=0.5) if case.get("bias") else None
        u = torch.rand((R,), generator=g, device="cuda", dtype=torch.float64)
        at = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        drop = torch.rand((R,), generator=g, device="cuda") < case.get("ignored", 0.0)
        t["targets"] = torch.where(drop, -1, at)
        return t
    if case["op"] == "experts":
        R, E, K, N = case["rows"], case["experts"], case["dim"], case["out"]
        t = {"x": normal(R, K), "w": normal(E, K, N, std=K ** -0.5)}
        t["b"] = normal(E, N, std=0.1) if case.get("bias") else None
        if case["form"] == "train":
            t["g"] = normal(R, N)
        t["sizes"] = _sizes(case, seed)
        return t
    # gradients: a few directions that many rows share, and noise of every row
    t = {"g": [], "p": [], "m": []}
    for m, n in _shapes(case):
        def grad():
            return normal(m, 8) @ normal(8, n) * 3e-4 + normal(m, n, std=1e-3)
        t["g"].append(grad())
        if case["op"] == "update":
            t["m"].append(grad() * 5)
            t["p"].append(normal(m, n, std=0.02))
    if case.get("stacked"):
        t["g"] = [torch.stack(t["g"])]
    return t


# ----------------------------------------------------------- the framework's
def _dtmi():
    pkg = str(Path(__file__).resolve().parents[1] / "distributed-training_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    from dtmi import _lib, autograd, device, optim
    _lib.lib()
    return autograd, device, optim


class _Memory:
    """A DeviceArray's memory as torch takes it (no copy; keeps the array alive)."""

    def __init__(self, a):
        self.array = a
        self.__cuda_array_interface__ = {"shape": a.shape, "typestr": a.dtype.str, "data": (a.ptr, False),
                                         "strides": tuple(s * a.itemsize for s in a.strides), "version": 2}


def _tensor(a):
    return torch.as_tensor(_Memory(a), device="cuda")


def _array(t, dev):
    """A DeviceArray with a torch tensor's values and strides."""
    extent = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    a = dev.empty((extent,), str(t.dtype).split(".")[1])
    a = dev.DeviceArray(a.block, tuple(t.shape), a.dtype, 0, t.stride())
    _tensor(a).copy_(t)
    return a


LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def prepare(case, seed):
    torch.cuda.synchronize()
    t = _inputs(case, seed)
    s = {"op": case["op"], "form": case.get("form"), "own": own}
    if not own:
        s.update(t)
        torch.cuda.synchronize()
        return s
    A, dev, O = _dtmi()
    s["A"], s["O"] = A, O
    for k, v in t.items():
        if k in ("targets", "sizes"):
            s[k] = A.Indices(v.cpu().numpy() if torch.is_tensor(v) else v)
        elif isinstance(v, list):
            s[k] = [_array(x, dev) for x in v]
        else:
            s[k] = None if v is None else _array(v, dev)
    torch.cuda.synchronize()  # the arrays were written on torch's stream
    if case["op"] == "update":
        s["opt"] = O.Muon(s["p"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
        for a, m in zip(s["opt"].m, s["m"]):
            a.assign(m)
        torch.cuda.synchronize()
    return s


def _own(s):
    op = s["op"]
    if op == "update":
        s["opt"].step(s["g"])
        return [_tensor(a) for a in s["p"] + s["opt"].m]
    if op == "ortho":
        return [_tensor(a) for a in s["O"].orthogonalize(s["g"])]
    A = s["A"]
    train = s["form"] == "train"
    leaves = [None if s[k] is None else A.Tensor(s[k], requires_grad=train) for k in ("x", "w", "b")]
    if op == "loss":
        y = A.linear_cross_entropy(leaves[0], leaves[1], s["targets"], leaves[2], ignore=-1,
                                   reduction="mean" if train else "none")
    else:
        y = A.expert_linear(leaves[0], leaves[1], s["sizes"], leaves[2])
    if not train:
        return _tensor(y.data)
    y.backward(s.get("g"))
    return [_tensor(y.data)] + [_tensor(x.grad) for x in leaves if x is not None]


# -------------------------------------------------------------- plain forms
def _loss(s):
    x, w, b, t = s["x"], s["w"], s["b"], s["targets"]
    z = torch.matmul(x, w)
    if b is not None:
        z = z + b
    ok = t >= 0
    at = torch.where(ok, t, 0)
    m = z.amax(1, keepdim=True)
    rows = torch.arange(len(t), device="cuda")
    zt = z[rows, at]
    p = torch.exp(z - m)
    total = p.sum(1, keepdim=True)
    l = torch.where(ok, torch.log(total[:, 0]) + m[:, 0] - zt, 0.0)
    if s["form"] != "train":
        return l
    n = ok.sum().clamp(min=1)
    p = p / total
    p[rows, at] -= 1.0
    p = p * (ok[:, None] / n)
    dx, dw = torch.matmul(p, w.T), torch.matmul(x.T, p)
    out = [l.sum() / n, dx, dw]
    return out if b is None else out + [p.sum(0)]


def _experts(s):
    x, w, b, g = s["x"], s["w"], s["b"], s.get("g")
    y = x.new_zeros(x.shape[0], w.shape[2])
    train = s["form"] == "train"
    if train:
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        db = None if b is None else torch.zeros_like(b)
    at = 0
    for e, n in enumerate(s["sizes"]):
        if n == 0:
            continue
        r = slice(at, at + n)
        at += n
        y[r] = torch.matmul(x[r], w[e]) if b is None else torch.matmul(x[r], w[e]) + b[e]
        if train:
            dx[r] = torch.matmul(g[r], w[e].T)
            dw[e] = torch.matmul(x[r].T, g[r])
            if b is not None:
                db[e] = g[r].sum(0)
    if not train:
        return y
    return [y, dx, dw] if b is None else [y, dx, dw, db]


def _newton_schulz(g):
    """[..., m, n]"""
    a, b, c = COEFFICIENTS
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2).contiguous() if tall else g
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + EPS)
    for _ in range(5):
        gram = torch.matmul(x, x.transpose(-1, -2).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return x.transpose(-1, -2).contiguous() if tall else x


def _update(s):
    for p, m, g in zip(s["p"], s["m"], s["g"]):
        m.mul_(MOMENTUM).add_(g)
        o = _newton_schulz(g + MOMENTUM * m)
        rate = LR * math.sqrt(max(1.0, p.shape[1] / p.shape[0]))
        p.mul_(1 - LR * DECAY).sub_(rate * o)
    return s["p"] + s["m"]


def run(state):
    if state["own"]:
        return _own(state)
    if state["op"] == "loss":
        return _loss(state)
    if state["op"] == "experts":
        return _experts(state)
    if state["op"] == "update":
        return _update(state)
    return [_newton_schulz(g) for g in state["g"]]


# ------------------------------------------------------------------- work
def work(case):
    """One pass: inputs read once, outputs written once. A Newton-Schulz step of an m x n
    matrix (m <= n) needs half of X X^T and of its square, which are symmetric."""
    es = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "loss":
        R, C, V = case["rows"], case["dim"], case["vocab"]
        one = R * C + C * V + (V if case.get("bias") else 0)
        if case["form"] == "train":
            return {"bytes": es * 2 * one + 8 * R, "flops": 6 * R * C * V}
        return {"bytes": es * (one + R) + 8 * R, "flops": 2 * R * C * V}
    if case["op"] == "experts":
        R, E, K, N = case["rows"], case["experts"], case["dim"], case["out"]
        used = R - case.get("unused", 0)
        w = min(E, max(1, used)) * K * N
        if case["form"] == "train":
            return {"bytes": es * (2 * R * K + 2 * R * N + w + E * K * N), "flops": 6 * used * K * N}
        return {"bytes": es * (R * K + R * N + w), "flops": 2 * used * K * N}
    n = sum(m * k for m, k in _shapes(case))
    return {"bytes": es * n * (5 if case["op"] == "update" else 2),
            "flops": sum(_steps_flops(m, k) for m, k in _shapes(case))}


# ------------------------------------------------------------------ exact
def _exact_loss(t, case):
    x, w, b, at = t["x"], t["w"].contiguous(), t["b"], t["targets"]
    train = case["form"] == "train"
    count = max(1, int((at >= 0).sum()))
    leaves = [v.clone().requires_grad_(train) for v in (x, w, b) if v is not None]
    losses, grads = [], [torch.zeros_like(v) for v in leaves]
    for lo in range(0, len(x), 1024):
        hi = min(len(x), lo + 1024)
        z = leaves[0][lo:hi] @ leaves[1]
        if b is not None:
            z = z + leaves[2]
        ok = at[lo:hi] >= 0
        l = torch.logsumexp(z, 1) - torch.gather(z, 1, at[lo:hi].clamp(min=0)[:, None])[:, 0]
        l = torch.where(ok, l, torch.zeros_like(l))
        losses.append(l.detach())
        if train:
            for acc, d in zip(grads, torch.autograd.grad(l.sum() / count, leaves)):
                acc += d
    l = torch.cat(losses)
    return [l.sum() / count] + grads if train else l


def _exact_experts(t, case):
    x, w, b, g = t["x"], t["w"], t["b"], t.get("g")
    train = case["form"] == "train"
    leaves = [v.clone().requires_grad_(train) for v in (x, w, b) if v is not None]
    rows = torch.split(leaves[0][:sum(t["sizes"])], t["sizes"])
    parts = [r @ leaves[1][e] + (leaves[2][e] if b is not None else 0.0) for e, r in enumerate(rows)]
    y = torch.cat(parts + [x.new_zeros(case["rows"] - sum(t["sizes"]), case["out"])])
    if not train:
        return y
    return [y.detach(), *torch.autograd.grad(y, leaves, g)]


def _exact_ortho(g):
    """The steps as one polynomial of the Gram matrix: with G = X X^T the step's factor is
    H = a + b G + c G^2, and G becomes H G H."""
    if g.shape[0] > g.shape[1]:
        return _exact_ortho(g.T).T.contiguous()
    a, b, c = COEFFICIENTS
    x = g / (torch.linalg.norm(g) + EPS)
    one = torch.eye(g.shape[0], device="cuda", dtype=torch.float64)
    gram, factor = x @ x.T, one
    for _ in range(5):
        h = a * one + b * gram + c * (gram @ gram)
        gram, factor = h @ gram @ h, h @ factor
    return factor @ x


def exact(case, seed):
    t = {k: [x.double() if torch.is_tensor(x) else x for x in v] if isinstance(v, list)
         else v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    if case["op"] == "loss":
        return _exact_loss(t, case)
    if case["op"] == "experts":
        return _exact_experts(t, case)
    if case["op"] == "ortho":
        if case.get("stacked"):
            return [torch.stack([_exact_ortho(x) for x in t["g"][0]])]
        return [_exact_ortho(x) for x in t["g"]]
    ps, ms = [], []
    for p, m, g in zip(t["p"], t["m"], t["g"]):
        m = MOMENTUM * m + g
        o = _exact_ortho(g + MOMENTUM * m)
        ps.append(p - LR * DECAY * p - LR * max(1.0, p.shape[1] / p.shape[0]) ** 0.5 * o)
        ms.append(m)
    return ps + ms
