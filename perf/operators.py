"""The loss at the end of a model and the update of its matrices, as cases that can be timed.

`linear_cross_entropy` is the softmax cross entropy of x.w (+ bias), whose logits are wanted for nothing else, and its
gradient; `orthogonalize` makes a matrix's singular values nearly one by five Newton-Schulz steps, and `muon_step` updates a
model's matrices with it.  Everything is f32, targets are whole numbers, one below zero leaves its row out.

With `own` false `run` computes them from products, exponentials and sums of whole matrices; with `own` true it makes the
package's calls.  `exact` says what comes out in 64 bits.
"""
import math

import torch

own = False

STEPS, A, B, C, EPS = 5, 3.4445, -4.7750, 2.0315, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01

# Upper ends of the drawn sizes: no drawn case costs more than the largest listed one of its kind.
MAX_LOSS_FLOPS, MAX_STEP_FLOPS, MAX_UPDATE_FLOPS = 0.15e12, 2.5e12, 1.3e12
MAX_WEIGHT, MAX_LOGITS = 6.0e7, 4.2e8


def listed():
    return [
        # The score of a few tokens against a vocabulary: bound by reading the weight once.
        {"name": "loss-8-rows", "kind": "loss", "rows": 8, "k": 1024, "n": 32000, "tied": False, "bias": False,
         "masked": False, "reduction": "none"},
        # Evaluating a language model whose output weight is the embedding, stored [vocabulary, features]; padded batch.
        {"name": "loss-evaluation", "kind": "loss", "rows": 2048, "k": 768, "n": 32768, "tied": True, "bias": False,
         "masked": True, "reduction": "mean"},
        # The last layer of a small classifier, trained on a small batch: launches and host work.
        {"name": "step-classifier", "kind": "step", "rows": 32, "k": 64, "n": 96, "tied": False, "bias": True,
         "masked": False, "reduction": "mean"},
        # Sizes as data sets have them; no row of the weight is aligned.
        {"name": "step-ragged", "kind": "step", "rows": 1000, "k": 333, "n": 7777, "tied": False, "bias": True,
         "masked": True, "reduction": "mean"},
        # One short sequence against a large vocabulary: the weight and its gradient outweigh the products.
        {"name": "step-short", "kind": "step", "rows": 128, "k": 1024, "n": 32000, "tied": False, "bias": False,
         "masked": False, "reduction": "sum"},
        # The head of a language model, trained on a batch of sequences.
        {"name": "step-head", "kind": "step", "rows": 4096, "k": 1024, "n": 32000, "tied": False, "bias": False,
         "masked": False, "reduction": "mean"},
        # The largest: a long batch, a vocabulary as tokenisers leave it, tied weight, padding.
        {"name": "step-large", "kind": "step", "rows": 8192, "k": 1024, "n": 50257, "tied": True, "bias": False,
         "masked": True, "reduction": "mean"},
        # A matrix of a small network: fifteen dependent products that fill no SM.
        {"name": "orthogonalize-small", "kind": "orthogonalize", "batch": 1, "rows": 64, "cols": 32},
        # One square matrix of a transformer.
        {"name": "orthogonalize-768", "kind": "orthogonalize", "batch": 1, "rows": 768, "cols": 768},
        # Taller than wide, odd in both.
        {"name": "orthogonalize-ragged", "kind": "orthogonalize", "batch": 3, "rows": 1001, "cols": 333},
        # The matrices of a small transformer: four square ones a layer and the two of the MLP.
        {"name": "muon-model", "kind": "muon", "layers": 5, "c": 512, "f": 2048},
        # The largest: layers of transformer size, one of them.
        {"name": "muon-large", "kind": "muon", "layers": 1, "c": 2048, "f": 8192},
    ]


# --------------------------------------------------------------------------- drawn cases
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Spread over the logarithm of [lo, hi]; half of them round (multiples of 64, or of 8 below 128), half as they come."""
    v = _log_int(rng, lo, hi)
    if rng.random() < 0.5:
        unit = 64 if v >= 128 else 8
        v = max(unit, (v + unit // 2) // unit * unit)
    return max(lo, min(hi, v))


def _fit(sizes, cost, limit):
    """Halves the largest of `sizes` until cost(sizes) is within limit."""
    while cost(sizes) > limit:
        i = max(range(len(sizes)), key=lambda j: sizes[j])
        sizes[i] = max(1, (sizes[i] + 1) // 2)
    return sizes


def draw(rng):
    kind = rng.choice(["loss", "step", "step", "orthogonalize", "muon"])
    if kind in ("loss", "step"):
        s = [_size(rng, 1, 8192), _size(rng, 16, 4096), _size(rng, 32, 65536)]
        _fit(s, lambda v: (2.0 if kind == "loss" else 6.0) * v[0] * v[1] * v[2],
             MAX_LOSS_FLOPS if kind == "loss" else MAX_STEP_FLOPS)
        _fit(s, lambda v: v[1] * v[2], MAX_WEIGHT)
        _fit(s, lambda v: v[0] * v[2], MAX_LOGITS)
        return {"kind": kind, "rows": s[0], "k": s[1], "n": s[2], "tied": rng.random() < 0.4, "bias": rng.random() < 0.3,
                "masked": s[0] >= 16 and rng.random() < 0.5, "reduction": rng.choice(["none", "sum", "mean", "mean"])}
    if kind == "orthogonalize":
        s = [_size(rng, 8, 4096), _size(rng, 8, 4096)]
        batch = 1 if rng.random() < 0.5 else _log_int(rng, 2, 16)
        _fit(s, lambda v: batch * _newton_schulz_flops(*v), MAX_UPDATE_FLOPS)
        return {"kind": kind, "batch": batch, "rows": s[0], "cols": s[1]}
    layers, c = rng.randint(1, 5), _size(rng, 32, 1536)
    while layers * sum(_newton_schulz_flops(*s) for s in _matrices({"layers": 1, "c": c, "f": 4 * c})) > MAX_UPDATE_FLOPS:
        c = (c + 1) // 2
    return {"kind": "muon", "layers": layers, "c": c, "f": 4 * c + rng.choice([0, 0, -3, 5])}


def _matrices(case):
    c, f = case["c"], case["f"]
    return [(c, c), (c, c), (c, c), (c, c), (c, f), (f, c)] * case["layers"]


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    state = {"case": case}
    if case["kind"] in ("loss", "step"):
        rows, k, n = case["rows"], case["k"], case["n"]
        # a weight of small numbers, features that lean towards the class they belong to, as after some training
        stored = normal(n, k) if case["tied"] else normal(k, n)
        stored *= 0.64 / math.sqrt(k)
        w = stored.t() if case["tied"] else stored
        targets = torch.randint(0, n, (rows,), device="cuda", generator=gen)
        x = normal(rows, k) + 8.0 * (w[:, targets] / 0.64).t()
        if case["masked"]:
            targets = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.15, torch.full_like(targets, -1), targets)
            targets[0] = 0
        bias = 0.3 * normal(n) if case["bias"] else None
        weights = torch.rand(rows, device="cuda", generator=gen) + 0.5 if case["reduction"] == "none" else torch.ones(1, device="cuda")
        state.update(x=x, w=w, bias=bias, targets=targets, grad=weights)
    elif case["kind"] == "orthogonalize":
        state["g"] = torch.stack([_gradient(normal, case["rows"], case["cols"]) for _ in range(case["batch"])])
    else:
        shapes = _matrices(case)
        state["params"] = [normal(*s) / math.sqrt(s[0]) for s in shapes]
        state["momenta"] = [_gradient(normal, *s) for s in shapes]
        state["grads"] = [_gradient(normal, *s) for s in shapes]
    if own:
        _wrap(state)
    return state


def _gradient(normal, rows, cols):
    """A few strong directions above noise, as the gradients of a layer have them."""
    r = min(rows, cols, 16)
    return 1e-3 * (normal(rows, r) @ normal(r, cols) / r + 0.2 * normal(rows, cols))


def _wrap(state):
    """The package's tensors over the same memory: what its user has in hand."""
    from framework_b200 import DeviceTensor
    for name, value in list(state.items()):
        if isinstance(value, torch.Tensor) and value.dtype == torch.float32:
            state["t_" + name] = DeviceTensor.from_torch(value)
        elif isinstance(value, list):
            state["t_" + name] = [DeviceTensor.from_torch(v) for v in value]
        elif value is None:
            state["t_" + name] = None


# --------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["kind"] in ("loss", "step"):
        return _own_loss(state, case) if own else _plain_loss(state, case)
    if case["kind"] == "orthogonalize":
        if own:
            import framework_b200 as F
            return F.orthogonalize(state["t_g"], steps=STEPS, coefficients=(A, B, C), eps=EPS).torch_view()
        return _plain_orthogonalize(state["g"])
    if own:
        import framework_b200 as F
        F.muon_step(state["t_params"], state["t_momenta"], state["t_grads"], lr=LR, momentum=MOMENTUM, nesterov=True,
                    weight_decay=DECAY, steps=STEPS, coefficients=(A, B, C), eps=EPS, scale="shape")
    else:
        _ = [_plain_update(p, m, g) for p, m, g in zip(state["params"], state["momenta"], state["grads"])]
    return {"params": state["params"], "momenta": state["momenta"]}


def _own_loss(state, case):
    import framework_b200 as F
    x, w, bias, targets = state["t_x"], state["t_w"], state["t_bias"], state["targets"]
    loss, lse = F.linear_cross_entropy(x, w, targets, bias, reduction=case["reduction"])
    out = {"loss": loss.torch_view(), "lse": lse.torch_view()}
    if case["kind"] == "step":
        grads = F.linear_cross_entropy_backward(state["t_grad"], x, w, targets, lse, bias, reduction=case["reduction"],
                                                want_dbias=bias is not None)
        out.update({name: t.torch_view() for name, t in zip(("dx", "dw", "dbias"), grads)})
    return out


def _plain_loss(state, case):
    x, w, bias, targets, grad = (state[n] for n in ("x", "w", "bias", "targets", "grad"))
    kept = targets >= 0
    index = targets.clamp(min=0)[:, None]
    z = x @ w
    if bias is not None:
        z += bias
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    each = torch.where(kept, (lse - z.gather(1, index))[:, 0], 0.0)
    count = kept.sum()
    loss = each if case["reduction"] == "none" else each.sum(dtype=torch.float64).reshape(1)
    if case["reduction"] == "mean":
        loss = loss / count
    out = {"loss": loss.float(), "lse": lse[:, 0]}
    if case["kind"] == "step":
        g = torch.where(kept, grad / count if case["reduction"] == "mean" else grad, 0.0)
        d = torch.exp(z - lse)
        d.scatter_add_(1, index, torch.full_like(lse, -1.0))
        d *= g[:, None]
        out["dx"] = d @ w.t()
        # the gradient of a tied weight has the weight's logical shape, [features, classes]
        out["dw"] = x.t() @ d
        if bias is not None:
            out["dbias"] = d.sum(0)
    return out


def _plain_orthogonalize(g):
    tall = g.shape[-2] > g.shape[-1]
    x = g.mT if tall else g
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().float()
    x = x / (norm + EPS)
    for _ in range(STEPS):
        a = x @ x.mT
        x = A * x + (B * a + C * (a @ a)) @ x
    return x.mT if tall else x


def _plain_update(p, m, g):
    m.mul_(MOMENTUM).add_(g)
    o = _plain_orthogonalize(g + MOMENTUM * m)
    p.mul_(1.0 - LR * DECAY).sub_(o, alpha=LR * math.sqrt(max(1.0, p.shape[1] / p.shape[0])))


# --------------------------------------------------------------------------- cost and truth
def _newton_schulz_flops(rows, cols):
    """Of the five steps: X X^T and its square, symmetric both, and one product with X."""
    m, n = float(min(rows, cols)), float(max(rows, cols))
    return STEPS * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    if case["kind"] in ("loss", "step"):
        m, k, n = float(case["rows"]), float(case["k"]), float(case["n"])
        bias = n if case["bias"] else 0.0
        read = 4 * (m * k + k * n + bias) + 8 * m
        if case["kind"] == "loss":
            return {"bytes": read + 8 * m, "flops": 2.0 * m * n * k}
        return {"bytes": read + 8 * m + 4 * (m * k + k * n + bias), "flops": 6.0 * m * n * k}
    if case["kind"] == "orthogonalize":
        r, c = case["rows"], case["cols"]
        return {"bytes": 8.0 * case["batch"] * r * c, "flops": case["batch"] * _newton_schulz_flops(r, c)}
    shapes = _matrices(case)
    return {"bytes": 20.0 * sum(r * c for r, c in shapes), "flops": sum(_newton_schulz_flops(r, c) for r, c in shapes)}


def exact(case, seed):
    """From the definitions, in 64 bits: log-sum-exp and one-hot targets; the polynomial of each step applied as one matrix."""
    s = prepare(case, seed)
    if case["kind"] == "orthogonalize":
        return _exact_orthogonalize(s["g"].double())
    if case["kind"] == "muon":
        out = {"params": [], "momenta": []}
        for p, m, g in zip(s["params"], s["momenta"], s["grads"]):
            m = MOMENTUM * m.double() + g.double()
            shape = max(1.0, p.shape[1] / p.shape[0]) ** 0.5
            out["momenta"].append(m)
            out["params"].append((1.0 - LR * DECAY) * p.double() - LR * shape * _exact_orthogonalize(g.double() + MOMENTUM * m))
        return out
    x, w, t = s["x"].double(), s["w"].double(), s["targets"]
    z = torch.addmm(s["bias"].double(), x, w) if s["bias"] is not None else x @ w
    lse = torch.logsumexp(z, 1)
    rows = torch.nonzero(t >= 0)[:, 0]
    each = torch.zeros_like(lse)
    each[rows] = lse[rows] - z[rows, t[rows]]
    weight = torch.zeros_like(lse)
    weight[rows] = 1.0 / rows.numel() if case["reduction"] == "mean" else 1.0
    out = {"loss": each if case["reduction"] == "none" else (each * weight).sum().reshape(1), "lse": lse}
    if case["kind"] == "step":
        d = (z - lse[:, None]).exp_()
        d[rows, t[rows]] -= 1.0
        d *= (weight * s["grad"].double())[:, None]
        out.update(dx=d @ w.T, dw=x.T @ d)
        if s["bias"] is not None:
            out["dbias"] = d.sum(0)
    return out


def _exact_orthogonalize(g):
    x = g / (torch.linalg.matrix_norm(g, keepdim=True) + EPS)
    tall = x.shape[-2] > x.shape[-1]
    eye = torch.eye(min(x.shape[-2:]), dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        y = x.mT @ x if tall else x @ x.mT
        q = A * eye + y @ (B * eye + C * y)
        x = x @ q if tall else q @ x
    return x
