"""Cross entropy of a projection and its gradient against the formulas in 64 bits.

What the results may be off follows from the products.  With S = sum_k |x| |w|, a logit may be off by E = 4e-6 S: operands of 22 bits and
the accumulate's truncation make 1e-6 S for pieces of 1024, a chain of K f32 additions sqrt(K) 2^-24 S, 4e-6 S at K = 4500.  A row's
log-sum-exp is off by at most its logits' E, plus roundings of the sum (2e-6) and of the result; exp(z - lse) relatively by 2 E
and the roundings of its argument and of exp (2e-6); a gradient by the sum of what its terms are off, and its own product's 4e-6."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PRODUCT = 4e-6


def tensor(F, t):
    return F.DeviceTensor.from_torch(t)


def make(seed, rows, k, n, layout="stored", bias=False, masked=False, dtype=torch.int64, lead=None, spread=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)
    x = normal(*(lead or (rows,)), k)
    if layout == "stored":
        w = normal(k, n)
    elif layout == "tied":
        w = normal(n, k).t()
    elif layout == "columns":                 # every second column of a wider weight
        w = normal(k, 2 * n)[:, ::2]
    elif layout == "part":                    # a part of a wider weight, off a 16-byte boundary
        w = normal(k, n + 3)[:, 1:n + 1]
    elif layout == "broadcast":               # one column for all classes
        w = normal(k, 1).expand(k, n)
    w = w * (spread / k ** 0.5) if layout in ("stored", "tied") else w.mul_(spread / k ** 0.5) if layout != "broadcast" else w
    targets = torch.randint(0, n, tuple(lead or (rows,)), device="cuda", generator=gen).to(dtype)
    if masked:
        left_out = torch.rand(targets.shape, device="cuda", generator=gen) < 0.3
        left_out.view(-1)[0] = rows > 1
        targets = torch.where(left_out, torch.full_like(targets, -1), targets)
    return x, w, targets, (0.5 * normal(n) if bias else None)


def truth(x, w, targets, bias, reduction, grad):
    """-> values and bounds on their errors, all in 64 bits."""
    k, n = w.shape
    x2, w2, t = x.reshape(-1, k).double(), w.double(), targets.reshape(-1).long()
    z = x2 @ w2 + (0 if bias is None else bias.double())
    size = x2.abs() @ w2.abs()
    e = PRODUCT * size.amax(1) + 2.0 ** -23 * z.abs().amax(1)
    lse = torch.logsumexp(z, 1)
    rows = (t >= 0).nonzero()[:, 0]
    loss, weight = torch.zeros_like(lse), torch.zeros_like(lse)
    loss[rows] = lse[rows] - z[rows, t[rows]]
    off_lse = e + 2e-6 + 2.0 ** -23 * lse.abs()
    off_loss = torch.where(t >= 0, e + off_lse + 2.0 ** -23 * loss.abs(), 0.0)
    weight[rows] = grad.reshape(-1).double().expand(t.numel())[rows] if reduction != "none" else grad.reshape(-1).double()[rows]
    if reduction == "mean":
        weight /= rows.numel()
    p = (z - lse[:, None]).exp()
    d = p.clone()
    d[rows, t[rows]] -= 1
    d *= weight[:, None]
    off_d = p * (2 * e + 2e-6)[:, None] * weight.abs()[:, None] + 2.0 ** -23 * d.abs()
    off_g = off_d + PRODUCT * d.abs()
    tiny = 2.0 ** -40 * float(weight.abs().max())      # products of parts too small for the planes
    values = {"lse": lse, "dx": d @ w2.T, "dw": x2.T @ d, "dbias": d.sum(0)}
    offs = {"lse": off_lse, "dx": off_g @ w2.abs().T + tiny * w2.abs().sum(1), "dw": x2.abs().T @ off_g + tiny * x2.abs().sum(0)[:, None],
            "dbias": off_g.sum(0) + tiny}
    if reduction == "none":
        values["loss"], offs["loss"] = loss, off_loss
    else:
        scale = 1 if reduction == "sum" else max(rows.numel(), 1)
        values["loss"] = loss.sum().reshape(1) / scale
        offs["loss"] = off_loss.sum().reshape(1) / scale + 2.0 ** -24 * values["loss"].abs()
    return values, offs


def close(got, value, off, what):
    got = got.double().reshape(value.shape)
    worst = ((got - value).abs() - off).max() if value.numel() else torch.zeros(())
    assert torch.isfinite(got).all() and float(worst) <= 0, f"{what}: {float((got - value).abs().max())} off, {float(worst)} more than it may be"


def compare(F, x, w, targets, bias, reduction="mean", need=("dx", "dw", "dbias")):
    gen = torch.Generator(device="cuda").manual_seed(5)
    grad = torch.rand(targets.shape if reduction == "none" else (1,), device="cuda", generator=gen) + 0.5
    values, offs = truth(x, w, targets, bias, reduction, grad)
    tb = None if bias is None else tensor(F, bias)
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), targets, tb, reduction=reduction)
    assert lse.shape == tuple(targets.shape) and loss.shape == (tuple(targets.shape) if reduction == "none" else (1,))
    got = F.linear_cross_entropy_backward(tensor(F, grad), tensor(F, x), tensor(F, w), targets, lse, tb, reduction=reduction,
                                          need_dx="dx" in need, need_dw="dw" in need, want_dbias="dbias" in need)
    F.device_status()
    close(lse.torch_view(), values["lse"], offs["lse"], "lse")
    close(loss.torch_view(), values["loss"], offs["loss"], "loss")
    for name, t in zip(("dx", "dw", "dbias"), got):
        if name in need:
            assert t.shape == {"dx": tuple(x.shape), "dw": tuple(w.shape), "dbias": (w.shape[1],)}[name]
            close(t.torch_view(), values[name], offs[name], name)
        else:
            assert t is None
    return loss, lse, got


SIZES = [(1, 1, 1), (1, 1, 2), (1, 16, 1), (2, 3, 5), (1, 64, 32000), (8, 40, 4097), (9, 64, 300), (16, 256, 2048), (17, 33, 65), (32, 64, 96),
         (127, 96, 511), (129, 70, 1025), (256, 256, 256), (300, 513, 1000), (1000, 333, 777), (257, 1030, 2049), (40, 2048, 1500), (520, 64, 9000)]


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("layout", ["stored", "tied"])
def test_loss_and_gradients(F, rows, k, n, layout):
    odd = (rows + k + n) % 2 == 1
    x, w, t, b = make(rows * 7 + n, rows, k, n, layout, bias=odd, masked=not odd, dtype=torch.int32 if odd else torch.int64, spread=2.0)
    compare(F, x, w, t, b)


@pytest.mark.parametrize("piece", ["256", "768"])
@pytest.mark.parametrize("lone", ["0", "1"])
@pytest.mark.parametrize("layout", ["stored", "tied"])
@pytest.mark.parametrize("rows,k,n", [(300, 200, 1000), (257, 130, 2049)])
def test_pieces_of_the_classes(F, monkeypatch, piece, lone, layout, rows, k, n):
    """The backward in pieces, the last one ragged, as many classes and rows make it; with tiles of pairs and of single CTAs."""
    monkeypatch.setenv("MNI_B200_LOSS_PIECE", piece)
    monkeypatch.setenv("MNI_B200_FUSED_LONE", lone)
    compare(F, *make(rows + n, rows, k, n, layout, bias=True, masked=True, spread=2.0))


@pytest.mark.parametrize("rows,k,n", [(4096, 8, 12), (4097, 8, 12), (50, 64, 128), (50, 65, 129), (30, 250, 30), (30, 260, 30), (20, 8, 1024), (20, 9, 1025)])
def test_few_short_rows(F, rows, k, n):
    """Both sides of the limits of the kernel that makes logits and what becomes of them in one launch."""
    compare(F, *make(rows + k, rows, k, n, bias=True, masked=True))


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("rows,k,n", [(5, 32, 100), (70, 48, 333), (600, 128, 1500)])
def test_reductions(F, reduction, rows, k, n):
    compare(F, *make(3, rows, k, n, bias=True, masked=True), reduction=reduction)


@pytest.mark.parametrize("layout", ["columns", "part", "broadcast"])
@pytest.mark.parametrize("rows,k,n", [(4, 24, 60), (300, 200, 700)])
def test_weights_of_any_stride(F, layout, rows, k, n):
    compare(F, *make(9, rows, k, n, layout, bias=True))


@pytest.mark.parametrize("rows", [6, 210])
def test_features_of_any_stride(F, rows):
    """Leading dims that merge, that do not, a column stride, one row for all."""
    x, w, t, _ = make(4, rows, 52, 500, lead=(rows // 2, 2))
    compare(F, x, w, t, None)
    other = torch.randn(2, rows // 2, 52, device="cuda").transpose(0, 1)
    compare(F, other, w, t, None)
    compare(F, torch.randn(rows // 2, 2, 104, device="cuda")[:, :, ::2], w, t, None)
    compare(F, torch.randn(rows // 2, 1, 52, device="cuda").expand(rows // 2, 2, 52), w, t, None)
    compare(F, torch.randn(1, 1, 52, device="cuda").expand(rows // 2, 2, 52), w, t, None)


@pytest.mark.parametrize("need", [("dx",), ("dw",), ("dbias",), ("dx", "dw"), ()])
@pytest.mark.parametrize("layout", ["stored", "tied"])
def test_gradients_that_are_wanted(F, need, layout):
    for rows in (7, 300):
        compare(F, *make(8, rows, 64, 600, layout, bias=True), need=need)


@pytest.mark.parametrize("rows,k,n", [(6, 32, 90), (300, 96, 800)])
def test_rows_left_out(F, rows, k, n):
    """Whatever they hold: no loss, no gradient, nothing in the gradients of the others."""
    x, w, t, b = make(2, rows, k, n, bias=True, masked=True)
    clean = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b))
    grad = tensor(F, torch.ones(1, device="cuda"))
    want = F.linear_cross_entropy_backward(grad, tensor(F, x), tensor(F, w), t, clean[1], tensor(F, b), want_dbias=True)
    dirty = x.clone()
    dirty[t < 0] = float("nan")
    dirty[(t < 0).nonzero()[0]] = float("inf")
    loss, lse = F.linear_cross_entropy(tensor(F, dirty), tensor(F, w), t, tensor(F, b))
    got = F.linear_cross_entropy_backward(grad, tensor(F, dirty), tensor(F, w), t, lse, tensor(F, b), want_dbias=True)
    F.device_status()
    assert abs(float(loss.numpy()[0]) - float(clean[0].numpy()[0])) <= 2e-6 * float(clean[0].numpy()[0])
    for g, v in zip(got, want):
        assert np.isfinite(g.numpy()).all()
        assert np.abs(g.numpy() - v.numpy()).max() <= 2e-5 * np.abs(v.numpy()).max()
    assert not got[0].torch_view()[t < 0].any()
    # no row at all
    none = torch.full_like(t, -7)
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), none, tensor(F, b))
    got = F.linear_cross_entropy_backward(grad, tensor(F, x), tensor(F, w), none, lse, tensor(F, b), want_dbias=True, reduction="sum")
    assert np.isnan(loss.numpy()).all() and not any(g.numpy().any() for g in got)
    assert float(F.linear_cross_entropy(tensor(F, x), tensor(F, w), none, reduction="sum")[0].numpy()[0]) == 0.0


@pytest.mark.parametrize("rows,k,n", [(5, 32, 90), (300, 96, 800)])
def test_a_target_that_is_no_class_shows(F, rows, k, n):
    x, w, t, _ = make(2, rows, k, n)
    t[2] = n
    t[3] = 2 ** 40
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, reduction="none")
    bad = np.isnan(loss.numpy())
    assert bad[2] and bad[3] and bad.sum() == 2 and np.isfinite(lse.numpy()).all()
    dx, dw = F.linear_cross_entropy_backward(tensor(F, torch.ones(rows, device="cuda")), tensor(F, x), tensor(F, w), t, lse, reduction="none")
    F.device_status()
    bad = np.isnan(dx.numpy()).all(1)
    assert bad[2] and bad[3] and bad.sum() == 2 and np.isnan(dw.numpy()).all()


@pytest.mark.parametrize("rows,k,n", [(5, 16, 70), (200, 48, 5000)])
def test_classes_masked_by_the_bias(F, rows, k, n):
    """-inf and the lowest f32 leave classes out, whole stretches of them; of a row that has no class left the result is as log(0) makes it."""
    x, w, t, b = make(6, rows, k, n, bias=True)
    for lowest in (float("-inf"), torch.finfo(torch.float32).min):
        b2 = b.clone()
        b2[: n // 2 + 3] = lowest
        t2 = t % (n - n // 2 - 3) + n // 2 + 3
        kept = slice(n // 2 + 3, n)
        loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t2, tensor(F, b2))
        grads = F.linear_cross_entropy_backward(tensor(F, torch.ones(1, device="cuda")), tensor(F, x), tensor(F, w), t2, lse, tensor(F, b2),
                                                want_dbias=True)
        values, offs = truth(x, w[:, kept], t2 - (n // 2 + 3), b[kept], "mean", torch.ones(1, device="cuda"))
        close(loss.torch_view(), values["loss"], offs["loss"], "loss")
        close(lse.torch_view(), values["lse"], offs["lse"], "lse")
        close(grads[0].torch_view(), values["dx"], offs["dx"], "dx")
        close(grads[1].torch_view()[:, kept], values["dw"], offs["dw"], "dw")
        assert not grads[1].torch_view()[:, : n // 2 + 3].any() and not grads[2].torch_view()[: n // 2 + 3].any()
    b3 = torch.full_like(b, float("-inf"))
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b3), reduction="none")
    F.device_status()
    assert (lse.numpy() == -np.inf).all() and np.isnan(loss.numpy()).all()


@pytest.mark.parametrize("rows,k,n", [(5, 16, 70), (200, 48, 3000)])
def test_large_logits(F, rows, k, n):
    """Logits of some thousands: nothing overflows, and what is one class's is one."""
    x, w, t, _ = make(6, rows, k, n, spread=3000.0)
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, reduction="none")
    dx, dw = F.linear_cross_entropy_backward(tensor(F, torch.ones(rows, device="cuda")), tensor(F, x), tensor(F, w), t, lse, reduction="none")
    F.device_status()
    z = x.double() @ w.double()
    e = PRODUCT * (x.double().abs() @ w.double().abs()).amax(1) + 2.0 ** -22 * z.abs().amax(1)
    assert ((lse.torch_view().double() - torch.logsumexp(z, 1)).abs() <= e + 1e-6).all()
    assert np.isfinite(loss.numpy()).all() and np.isfinite(dx.numpy()).all() and np.isfinite(dw.numpy()).all()


def test_infinite_and_nan_logits(F):
    x, w, t, _ = make(6, 40, 32, 500)
    x[3, 0] = float("nan")
    x[5] = 0.0
    x[5, 1] = float("inf")
    w[1] = 1.0
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, reduction="none")
    F.device_status()
    others = [r for r in range(40) if r not in (3, 5)]
    assert np.isnan(lse.numpy()[3]) and not np.isfinite(lse.numpy()[5]) and np.isfinite(loss.numpy()[others]).all()


def test_no_rows(F):
    x, w = torch.empty(0, 8, device="cuda"), torch.randn(8, 12, device="cuda")
    t = torch.empty(0, dtype=torch.int64, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, reduction=reduction)
        grad = tensor(F, torch.ones(0 if reduction == "none" else 1, device="cuda"))
        dx, dw, dbias = F.linear_cross_entropy_backward(grad, tensor(F, x), tensor(F, w), t, lse, reduction=reduction, want_dbias=True)
        assert dx.shape == (0, 8) and not dw.numpy().any() and not dbias.numpy().any()
        if reduction != "none":
            value = loss.numpy()[0]
            assert value == 0.0 if reduction == "sum" else np.isnan(value)


@pytest.mark.parametrize("rows,k,n", [(6, 20, 33), (6, 64, 2000), (300, 101, 1003), (260, 256, 1024)])
@pytest.mark.parametrize("layout", ["stored", "tied"])
@pytest.mark.parametrize("accumulate", [False, True])
def test_outputs_stay_in_their_place(F, rows, k, n, layout, accumulate):
    """Into buffers between guard zones; accumulated into what is there, or overwriting it."""
    from conftest import Guarded
    from framework_b200 import _lib
    x, w, t, b = make(1, rows, k, n, layout, bias=True, masked=True)
    _, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b))
    grad = tensor(F, torch.ones(1, device="cuda"))
    plain = F.linear_cross_entropy_backward(grad, tensor(F, x), tensor(F, w), t, lse, tensor(F, b), want_dbias=True)
    base = [np.random.default_rng(i).standard_normal(s).astype(np.float32) for i, s in enumerate([(rows, k), (n, k) if layout == "tied" else (k, n), (n,)])]
    outs = [Guarded(F, v.shape, v if accumulate else None) for v in base]
    dw = outs[1].tensor.permute([1, 0]) if layout == "tied" else outs[1].tensor
    flags = (_lib.ACCUMULATE_DA | _lib.ACCUMULATE_DB | _lib.ACCUMULATE_DBIAS) if accumulate else 0
    got = F.linear_cross_entropy_backward(grad, tensor(F, x), tensor(F, w), t, lse, tensor(F, b), want_dbias=True, flags=flags,
                                          dx=outs[0].tensor, dw=dw, dbias=outs[2].tensor)
    F.device_status()
    for i, o in enumerate(outs):
        o.check(f"output {i}")
        want = plain[i].numpy()
        if accumulate:
            want = want + (base[i].T if i == 1 and layout == "tied" else base[i])
        assert np.abs(got[i].numpy() - want).max() <= 2e-6 * max(1.0, np.abs(want).max())


@pytest.mark.parametrize("rows,k,n", [(4, 48, 700), (300, 128, 3000)])
def test_the_gradient_is_the_derivative(F, rows, k, n):
    """Central differences of the operator's own loss, along its gradient and a random direction.  A sum over rows is off by 2e-6 a row
    or less, so a difference quotient by that over h, and by h^2 / 6 of a third derivative, which is below one a row for steps
    that change no logit by more than one."""
    x, w, t, b = make(12, rows, k, n, bias=True)
    def total(x, w, b):
        return float(F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b), reduction="none")[0].torch_view().double().sum())
    _, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b), reduction="sum")
    dx, dw, db = F.linear_cross_entropy_backward(tensor(F, torch.ones(1, device="cuda")), tensor(F, x), tensor(F, w), t, lse, tensor(F, b),
                                                 reduction="sum", want_dbias=True)
    h = 0.05
    gen = torch.Generator(device="cuda").manual_seed(1)
    for which, g in enumerate((dx, dw, db)):
        base = (x, w, b)[which]
        v = torch.randn(base.shape, device="cuda", generator=gen)
        v = (v / v.norm() + g.torch_view() / g.torch_view().norm()) / 2
        args = [x, w, b]
        ends = []
        for sign in (1, -1):
            args[which] = base + sign * h * v
            ends.append(total(*args))
        want = (ends[0] - ends[1]) / (2 * h)
        got = float((g.torch_view().double() * v.double()).sum())
        assert abs(got - want) <= rows * (2e-6 / h + h * h / 6), (which, got, want)


@pytest.mark.parametrize("rows,k,n", [(4, 256, 3000), (300, 128, 3000)])
def test_captured_and_replayed(F, rows, k, n):
    """A graph takes the values of the moment, on its own stream, with eager calls between."""
    x, w, t, b = make(1, rows, k, n, bias=True, masked=True)
    grad = torch.ones(1, device="cuda")
    tx, tw, tb, tg = (tensor(F, v) for v in (x, w, b, grad))

    def step():
        loss, lse = F.linear_cross_entropy(tx, tw, t, tb)
        return (loss, lse) + tuple(F.linear_cross_entropy_backward(tg, tx, tw, t, lse, tb, want_dbias=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    for seed in (21, 22):
        fresh = make(seed, rows, k, n, bias=True, masked=True)
        for mine, new in zip((x, w, t, b), fresh):
            mine.copy_(new)
        eager = [v.numpy() for v in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(out, eager):
            assert np.array_equal(a.numpy(), e)
    F.device_status()


def test_the_same_call_gives_the_same_bits(F):
    for rows, k, n in ((8, 512, 5000), (500, 256, 5000)):
        x, w, t, b = make(1, rows, k, n, bias=True, masked=True)
        runs = []
        for _ in range(3):
            loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b))
            runs.append([v.numpy() for v in (loss, lse, *F.linear_cross_entropy_backward(tensor(F, torch.ones(1, device="cuda")), tensor(F, x),
                                                                                         tensor(F, w), t, lse, tensor(F, b), want_dbias=True))])
        for other in runs[1:]:
            for a, e in zip(other, runs[0]):
                assert np.array_equal(a, e)


def test_tensors_are_checked_before_anything_runs(F):
    from framework_b200 import DeviceTensor, ops

    def t(*shape):
        n = 1
        for s in shape:
            n *= s
        return DeviceTensor(torch.empty(max(n, 1), device="cuda"), shape)
    good = torch.zeros(6, dtype=torch.int64, device="cuda")
    before = F.launch_count()
    for args, error in [((t(6, 8), t(8, 10), good.cpu()), ValueError), ((t(6, 8), t(9, 10), good), ValueError), ((t(8), t(8, 10), good), ValueError), ((t(6, 8), t(8, 10), good[:5]), ValueError),
                        ((t(6, 8), t(8, 10), good.float()), TypeError), ((t(6, 8), t(8, 10), [0] * 6), TypeError), ((None, t(8, 10), good), TypeError),
                        ((t(6, 8), t(8, 10), good, t(9)), ValueError), ((t(2, 3, 8), t(8, 10), good), ValueError)]:
        with pytest.raises(error):
            ops.linear_cross_entropy(*args)
    with pytest.raises(ValueError, match="lse"):
        ops.linear_cross_entropy_backward(t(1), t(6, 8), t(8, 10), good, t(5))
    with pytest.raises(ValueError, match="grad"):
        ops.linear_cross_entropy_backward(t(1), t(6, 8), t(8, 10), good, t(6), reduction="none")
    with pytest.raises(ValueError, match="at least 2D"):
        ops.orthogonalize(t(6))
    with pytest.raises(ValueError, match="same shape"):
        ops.muon_step([t(4, 5)], [t(4, 5)], [t(5, 4)], lr=0.1)
    with pytest.raises(ValueError, match="same length"):
        ops.muon_step([t(4, 5)], [], [t(5, 4)], lr=0.1)
    with pytest.raises(ValueError, match="contiguous"):
        ops.muon_step([t(4, 5).permute([1, 0])], [t(5, 4)], [t(5, 4)], lr=0.1)
    with pytest.raises(ValueError, match="matrices"):
        ops.muon_step([t(4)], [t(4)], [t(4)], lr=0.1)
    assert F.launch_count() == before
