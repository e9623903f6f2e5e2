"""Cross entropy of a projection where it is computed from 16-bit planes (more than 8 rows and 2^23 multiply-adds), against 64 bits.

What a product is off, relative to the sum S of its terms' sizes: f16 planes keep 22 bits of each operand (2^-23 each) and leave out lo * lo
(2^-22 at most); three bf16 planes drop what is below 2^-23 of each operand and the two products of 2^-7 by 2^-15 (2^-21); the tensor core's
accumulate truncates, 7.5e-10 an element, over 512 elements, and pieces of 512 are added in f32.  Gradients d of logits are held
at 2^14 in f16: beside the 22 bits there is an absolute 2^-51 of what lies below lo's last bit, and as much again where lo * lo is left out of
small ones, 2^-50 of a row's weight together."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = 2.0 ** -24
SMALLEST = 2.0 ** -50


def product(k, wide=False):
    operands = 2 * 2.0 ** -23 + 2.0 ** -21 if wide else 2 * 2.0 ** -23 + 2.0 ** -22
    return operands + min(k, 512) * 7.5e-10 + (k / 512 + 2) * HALF_STEP


def tensor(F, t):
    return F.DeviceTensor.from_torch(t)


def truth(x, w, t, bias, weight, wide=False):
    """Rows' lse and loss, dx, dw, dbias for rows weighted by `weight` (0: left out), and how far each may be off."""
    rows, (k, n) = x.shape[0], w.shape
    x, w = x.double(), w.double()
    z = x @ w + (0 if bias is None else bias.double())
    lse = torch.logsumexp(z, 1)
    off_z = product(k, wide) * (x.abs() @ w.abs()) + 2 * HALF_STEP * z.abs()
    # a sum of exponentials: of each its argument's rounding and 2 ulp; the additions of a stretch, of stretches and the logarithm
    off_lse = off_z.amax(1) + 2e-6 + 2 * HALF_STEP * lse.abs()
    at = torch.arange(rows, device=x.device)
    loss = lse - z[at, t.clamp(min=0)]
    off_loss = off_z[at, t.clamp(min=0)] + off_lse + HALF_STEP * loss.abs()
    u = z - lse[:, None]
    p = u.exp()
    off = p * torch.expm1(off_z + off_lse[:, None] + 2 * HALF_STEP * u.abs() + 1e-6) + SMALLEST
    d = p
    d[at, t.clamp(min=0)] -= 1
    off += 2.0 ** -22 * d.abs()
    d *= weight[:, None]
    off = off * weight.abs()[:, None] + 2 * HALF_STEP * d.abs()
    values = {"lse": lse, "loss": loss, "dx": d @ w.T, "dw": x.T @ d, "dbias": d.sum(0)}
    offs = {"lse": off_lse, "loss": off_loss, "dx": off @ w.abs().T + product(n, wide) * (d.abs() @ w.abs().T),
            "dw": x.abs().T @ off + product(rows, wide) * (x.abs().T @ d.abs()), "dbias": off.sum(0) + (rows / 32 + 64) * HALF_STEP * d.abs().sum(0)}
    return values, offs


def step(F, x, w, t, bias, reduction, grad):
    tb = None if bias is None else tensor(F, bias)
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tb, reduction=reduction)
    dx, dw, dbias = F.linear_cross_entropy_backward(tensor(F, grad), tensor(F, x), tensor(F, w), t, lse, tb, reduction=reduction, want_dbias=True)
    F.device_status()
    return {name: v.torch_view() for name, v in (("loss", loss), ("lse", lse), ("dx", dx), ("dw", dw), ("dbias", dbias))}


def close(got, values, offs, names=("loss", "lse", "dx", "dw", "dbias"), rows=slice(None)):
    for name in names:
        part = rows if name in ("loss", "lse", "dx") else slice(None)
        far = (got[name].double().reshape(values[name].shape) - values[name]).abs()[part]
        may = offs[name][part]
        assert bool((far <= may).all()), f"{name}: {float(far.max())} off, {float((far / may).nan_to_num().max())} times what it may be"


def make(seed, rows, k, n):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, k, device="cuda", generator=gen)
    w = torch.randn(k, n, device="cuda", generator=gen) * (1.5 / k ** 0.5)
    return gen, x, w, torch.randint(0, n, (rows,), device="cuda", generator=gen)


@pytest.mark.parametrize("lone", ["0", "1"])
@pytest.mark.parametrize("rows,k,n", [(9, 300, 9000), (300, 64, 2000), (130, 1100, 700), (700, 33, 1001), (64, 40, 9000)])
def test_within_what_planes_keep(F, monkeypatch, rows, k, n, lone):
    monkeypatch.setenv("MNI_B200_FUSED_LONE", lone)
    gen, x, w, t = make(rows, rows, k, n)
    bias = 0.5 * torch.randn(n, device="cuda", generator=gen)
    grad = torch.rand(rows, device="cuda", generator=gen) + 0.5
    close(step(F, x, w, t, bias, "none", grad), *truth(x, w, t, bias, grad.double()))


@pytest.mark.parametrize("turned", [False, True])
def test_classes_that_are_improbable_in_every_row(F, turned):
    """Probabilities of 1e-10 to 1e-18: their dw columns and dbias are right to 2^-50 of the rows' weights, which the largest still show."""
    rows, k, n = 300, 64, 2000
    gen, x, w, t = make(4, rows, k, n)
    if turned:
        w = w.t().contiguous().t()
    bias = torch.zeros(n, device="cuda")
    bias[1000:] = -torch.linspace(16, 34, n - 1000, device="cuda")
    t = t % 1000
    grad = torch.rand(rows, device="cuda", generator=gen) + 0.5
    values, offs = truth(x, w, t, bias, grad.double())
    got = step(F, x, w, t, bias, "none", grad)
    close(got, values, offs)
    far = (got["dbias"].double() - values["dbias"]).abs() / values["dbias"]
    assert float(far[1000:1100].max()) <= 1e-3 and float(values["dbias"][1050]) < 300 * 1e-9


@pytest.mark.parametrize("lone", ["0", "1"])
@pytest.mark.parametrize("where", ["x", "w", "both"])
def test_operands_whose_range_f16_does_not_hold(F, monkeypatch, where, lone):
    """Kept rows, classes and features of sizes from 2^-40 to 1: three bf16 planes, for operands and gradients alike."""
    monkeypatch.setenv("MNI_B200_FUSED_LONE", lone)
    rows, k, n = 300, 100, 1500
    gen, x, w, t = make(6, rows, k, n)
    if where != "w":
        x *= torch.exp2(-40 * torch.rand(rows, k, device="cuda", generator=gen))
    if where != "x":
        w *= torch.exp2(-40 * torch.rand(k, n, device="cuda", generator=gen))
    bias = 0.5 * torch.randn(n, device="cuda", generator=gen)
    grad = torch.rand(rows, device="cuda", generator=gen) + 0.5
    grad[::7] = 0
    t[::7] = -1
    values, offs = truth(x, w, t, bias, torch.where(t >= 0, grad, 0.0).double(), wide=True)
    got = step(F, x, w, t, bias, "none", grad)
    assert not got["loss"][::7].any() and not got["dx"][::7].any()
    close(got, values, offs, names=("lse", "dx", "dw", "dbias"))
    close(got, values, offs, names=("loss",), rows=t >= 0)


def test_infinite_and_nan_rows_that_are_kept(F):
    """Their own loss and gradient show it; the other rows' are what they would be without them."""
    rows, k, n = 300, 32, 2000
    gen, x, w, t = make(8, rows, k, n)
    w[1] = 1.0
    values, offs = truth(x, w, t, None, torch.ones(rows, device="cuda").double(), wide=True)
    x[3, 0] = float("nan")
    x[5] = 0.0
    x[5, 1] = float("inf")
    got = step(F, x, w, t, None, "none", torch.ones(rows, device="cuda"))
    bad = torch.tensor([3, 5], device="cuda")
    others = torch.ones(rows, dtype=torch.bool, device="cuda")
    others[bad] = False
    assert torch.isnan(got["lse"][3]) and not torch.isfinite(got["lse"][5])
    assert torch.isnan(got["loss"][bad]).all() and torch.isnan(got["dx"][bad]).all()
    close(got, values, offs, names=("loss", "lse", "dx"), rows=others)
    assert torch.isnan(got["dw"]).all() and torch.isnan(got["dbias"]).all()


@pytest.mark.parametrize("rows", [4096, 4097, 9000])
def test_mean_over_many_rows(F, rows):
    """Rows are counted by a launch of their own from 4097 on."""
    k, n = 40, 100
    gen, x, w, t = make(rows, rows, k, n)
    t = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.3, torch.full_like(t, -100), t)
    bias = 0.5 * torch.randn(n, device="cuda", generator=gen)
    kept = t >= 0
    weight = kept.double() * 1.25 / int(kept.sum())
    values, offs = truth(x, w, t, bias, weight)
    values["loss"] = values["loss"][kept].mean().reshape(1)
    offs["loss"] = offs["loss"][kept].mean().reshape(1) + 2 * HALF_STEP * values["loss"].abs()
    got = step(F, x, w, t, bias, "mean", torch.full((1,), 1.25, device="cuda"))
    close(got, values, offs)


def test_rows_beyond_what_a_piece_holds(F):
    """A piece of the classes is never less than 256 of them, however many the rows: two pieces here."""
    rows, k, n = 270000, 8, 300
    gen, x, w, t = make(2, rows, k, n)
    weight = torch.full((rows,), 1.0 / rows, device="cuda", dtype=torch.float64)
    values, offs = truth(x, w, t, None, weight)
    values["loss"], offs["loss"] = values["loss"].mean().reshape(1), offs["loss"].mean().reshape(1) + HALF_STEP * values["loss"].mean().abs().reshape(1)
    close(step(F, x, w, t, None, "mean", torch.ones(1, device="cuda")), values, offs)


@pytest.mark.parametrize("rows,k,n", [(6, 33, 70), (5, 130, 4097), (300, 101, 1003), (131, 33, 2051)])
@pytest.mark.parametrize("tied", [False, True])
def test_nothing_comes_from_what_scratch_held(F, rows, k, n, tied):
    """In a caller's scratch full of NaN (of 16 and of 32 bits), with sizes that leave the last tiles and pitches ragged: the same bits."""
    import ctypes as C
    gen, x, w, t = make(rows, rows, k, n)
    if tied:
        w = w.t().contiguous().t()
    t[1] = -1
    bias = 0.5 * torch.randn(n, device="cuda", generator=gen)
    one = torch.ones(1, device="cuda")
    want = step(F, x, w, t, bias, "mean", one)
    size = 64 << 20
    scratch = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
    lib = F._lib.lib()
    F._lib.check(lib.mni_b200_workspace_set(C.c_void_p(scratch.data_ptr()), size))
    try:
        got = step(F, x, w, t, bias, "mean", one)
        torch.cuda.synchronize()
    finally:
        F._lib.check(lib.mni_b200_workspace_set(None, 0))
    assert bool((scratch != 0xff).any())
    for name, v in want.items():
        assert torch.equal(got[name], v), name
