"""GPU: calls of the cross entropy of a projection and of Newton-Schulz updates that are allowed and seldom made."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def tensor(F, t):
    return F.DeviceTensor.from_torch(t)


def test_another_device_than_the_current_one_is_refused(F):
    """Kernels go to the current device's stream.  The tensors here have a device and a shape and no memory."""
    from conftest import fake_cuda
    there = f"cuda:{torch.cuda.current_device() + 1}"

    def fake(shape, dtype=torch.float32):
        flat = fake_cuda(int(np.prod(shape)), there, dtype)
        return flat if dtype != torch.float32 else F.DeviceTensor(flat, shape)
    x, w, t = fake((6, 8)), fake((8, 10)), fake((6,), torch.int64)
    before = F.launch_count()
    for call in (lambda: F.linear_cross_entropy(x, w, t), lambda: F.linear_cross_entropy_backward(fake((1,)), x, w, t, fake((6,))),
                 lambda: F.orthogonalize(x), lambda: F.muon_step([x], [fake((6, 8))], [fake((6, 8))], lr=0.1)):
        with pytest.raises(ValueError, match=f"the tensors are on {there}, the current device is"):
            call()
    assert F.launch_count() == before


@pytest.mark.parametrize("rows", [6, 300])
@pytest.mark.parametrize("layout", ["stored", "tied"])
def test_the_layout_of_dw_is_its_strides(F, rows, layout):
    """The C interface's flag for a turned dw says nothing here, where dw's strides say it."""
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, 64, device="cuda", generator=gen)
    w = torch.randn(64, 500, device="cuda", generator=gen) if layout == "stored" else torch.randn(500, 64, device="cuda", generator=gen).t()
    t = torch.randint(0, 500, (rows,), device="cuda", generator=gen)
    one = tensor(F, torch.ones(1, device="cuda"))
    _, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t)
    want = F.linear_cross_entropy_backward(one, tensor(F, x), tensor(F, w), t, lse)
    for dw in (None, tensor(F, torch.empty(64, 500, device="cuda")), tensor(F, torch.empty(500, 64, device="cuda").t())):
        got = F.linear_cross_entropy_backward(one, tensor(F, x), tensor(F, w), t, lse, flags=F._lib.DB_TRANSPOSED, dw=dw)
        F.device_status()
        assert got[1].shape == (64, 500)
        # (of either layout the sums are the same up to their order: 300 terms)
        assert float((got[1].torch_view() - want[1].torch_view()).abs().max()) <= 1e-5 * float(want[1].torch_view().abs().max())


def test_strides_that_are_not_given(F):
    """A view with fewer strides than dims: those left out are 0, for dw's layout as for what the kernels read; as a given dw it is refused."""
    x, column = torch.randn(6, 8, device="cuda"), torch.randn(8, device="cuda")
    t = torch.zeros(6, dtype=torch.int64, device="cuda")
    w = F.DeviceTensor(column, (8, 10), (1, 8))
    w.strides = (1,)
    one = tensor(F, torch.ones(1, device="cuda"))
    loss, lse = F.linear_cross_entropy(tensor(F, x), w, t)
    dx, dw = F.linear_cross_entropy_backward(one, tensor(F, x), w, t, lse)
    assert dw.strides == (10, 1) and abs(float(loss.numpy()[0]) - np.log(10)) <= 1e-6
    short = F.DeviceTensor(torch.empty(80, device="cuda"), (8, 10), (1, 8))
    short.strides = (1,)
    with pytest.raises(ValueError, match="dw contiguous or the transposing view"):
        F.linear_cross_entropy_backward(one, tensor(F, x), w, t, lse, dw=short)
    F.device_status()


@pytest.mark.parametrize("shape", [(64, 8192), (8192, 64), (100, 5000), (5003, 101), (3, 12000), (128, 4096), (1, 100000), (100000, 1)])
def test_thin_matrices(F, shape):
    """A short side and thousands on the other: one or a few tiles whose contraction is the long side."""
    from test_muon_gpu import close, gradient, truth
    g = gradient(sum(shape), *shape)
    got = F.orthogonalize(tensor(F, g)).torch_view()
    F.device_status()
    close(got, *truth(g))


@pytest.mark.parametrize("tile", ["64", "128", "256"])
def test_updates_take_nothing_from_what_scratch_held(F, monkeypatch, tile):
    """As for the loss: scratch full of NaN, ragged matrices, each tiling."""
    import ctypes as C

    from test_muon_gpu import gradient
    monkeypatch.setenv("MNI_B200_NEWTON_TILE", tile)
    shapes = [(33, 65), (1, 1), (130, 257), (257, 130), (300, 301), (2, 70, 45)]
    start = [[gradient(7 * i + j, *s) for i, s in enumerate(shapes)] for j in range(3)]

    def run():
        ps, ms, gs = ([t.clone() for t in ts] for ts in start)
        F.muon_step([tensor(F, t) for t in ps], [tensor(F, t) for t in ms], [tensor(F, t) for t in gs], lr=0.05)
        out = [F.orthogonalize(tensor(F, g), steps=s).torch_view().clone() for g in gs for s in (0, 2)]
        F.device_status()
        return ps + ms + out
    want = run()
    size = 64 << 20
    scratch = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
    lib = F._lib.lib()
    F._lib.check(lib.mni_b200_workspace_set(C.c_void_p(scratch.data_ptr()), size))
    try:
        got = run()
        torch.cuda.synchronize()
    finally:
        F._lib.check(lib.mni_b200_workspace_set(None, 0))
    assert bool((scratch != 0xff).any())
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(got, want))


@pytest.mark.parametrize("before", ["nothing", "a small call"])
def test_a_first_call_that_is_captured_is_refused_and_the_capture_goes_on(F, before):
    """Scratch cannot be allocated, nor grow, while a stream captures: nothing is recorded, and the capture stays valid."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    # (each needs more than the MB that the library's scratch is larger than a small call's)
    x, w = torch.randn(300, 256, device="cuda", generator=gen), torch.randn(256, 2000, device="cuda", generator=gen)
    t = torch.randint(0, 2000, (300,), device="cuda", generator=gen)
    p, m, g = (torch.randn(400, 500, device="cuda", generator=gen) for _ in range(3))
    one, lse = tensor(F, torch.ones(1, device="cuda")), tensor(F, torch.ones(300, device="cuda"))
    tx, tw, tp, tm, tg = (tensor(F, v) for v in (x, w, p, m, g))
    kept = p.clone(), m.clone()
    F.device_status()
    F._lib.check(F._lib.lib().mni_b200_release())
    if before != "nothing":
        F.linear_cross_entropy(tensor(F, x[:9, :4].contiguous()), tensor(F, w[:4, :5].contiguous()), t[:9] % 5)
    stream = torch.cuda.Stream()
    total = torch.zeros(1, device="cuda")
    calls = (lambda: F.linear_cross_entropy(tx, tw, t), lambda: F.linear_cross_entropy_backward(one, tx, tw, t, lse), lambda: F.orthogonalize(tg),
             lambda: F.muon_step([tp], [tm], [tg], lr=0.1))
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        launched = F.launch_count()
        with torch.cuda.graph(graph, stream=stream):
            for call in calls:
                with pytest.raises(F._lib.MniError) as e:
                    call()
                assert e.value.status == 7 and "captur" in e.value.message, e.value
            total += 1
        assert F.launch_count() == launched
    graph.replay()
    torch.cuda.synchronize()
    assert float(total) == 1.0 and torch.equal(p, kept[0]) and torch.equal(m, kept[1])
    for call in calls:
        call()
    F.device_status()


@pytest.mark.parametrize("rows", [6, 256])
def test_features_seen_through_unusual_views(F, rows):
    """One feature for all columns, extents of one with any stride, as many dims as a view may have."""
    from test_linear_cross_entropy_gpu import compare, make
    _, w, t, b = make(3, rows, 48, 700, bias=True)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    compare(F, torch.randn(rows, 1, device="cuda", generator=gen).expand(rows, 48), w, t, b)
    compare(F, torch.randn(1, 1, device="cuda", generator=gen).expand(rows, 48), w, t, b)
    flat = torch.randn(rows, 48, device="cuda", generator=gen)
    compare(F, flat.as_strided((1, rows, 1, 48), (7, 48, 1000003, 1)), w, t.reshape(1, rows, 1), b)
    if rows == 256:
        x = torch.randn(2, 2, 4, 2, 2, 2, 2, 96, device="cuda", generator=gen)[..., ::2].permute(3, 1, 0, 2, 6, 4, 5, 7)
        compare(F, x, w, t.reshape(x.shape[:-1]), b)


@pytest.mark.parametrize("misalign", [1, 2])
@pytest.mark.parametrize("layout", ["stored", "tied"])
@pytest.mark.parametrize("rows,k,n", [(6, 32, 2000), (300, 101, 1003), (260, 128, 1024)])
def test_everything_off_a_16_byte_boundary(F, rows, k, n, layout, misalign):
    """Operands, bias, lse and gradients one or two floats behind a boundary, between guard zones."""
    from conftest import Guarded
    from test_linear_cross_entropy_gpu import close, make, truth

    def moved(t):
        flat = torch.empty(t.numel() + misalign, device="cuda")
        flat[misalign:] = t.reshape(-1)
        return flat[misalign:].view(t.shape)
    x, w, t, b = make(1, rows, k, n, "stored", bias=True, masked=True)
    x, b = moved(x), moved(b)
    w = moved(w) if layout == "stored" else moved(w.t().contiguous()).t()
    values, offs = truth(x, w, t, b, "mean", torch.ones(1, device="cuda"))
    loss, lse = F.linear_cross_entropy(tensor(F, x), tensor(F, w), t, tensor(F, b))
    outs = [Guarded(F, s, None, misalign) for s in ((rows, k), (n, k) if layout == "tied" else (k, n), (n,))]
    dw = outs[1].tensor.permute([1, 0]) if layout == "tied" else outs[1].tensor
    got = F.linear_cross_entropy_backward(tensor(F, moved(torch.ones(1, device="cuda"))), tensor(F, x), tensor(F, w), t, tensor(F, moved(lse.torch_view())),
                                          tensor(F, b), want_dbias=True, dx=outs[0].tensor, dw=dw, dbias=outs[2].tensor)
    F.device_status()
    for i, o in enumerate(outs):
        o.check(f"output {i}")
    close(loss.torch_view(), values["loss"], offs["loss"], "loss")
    for name, g in zip(("dx", "dw", "dbias"), got):
        close(g.torch_view(), values[name], offs[name], name)


@pytest.mark.parametrize("reserve", [60, 140])
def test_beside_a_kernel_that_takes_the_other_sms(F, reserve):
    """Grids of few CTAs, down to eight: tiles that wait for one another are drawn in an order in which the first can always run."""
    from test_linear_cross_entropy_gpu import compare, make
    from test_muon_gpu import close, gradient, truth
    g = [gradient(3, 300, 260), gradient(4, 520, 700)]
    F.sm_reserve(reserve)
    try:
        got = [F.orthogonalize(tensor(F, v)).torch_view() for v in g]
        F.device_status()
        compare(F, *make(5, 300, 128, 1500, bias=True, masked=True))
    finally:
        F.sm_reserve(0)
    for v, a in zip(g, got):
        close(a, *truth(v))
