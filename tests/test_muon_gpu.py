"""Newton-Schulz updates against the recursion in 64 bits.

A step x' = q(x x^T) x, q = a + b A + c A^2, turns an error of x into at most L = max |p'| <= 4.3 of it, p(s) = a s + b s^3 + c s^5 on the
singular values that occur (0 to 1.21).  Its own three products, each off by PRODUCT of its size, add at most PRODUCT * R |x|, where
R = a + 2 |b| + 4 |c| covers them for singular values up to 1.21 (s^2 <= 1.47, s^4 <= 2.15).  `bound` adds that up over the steps."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
PRODUCT, L, R = 2e-6, 4.3, 3.4445 + 2 * 4.775 + 4 * 2.0315


def tensor(F, t):
    return F.DeviceTensor.from_torch(t)


def truth(g, steps=5, eps=1e-7, coefficients=(A, B, C), slope=L, rounding=R):
    """-> the result in 64 bits and how far (2-norm) an f32 one may be off, for each matrix."""
    a, b, c = coefficients
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    off = 2.0 ** -22 * torch.linalg.matrix_norm(x)
    tall = x.shape[-2] > x.shape[-1]
    for _ in range(steps):
        off = slope * off + PRODUCT * rounding * torch.linalg.matrix_norm(x)
        y = x.mT @ x if tall else x @ x.mT
        q = b * y + c * y @ y
        x = a * x + (x @ q if tall else q @ x)
    return x, off


def close(got, want, off):
    assert torch.isfinite(got).all()
    far = torch.linalg.matrix_norm(got.double() - want)
    assert (far <= off).all(), (far, off)
    # and what f32 products deliver: within a few times of the 4e-6 that they are off at worst on these matrices
    assert (far <= 2e-5 * torch.linalg.matrix_norm(want) + 1e-30).all(), far / torch.linalg.matrix_norm(want)


def gradient(seed, *shape):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, device="cuda", generator=gen)
    r = min(shape[-2], shape[-1], 8)
    return 1e-3 * (normal(*shape[:-1], r) @ normal(*shape[:-2], r, shape[-1]) / r + 0.3 * normal(*shape))


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 3), (5, 5), (16, 64), (64, 16), (31, 33), (64, 32), (65, 64), (100, 257), (128, 128), (257, 130), (256, 512),
          (300, 300), (700, 333), (333, 1000), (1030, 520), (3, 4, 20), (2, 2, 65, 40), (5, 300, 260)]


@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(F, shape):
    g = gradient(sum(shape), *shape)
    got = F.orthogonalize(tensor(F, g))
    F.device_status()
    assert got.shape == shape
    close(got.torch_view(), *truth(g))


@pytest.mark.parametrize("tile", ["64", "128", "256"])
@pytest.mark.parametrize("shape", [(1, 1), (40, 70), (257, 130), (300, 300), (700, 333), (520, 1030), (3, 257, 513)])
def test_every_tiling(F, monkeypatch, tile, shape):
    """Tiles that one matrix of these sizes would not be given: ragged ones, and blocks below the diagonal read from above."""
    monkeypatch.setenv("MNI_B200_NEWTON_TILE", tile)
    g = gradient(sum(shape), *shape)
    got = F.orthogonalize(tensor(F, g)).torch_view()
    F.device_status()
    close(got, *truth(g))
    batch = (shape[0],) if len(shape) == 3 else ()
    p, m, u = (gradient(9 + i, *batch, *shape[-2:]) for i in range(3))
    want, _, off = step_truth(p, m, u, 0.05, 0.95, True, 0.02, 0.5)
    F.muon_step([tensor(F, p)], [tensor(F, m)], [tensor(F, u)], lr=0.05, weight_decay=0.02, scale=0.5)
    F.device_status()
    assert (torch.linalg.matrix_norm(p.double() - want) <= off + 2.0 ** -23 * torch.linalg.matrix_norm(want)).all()


def test_more_matrices_than_a_launch_takes(F):
    g = gradient(5, 700, 12, 9)
    got = F.orthogonalize(tensor(F, g)).torch_view()
    F.device_status()
    close(got, *truth(g))


def test_more_shapes_than_a_launch_takes(F):
    """Shapes of one launch run side by side, long and short, tall and wide."""
    shapes = [(16 + 24 * i, 300 - 23 * i) for i in range(12)] + [(64, 700), (900, 40)]
    ps, ms, gs = ([gradient(7 * i + j, *s) for i, s in enumerate(shapes)] for j in range(3))
    want = [step_truth(p, m, g, 0.05, 0.95, True, 0.0, 0.5) for p, m, g in zip(ps, ms, gs)]
    F.muon_step([tensor(F, t) for t in ps], [tensor(F, t) for t in ms], [tensor(F, t) for t in gs], lr=0.05, scale=0.5)
    F.device_status()
    for p, (wp, _, off) in zip(ps, want):
        assert torch.linalg.matrix_norm(p.double() - wp) <= off + 2.0 ** -23 * torch.linalg.matrix_norm(wp)


def test_two_streams_in_turn(F):
    """Calls on two streams, ordered by events as the scratch of a device asks for."""
    shapes = [(300, 500), (512, 128), (300, 500)]
    ps, ms, gs = ([gradient(11 * i + j, *s) for i, s in enumerate(shapes)] for j in range(3))
    qs, ns = ([t.clone() for t in ts] for ts in (ps, ms))
    for _ in range(4):
        F.muon_step([tensor(F, t) for t in qs], [tensor(F, t) for t in ns], [tensor(F, t) for t in gs], lr=0.05)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        streams[k % 2].wait_stream(streams[1 - k % 2])
        with torch.cuda.stream(streams[k % 2]):
            F.muon_step([tensor(F, t) for t in ps], [tensor(F, t) for t in ms], [tensor(F, t) for t in gs], lr=0.05)
    torch.cuda.synchronize()
    F.device_status()
    assert all(torch.equal(a, b) for a, b in zip(ps + ms, qs + ns))


def test_singular_values_are_nearly_one(F):
    gen = torch.Generator(device="cuda").manual_seed(3)
    g = torch.randn(200, 600, device="cuda", generator=gen)
    s = torch.linalg.svdvals(F.orthogonalize(tensor(F, g)).torch_view().double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1.0, 1e12, 1e30])
@pytest.mark.parametrize("shape", [(20, 30), (300, 200)])
def test_any_size_of_gradient(F, scale, shape):
    g = gradient(4, *shape) * scale
    got = F.orthogonalize(tensor(F, g), eps=0.0)
    close(got.torch_view(), *truth(g, eps=0.0))


@pytest.mark.parametrize("steps", [0, 5])
@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -138, 2.0 ** 127])
def test_norms_beyond_the_normal_range(F, scale, steps):
    """Elements of 8 bits times a power of two, exact where f32 has subnormals only; the norm's inverse, or the norm, is beyond f32's normal range."""
    g = torch.round(gradient(4, 40, 24) * 1e5).clamp(-127, 127) * 2.0 ** -7
    h = (g.double() * scale).float()
    assert torch.equal(h.double(), g.double() * scale)
    got = F.orthogonalize(tensor(F, h), steps=steps, eps=0.0).torch_view()
    want, off = truth(g, steps, eps=0.0)
    assert torch.isfinite(got).all() and torch.linalg.matrix_norm(got.double() - want) <= off


@pytest.mark.parametrize("steps", [0, 1, 3, 9])
@pytest.mark.parametrize("shape", [(24, 40), (270, 190)])
def test_steps(F, steps, shape):
    g = gradient(4, *shape)
    got = F.orthogonalize(tensor(F, g), steps=steps).torch_view()
    want, off = truth(g, steps)
    far = torch.linalg.matrix_norm(got.double() - want)
    assert (far <= off).all() and (far <= 4e-6 * (steps + 1) * torch.linalg.matrix_norm(want)).all()


@pytest.mark.parametrize("coefficients", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (3.0, -3.2, 1.2), (0.0, 0.0, 0.0), (1.0, 0.0, 0.0), (0.25, 0.0, 1.0)])
def test_other_coefficients(F, coefficients):
    """Some that converge to one, some that make the matrix large or small: the scales of the steps follow."""
    g = gradient(4, 150, 90)
    got = F.orthogonalize(tensor(F, g), steps=3, coefficients=coefficients).torch_view()
    want, _ = truth(g, 3, coefficients=coefficients)
    assert torch.linalg.matrix_norm(got.double() - want) <= 2e-5 * torch.linalg.matrix_norm(want)


def test_zero_and_not_finite(F):
    g = gradient(4, 3, 40, 60)
    g[1] = 0
    g[2, 5, 7] = float("nan")
    got = F.orthogonalize(tensor(F, g)).torch_view()
    F.device_status()
    close(got[:1], *truth(g[:1]))
    assert not got[1].any() and torch.isnan(got[2]).all()


def test_views(F):
    """Transposed, strided, broadcast: gathered on the device; the input is left as it was."""
    g = gradient(6, 80, 50)
    for view in (g.t(), g[::2], g[:, 3:40], torch.stack([g, g])[:, :, ::3], g[:40].unsqueeze(0).expand(3, 40, 50)):
        before = g.clone()
        close(F.orthogonalize(tensor(F, view)).torch_view(), *truth(view))
        assert torch.equal(g, before)


def step_truth(p, m, g, lr, mu, nesterov, decay, scale, steps=5):
    m2 = mu * m.double() + g.double()
    u = g.double() + mu * m2 if nesterov else m2
    o, off = truth(u, steps)
    return (1 - lr * decay) * p.double() - lr * scale * o, m2, lr * scale * off


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_muon_step(F, nesterov, decay):
    """A model's list: repeated shapes, odd ones, leading dims, empty ones, more than one step."""
    shapes = [(64, 64), (64, 256), (256, 64), (33, 65), (64, 64), (3, 20, 30), (1, 5), (300, 280), (0, 4), (300, 280)]
    ps, ms, gs = ([gradient(7 * i + j, *s) if 0 not in s else torch.empty(*s, device="cuda") for i, s in enumerate(shapes)] for j in range(3))
    ps = [50 * p for p in ps]
    for step in range(2):
        want = []
        for p, m, g, s in zip(ps, ms, gs, shapes):
            scale = max(1.0, s[-1] / max(s[-2], 1)) ** 0.5
            want.append(step_truth(p, m, g, 0.02, 0.9, nesterov, decay, scale))
        kept = [g.clone() for g in gs]
        F.muon_step([tensor(F, t) for t in ps], [tensor(F, t) for t in ms], [tensor(F, t) for t in gs], lr=0.02, momentum=0.9, nesterov=nesterov,
                    weight_decay=decay)
        F.device_status()
        for p, m, g, k, (wp, wm, off) in zip(ps, ms, gs, kept, want):
            if not p.numel():
                continue
            assert ((m.double() - wm).abs() <= 2.0 ** -23 * (wm.abs() + k.abs())).all() and torch.equal(g, k)
            far = torch.linalg.matrix_norm(p.double() - wp)
            assert (far <= off + 2.0 ** -23 * torch.linalg.matrix_norm(p.double())).all(), far


@pytest.mark.parametrize("scale,want", [("shape", 2.0), ("size", 0.2 * 160 ** 0.5), (0.5, 0.5)])
def test_scale_of_the_update(F, scale, want):
    p, m, g = torch.zeros(40, 160, device="cuda"), torch.zeros(40, 160, device="cuda"), gradient(3, 40, 160)
    F.muon_step([tensor(F, p)], [tensor(F, m)], [tensor(F, g)], lr=0.1, scale=scale)
    o, off = truth(g)
    assert torch.linalg.matrix_norm(p.double() + 0.1 * want * o) <= 0.1 * want * off + 1e-6


def test_the_same_tensor_twice_is_stepped_twice(F):
    p, m, g = (gradient(i, 48, 80) for i in range(3))
    p1, m1 = p.clone(), m.clone()
    for _ in range(2):
        F.muon_step([tensor(F, p1)], [tensor(F, m1)], [tensor(F, g)], lr=0.1)
    tp, tm, tg = tensor(F, p), tensor(F, m), tensor(F, g)
    F.muon_step([tp, tp], [tm, tm], [tg, tg], lr=0.1)
    F.device_status()
    assert torch.equal(p, p1) and torch.equal(m, m1)


def test_unaligned_and_bounded(F):
    """Every output between guard zones, off a 16-byte boundary."""
    from conftest import Guarded
    for shape in ((37, 21), (300, 257), (64, 64)):
        host = [gradient(i, *shape).cpu().numpy() for i in range(3)]
        for misalign in (0, 1, 3):
            boxes = [Guarded(F, shape, h, misalign) for h in host]
            F.muon_step([boxes[0].tensor], [boxes[1].tensor], [boxes[2].tensor], lr=0.05)
            F.device_status()
            for i, b in enumerate(boxes):
                b.check(str(i))
            p, m, g = (torch.from_numpy(h).cuda() for h in host)
            wp, _, off = step_truth(p, m, g, 0.05, 0.95, True, 0.0, max(1.0, shape[1] / shape[0]) ** 0.5)
            got = torch.from_numpy(boxes[0].tensor.numpy()).cuda()
            assert torch.linalg.matrix_norm(got.double() - wp) <= off + 2.0 ** -23 * torch.linalg.matrix_norm(wp)


def test_captured_and_replayed(F):
    shapes = [(64, 96), (300, 260), (64, 96)]
    ps, ms, gs = ([gradient(7 * i + j, *s) for i, s in enumerate(shapes)] for j in range(3))
    start = [[t.clone() for t in ts] for ts in (ps, ms)]
    tp, tm, tg = ([tensor(F, t) for t in ts] for ts in (ps, ms, gs))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.muon_step(tp, tm, tg, lr=0.05)
        torch.cuda.synchronize()
        first = [t.clone() for t in ps]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            F.muon_step(tp, tm, tg, lr=0.05)
    for kept, live in zip(start[0] + start[1], ps + ms):
        live.copy_(kept)
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    F.device_status()
    assert all(torch.equal(a, b) for a, b in zip(first, ps))


def test_the_step_that_training_takes(F):
    """Loss of a projection, its gradient, and the update of the projection: the operators as they are used together.  The first step's
    parameter against 64 bits; what the gradient is off by (1e-5 of its size at most) the orthogonalisation may turn into 3.45^5 times as much of the
    update's smallest directions, so it is given the same gradient here."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(500, 96, device="cuda", generator=gen)
    w = 0.1 * torch.randn(96, 700, device="cuda", generator=gen)
    t = torch.randint(0, 700, (500,), device="cuda", generator=gen)
    m = torch.zeros_like(w)
    tx, tw, tm = tensor(F, x), tensor(F, w), tensor(F, m)
    one = tensor(F, torch.ones(1, device="cuda"))
    before = w.clone()
    loss, lse = F.linear_cross_entropy(tx, tw, t)
    z = x.double() @ before.double()
    want = torch.nn.functional.cross_entropy(z, t)
    assert abs(float(loss.numpy()[0]) - float(want)) <= 1e-5 * float(want)
    _, dw = F.linear_cross_entropy_backward(one, tx, tw, t, lse, need_dx=False)
    F.muon_step([tw], [tm], [dw], lr=0.02, weight_decay=0.01)
    F.device_status()
    wp, wm, off = step_truth(before, torch.zeros_like(w), dw.torch_view(), 0.02, 0.95, True, 0.01, (700 / 96) ** 0.5)
    assert torch.linalg.matrix_norm(w.double() - wp) <= off + 2.0 ** -23 * torch.linalg.matrix_norm(wp)
    assert ((m.double() - wm).abs() <= 2.0 ** -23 * wm.abs()).all()


@pytest.mark.parametrize("tile", ["64", "256"])
def test_wait_limit_runs_out_then_the_library_recovers(F, monkeypatch, tile):
    """Copies of one stage that the test hook withholds: every role's wait ends, the status says so, and the next call is right."""
    g = gradient(8, 300, 280)
    assert F.device_status() == 0
    monkeypatch.setenv("MNI_B200_NEWTON_TILE", tile)
    monkeypatch.setenv("MNI_B200_WAIT_CYCLES", "2000000")           # about 1 ms
    monkeypatch.setenv("MNI_B200_TEST_WITHHOLD_KBLOCK", "3")
    F.orthogonalize(tensor(F, g))
    with pytest.raises(F._lib.MniError) as ei:
        F.device_status()
    assert ei.value.status == 8 and "bounded wait" in ei.value.message
    monkeypatch.delenv("MNI_B200_TEST_WITHHOLD_KBLOCK")
    monkeypatch.delenv("MNI_B200_WAIT_CYCLES")
    assert F.device_status() == 0
    close(F.orthogonalize(tensor(F, g)).torch_view(), *truth(g))
    assert F.device_status() == 0
