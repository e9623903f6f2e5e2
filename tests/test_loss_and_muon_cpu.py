"""CPU: what the cross entropy of a projection and the Newton-Schulz updates refuse, before they touch a device."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    from framework_b200 import _lib, build
    build.build_library()
    return _lib.lib()


def view(shape, strides=None, ptr=256):
    from framework_b200 import _lib
    from framework_b200.shapes import row_major_strides
    return _lib.make_view(ptr, shape, strides or row_major_strides(shape))


X, W, OK = (6, 8), (8, 10), 512


def forward(lib, x=X, w=W, targets=OK, bytes=8, reduction=2, loss=OK, lse=OK, flags=0, **kw):
    return lib.mni_b200_linear_cross_entropy_fwd(view(x, **kw), view(w), None, targets, bytes, reduction, loss, lse, flags, None)


def backward(lib, x=X, w=W, targets=OK, bytes=8, reduction=2, lse=OK, grad=OK, flags=0):
    return lib.mni_b200_linear_cross_entropy_bwd(view(x), view(w), None, targets, bytes, reduction, lse, grad, OK, OK, None, flags, None)


@pytest.mark.parametrize("call", [forward, backward])
@pytest.mark.parametrize("change,status,text", [
    (dict(x=(8,)), 1, "at least 2D"), (dict(w=(8,)), 1, "at least 2D"), (dict(w=(2, 8, 10)), 4, "a matrix is needed"),
    (dict(w=(9, 10)), 2, "inner dimensions must match: 8 vs 9"), (dict(x=(6, 0), w=(0, 10)), 4, "no classes or no features"),
    (dict(w=(8, 0)), 4, "no classes"), (dict(bytes=2), 4, "targets of 2 bytes"), (dict(reduction=3), 4, "unknown reduction 3"),
    (dict(reduction=-1), 4, "unknown reduction"), (dict(targets=None), 4, "targets is null"), (dict(targets=516), 4, "not aligned"),
    (dict(x=(1 << 20, 1 << 12, 8)), 9, "rows"), (dict(flags=1), 4, "flags 0x1"), (dict(flags=1 << 8), 4, "flags"), (dict(lse=None), 4, "null")])
def test_refusals_of_the_loss(lib, call, change, status, text):
    assert call(lib, **change) == status
    assert text in lib.mni_b200_last_error().decode()


def test_flags_of_the_forward_and_null_outputs(lib):
    assert forward(lib, flags=1 << 2) == 4                       # accumulating is the backward's
    assert forward(lib, loss=None) == 4
    assert backward(lib, grad=None) == 4
    assert lib.mni_b200_linear_cross_entropy_fwd(None, view(W), None, OK, 8, 2, OK, OK, 0, None) == 4
    assert lib.mni_b200_linear_cross_entropy_fwd(view(X, ptr=None), view(W), None, OK, 8, 2, OK, OK, 0, None) == 4


@pytest.mark.parametrize("change,status,text", [
    (dict(g=(4,)), 1, "at least 2D"), (dict(steps=-1), 4, "-1 steps"), (dict(steps=101), 4, "101 steps"), (dict(eps=-1.0), 4, "eps"),
    (dict(eps=float("nan")), 4, "eps"), (dict(a=float("inf")), 4, "finite"), (dict(c=float("nan")), 4, "finite"), (dict(a=1e8), 4, "larger than 1e9"), (dict(out=None), 4, "out is null"),
    (dict(g=(1 << 30, 1 << 10)), 9, "too large")])
def test_refusals_of_orthogonalize(lib, change, status, text):
    args = dict(g=(4, 6), out=OK, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7)
    args.update(change)
    g = view(args["g"])
    assert lib.mni_b200_orthogonalize(g, args["out"], args["steps"], args["a"], args["b"], args["c"], args["eps"], None) == status
    assert text in lib.mni_b200_last_error().decode()


def muon(lib, params, momenta, grads, rows, cols, count=None, steps=5, eps=1e-7):
    n = len(params)
    ptrs = [(C.c_void_p * n)(*v) for v in (params, momenta, grads)]
    sizes = [(C.c_int64 * n)(*v) for v in (rows, cols)]
    scales = (C.c_float * n)(*([1.0] * n))
    return lib.mni_b200_muon_step(n if count is None else count, *ptrs, *sizes, scales, 0.1, 0.9, 1, 0.0, steps, 3.4445, -4.775, 2.0315, eps, None)


def test_refusals_of_muon_step(lib):
    assert muon(lib, [256], [4096], [8192], [4], [4], count=-1) == 4
    assert muon(lib, [None], [4096], [8192], [4], [4]) == 4 and "null pointer" in lib.mni_b200_last_error().decode()
    assert muon(lib, [256], [4096], [8192], [-4], [4]) == 4
    assert muon(lib, [256], [4096], [8192], [1 << 32], [4]) == 9
    assert muon(lib, [256], [4096], [8192], [4], [4], steps=-2) == 4
    for arrays in (([256], [256], [8192]), ([256], [4096], [4096 + 60]), ([256], [4096], [256 - 4])):
        assert muon(lib, *arrays, [4], [4]) == 4 and "share memory" in lib.mni_b200_last_error().decode()
    assert lib.mni_b200_muon_step(1, None, None, None, None, None, None, 0.1, 0.9, 1, 0.0, 5, 1.0, 1.0, 1.0, 0.0, None) == 4
    assert muon(lib, [256], [4096], [8192], [0], [4]) == 0          # nothing to do, and nothing touched
    assert lib.mni_b200_muon_step(0, None, None, None, None, None, None, 0.1, 0.9, 1, 0.0, 5, 1.5, -0.5, 0.0, 0.0, None) == 0


def test_names_of_reductions_and_scales():
    from framework_b200 import ops
    with pytest.raises(ValueError, match="reduction must be one of"):
        ops.linear_cross_entropy(None, None, None, reduction="average")
    with pytest.raises(ValueError, match="scale must be"):
        ops.muon_step([], [], [], lr=0.1, scale="width")
