"""CPU: what the operators refuse on the host, for tensors that have a device and a shape and no memory."""
import pytest
import torch

from conftest import fake_cuda

X, W, ROWS = (6, 8), (8, 10), (6,)


@pytest.fixture(scope="module", autouse=True)
def library():
    from framework_b200 import build
    build.build_library()


def tensor(shape, device="cuda:0", strides=None):
    from framework_b200 import DeviceTensor
    n = 1
    for s in shape:
        n *= s
    return DeviceTensor(fake_cuda(n, device), shape, strides)


def targets():
    return fake_cuda(6, "cuda:0", torch.int64)


def test_every_tensor_of_a_call_is_on_one_device():
    """Those of another GPU would reach the kernels as plain pointers."""
    from framework_b200 import ops
    there = "cuda:1"
    with pytest.raises(ValueError, match="bias is on cuda:1.*cuda:0"):
        ops.linear_cross_entropy(tensor(X), tensor(W), targets(), tensor((10,), there))
    good = dict(grad=tensor((1,)), x=tensor(X), weight=tensor(W), targets=targets(), lse=tensor(ROWS))
    for name, value in [("grad", tensor((1,), there)), ("lse", tensor(ROWS, there)), ("bias", tensor((10,), there)), ("dx", tensor(X, there)),
                        ("dw", tensor(W, there)), ("dw", tensor((10, 8), there).permute([1, 0])), ("dbias", tensor((10,), there))]:
        with pytest.raises(ValueError, match=f"{name} is on cuda:1"):
            ops.linear_cross_entropy_backward(**{**good, name: value}, want_dbias=True)
    for which in range(6):
        lists = [[tensor((4, 5)), tensor((4, 5))] for _ in range(3)]
        lists[which // 2][which % 2] = tensor((4, 5), there)
        with pytest.raises(ValueError, match="on cuda"):
            ops.muon_step(*lists, lr=0.1)


@pytest.mark.parametrize("flag,wanted", [("ACCUMULATE_DA", "dx"), ("ACCUMULATE_DB", "dw"), ("ACCUMULATE_DBIAS", "dbias")])
def test_nothing_is_added_to_memory_that_was_not_given(flag, wanted):
    """A gradient that the call allocates itself holds whatever was there before."""
    from framework_b200 import _lib, ops
    with pytest.raises(ValueError, match=f"flags add to {wanted}, and none is given"):
        ops.linear_cross_entropy_backward(tensor((1,)), tensor(X), tensor(W), targets(), tensor(ROWS), flags=getattr(_lib, flag), want_dbias=True)


def test_host_memory_that_runs_out_is_an_error():
    """A list of half a million matrices, in a process that may have no more memory than it has: a status, and the process goes on."""
    import os
    import subprocess
    import sys
    program = """
import ctypes as C, resource
from framework_b200 import _lib
lib, n = _lib.lib(), 1 << 19
def pointers(base):
    return (C.c_void_p * n)(*range(base, base + 1024 * n, 1024))
lists = [pointers(1 << (40 + k)) for k in range(3)]
four, ones = (C.c_int64 * n)(*([4] * n)), (C.c_float * n)()
used = int(next(l for l in open("/proc/self/status") if l.startswith("VmSize")).split()[1]) * 1024
resource.setrlimit(resource.RLIMIT_AS, (used + (8 << 20), resource.RLIM_INFINITY))
status = lib.mni_b200_muon_step(n, *lists, four, four, ones, 0.1, 0.9, 1, 0.0, 5, 3.4445, -4.775, 2.0315, 1e-7, None)
print(status, lib.mni_b200_last_error().decode())
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.startswith("7 host memory"), done.stdout + done.stderr[-1000:]


LONG = 2 ** 31 - 1


@pytest.mark.parametrize("rows,k,n", [(LONG, 1, 4), (4, 1, LONG), (4, LONG, 1), (1 << 21, 1 << 20, 4), (LONG - 5000, LONG - 5000, 1), (9, 1 << 20, 1 << 21)])
def test_sizes_beyond_the_kernels_indices_are_refused(rows, k, n):
    """Views of stride 0 have any extent without the memory; what the call would need in scratch goes past 64 bits."""
    from framework_b200 import _lib
    lib = _lib.lib()
    x, w = _lib.make_view(256, (rows, k), (0, 0)), _lib.make_view(256, (k, n), (0, 0))
    assert lib.mni_b200_linear_cross_entropy_fwd(x, w, None, 512, 8, 2, 512, 512, 0, None) == 9
    assert "too many" in lib.mni_b200_last_error().decode()
    assert lib.mni_b200_linear_cross_entropy_bwd(x, w, None, 512, 8, 2, 512, 512, 512, 512, None, 0, None) == 9


def test_matrices_whose_tiles_outlast_a_wait_are_refused():
    """A tile's contraction over 2^27 elements takes longer than the tiles behind it may wait."""
    import ctypes as C

    from framework_b200 import _lib
    lib = _lib.lib()
    newton = (3.4445, -4.775, 2.0315, 1e-7)
    for rows, cols in ((4, (1 << 26) + 1), ((1 << 26) + 1, 4), (1, LONG)):
        assert lib.mni_b200_orthogonalize(_lib.make_view(256, (rows, cols), (0, 0)), 512, 5, *newton, None) == 9
        assert "too large" in lib.mni_b200_last_error().decode()
        one = [(C.c_void_p * 1)(1 << (40 + k)) for k in range(3)]
        sizes = (C.c_int64 * 1)(rows), (C.c_int64 * 1)(cols)
        assert lib.mni_b200_muon_step(1, *one, *sizes, (C.c_float * 1)(1.0), 0.1, 0.9, 1, 0.0, 5, *newton, None) == 9


def test_batches_whose_count_does_not_fit_are_refused():
    from framework_b200 import _lib
    lib = _lib.lib()
    for lead in ((1 << 30, 1 << 30, 1 << 4), (1 << 30, 1 << 20)):               # 2^64 matrices, which are none in 64 bits; 2^50
        g = _lib.make_view(256, (*lead, 4, 4), (0,) * (len(lead) + 2))
        assert lib.mni_b200_orthogonalize(g, 512, 5, 3.4445, -4.775, 2.0315, 1e-7, None) == 9
        assert "too many elements" in lib.mni_b200_last_error().decode()
