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
