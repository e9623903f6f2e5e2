"""GPU: a kernel whose warps trade registers is launched only if the compiler gave it as many as the trade counts on.

`setmaxnreg.inc` draws on what the block was launched with; beyond that it waits for good, which no limit of the library's ends.  A test
hook stands in for the number that the compiler gave, so that the call is refused before anything is launched.  The question
is asked before a kernel's first launch of a process, so each case has one of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CALLS = {
    "logits": """
x, w, t = rand(300, 256), rand(256, 2000), torch.zeros(300, dtype=torch.int64, device="cuda")
F.linear_cross_entropy(x, w, t)""",
    "logit_gradients": """
x, w, t = rand(300, 256), rand(256, 2000), torch.zeros(300, dtype=torch.int64, device="cuda")
F.linear_cross_entropy_backward(rand(1), x, w, t, rand(300))""",
    "newton_schulz": "F.orthogonalize(rand(300, 280))",
    "planes": "F.matmul(rand(4096, 1024), rand(1024, 4096))",
}


@pytest.mark.parametrize("call,env", [
    ("logits", {"MNI_B200_FUSED_LONE": "0"}), ("logits", {"MNI_B200_FUSED_LONE": "1"}),
    ("logit_gradients", {"MNI_B200_FUSED_LONE": "0"}), ("logit_gradients", {"MNI_B200_FUSED_LONE": "1"}),
    ("newton_schulz", {"MNI_B200_NEWTON_TILE": "64"}), ("newton_schulz", {"MNI_B200_NEWTON_TILE": "256"}),
    ("planes", {})])
def test_too_few_registers_are_refused(call, env):
    program = f"""
import torch
import framework_b200 as F

def rand(*shape):
    return F.DeviceTensor.from_torch(torch.rand(*shape, device="cuda"))
try:
    {CALLS[call].strip().replace(chr(10), chr(10) + "    ")}
except F._lib.MniError as e:
    assert e.status == 6 and "set-up failed: invalid configuration" in e.message, e
    torch.cuda.synchronize()
    print("refused")
"""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, env={**os.environ, **env, "MNI_B200_TEST_LAUNCH_REGS": "128"},
                          capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and "refused" in done.stdout, done.stdout + done.stderr[-2000:]
