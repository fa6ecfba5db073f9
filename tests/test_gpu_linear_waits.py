"""A wait of the block-FP8 products' kernels that runs out, on the GPU: it is reported, and nothing waits behind it."""
import ctypes
import os
import subprocess

import pytest
import torch

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "unimonomoe_b200", "csrc")


def test_a_wait_that_runs_out_is_reported_and_the_last(tmp_path):
    out = str(tmp_path / "waits.so")
    subprocess.run([os.environ.get("NVCC", "nvcc"), "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-I", os.path.join(CSRC, "linear"),
                    os.path.join(HERE, "linear_waits_kernel.cu"), "-o", out], check=True)
    launch = ctypes.CDLL(out).waits_launch
    launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_uint64]
    status, ns = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(4, 3, 2, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    limit = 2_000_000
    assert launch(status.data_ptr(), ns.data_ptr(), 4, limit) == 0
    code, where = status.tolist()
    assert code == 5 and 0 <= where < 4
    first, behind = ns[..., 0].cpu(), ns[..., 1].cpu()
    # A poll that fails takes 4 us at most, measured; the clock is read once in 64. 200 waits behind it, of two barriers, are 400 polls: 1.6 ms, where 64 polls
    # each would be 100 ms.
    assert bool((first.amax(1) >= limit).all()) and bool((first < 10 * limit).all())
    assert bool((behind < 20_000_000).all())
    assert int(torch.ones(8, device="cuda").sum()) == 8
