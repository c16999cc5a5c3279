"""The wait that all warps of the paged attention kernels use: one answer for all
lanes, whenever each of them comes to it, and an end when nothing arrives."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import gpu_util as G
from arcllm_b200 import build

pytestmark = pytest.mark.gpu
SRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "warp_wait.cu")
US, TIMEOUT = 1000, 1


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("wait") / "warp_wait.so")
    subprocess.run([build.NVCC] + build.ARCH + build.FLAGS + ["-shared", "-o", so, SRC], check=True, timeout=600)
    lib = C.CDLL(so)

    def go(lane_ns, arrive_ns, limit_ns):
        out = torch.full((33,), -1, dtype=torch.int32, device=G.dev())
        out[32] = 0
        torch.cuda.synchronize()
        assert lib.warp_wait_run(lane_ns, arrive_ns, limit_ns, C.c_void_p(out.data_ptr()),
                                 C.c_void_p(out.data_ptr() + 128)) == 0
        got = out.tolist()
        return got[:32], got[32]

    return go


def test_a_barrier_that_nothing_completes(run):
    for lane in (0, 50 * US):
        assert run(lane, 0, 2000 * US) == ([0] * 32, TIMEOUT)


def test_a_barrier_that_is_completed(run):
    for lane in (0, 50 * US):
        assert run(lane, 300 * US, 500000 * US) == ([1] * 32, 0)


def test_lanes_that_come_after_others_have_waited_longer_than_the_limit(run):
    """Lane 31 comes 3.1 ms after lane 0, the limit is 1 ms and the barrier is completed after 2: lanes that decided for
    themselves would give different answers."""
    assert run(100 * US, 2000 * US, 1000 * US) == ([1] * 32, 0)


def test_arrivals_around_the_limit(run):
    for arrive in range(1800, 2200, 10):
        got, err = run(0, arrive * US, 2000 * US)
        assert len(set(got)) == 1 and err == (0 if got[0] else TIMEOUT)
