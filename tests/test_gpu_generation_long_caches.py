"""The serving loop of test_gpu_generation_loop over caches long enough to be cut into ranges, with
short and long sequences side by side and one workspace whose leftovers are finite: eager steps,
replayed steps, and a sequence that ends and gives its place to a new one."""
import ctypes

import numpy as np
import pytest
import torch

from iom_b200.tensor import DataType
from generation_support import decode, encode
from gpu_support import gpu  # noqa: F401
import test_gpu_generation_loop as steps

pytestmark = pytest.mark.gpu

CAP = 2500


def begin(loop, rng, b, length):
    """Sequence b starts over with `length` rows in its caches."""
    for n in ("k", "v"):
        loop.host[n][b] = 0
        loop.host[n][b][:, :length] = decode(encode(rng.normal(0, 1, (steps.HKV, length, steps.D)), DataType.BF16),
                                             DataType.BF16)
        loop.put(n, loop.host[n])
    loop.lengths[b] = length


def test_serving_loop_over_long_caches(gpu, monkeypatch):
    monkeypatch.setattr(steps, "CAP", CAP)
    device, queue = gpu
    rng = np.random.default_rng(5)
    loop = steps.Loop(device, queue)
    need = queue.sdpa_tree_workspace_requirements(loop.dev["q"].view(), loop.dev["k"].view()).bytes
    assert need > 0
    loop.workspace.tensor()[:need // 4 * 4].view(torch.float32).fill_(2.0)
    for b, length in enumerate((2000, 1, 130)):
        begin(loop, rng, b, length)
    for _ in range(3):
        step = steps.draft(loop, rng)
        tokens = loop.step_operations()
        assert all(t > 0 for t in tokens)
        queue.wait(tokens[-1])
        steps.check_step(loop, *step)
    with queue.capture() as sequence:
        loop.step_operations()
    for turn, (b, length) in enumerate(((0, 5), (1, 1500), (2, 255), (0, 129), (1, 3), (0, 2400), (2, 2470))):
        begin(loop, rng, b, length)
        step = steps.draft(loop, rng)
        if turn % 2:
            queue.wait(loop.step_operations()[-1])
        else:
            queue.wait(sequence.replay())
        steps.check_step(loop, *step)
    sequence.close()
    count = ctypes.c_uint(99)
    assert device._lib.iomb_sdpa_wait_timeouts(ctypes.byref(count)) == 0 and count.value == 0
