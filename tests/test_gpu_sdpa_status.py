"""The status word of the attention calls is the call's own: whatever it held, of this or another
call, does not stay in it. (2, a wait that gave up, cannot be brought about without stopping a
kernel's own copies, and is not.)"""
import pytest
import torch

from iom_b200.tensor import DataType
from generation_support import device_words
from gpu_support import gpu, run  # noqa: F401
from test_gpu_sdpa_packed import Packed
from test_gpu_sdpa_tree import Tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,nodes,cap", [(64, 3, 200), (64, 3, 3000), (128, 100, 3000), (24, 3, 200)])
def test_tree(gpu, width, nodes, cap):
    device, queue = gpu
    case = Tree(device, DataType.BF16, 4, 2, width, nodes, cap, [20, 150 - nodes])
    run(queue, case.issue(queue))
    with queue.capture() as step:
        case.issue(queue)
    status = case.words["status"]
    for before, lengths, want in ((-1, [20, 50], 0), (-1, [20, cap], 1), (1, [20, 50], 0), (2, [cap, 0], 1), (0, [cap, 0], 1),
                                  (1, [0, cap - nodes], 0)):
        for call in (lambda: case.issue(queue), step.replay):
            status.fill_(before)
            case.words["lengths"].copy_(device_words(lengths))
            torch.cuda.synchronize()
            queue.wait(call())
            assert int(status.item()) == want
    step.close()


@pytest.mark.parametrize("width", [64, 24])
def test_packed(gpu, width):
    device, queue = gpu
    case = Packed(device, DataType.BF16, 4, 2, width, [0, 30, 200])
    for before, borders, want in ((-1, [0, 30, 200], 0), (-1, [0, 30, 201], 1), (1, [5, 5, 5], 0), (2, [9, 8, 200], 1)):
        case.status.fill_(before)
        case.offsets.copy_(device_words(borders))
        torch.cuda.synchronize()
        run(queue, case.issue(queue))
        assert int(case.status.item()) == want
