"""The workspace of iomb_sdpa_tree needs no set-up: whatever finite values it holds, from nobody or
from earlier calls, do not reach a result. The ranges of a call are fixed by the cache's capacity,
so short live lengths in a large cache leave ranges without a block, and their partials unwritten;
NaN there would only be noticed as a row to compute again, so the values here are finite."""
import numpy as np
import pytest
import torch

from iom_b200.tensor import DataType
from generation_support import device_words
from gpu_support import download, gpu, run  # noqa: F401
from test_gpu_sdpa_tree import Tree

pytestmark = pytest.mark.gpu


def give_workspace(device, queue, case, value):
    need = queue.sdpa_tree_workspace_requirements(case.dev["q"].view(), case.dev["k"].view())
    assert need.bytes, "the case is meant to be cut into ranges"
    case.workspace = device.create_workspace(need.bytes)
    case.workspace.tensor().view(torch.float32).fill_(value)
    torch.cuda.synchronize()


@pytest.mark.parametrize("value", [3.0, -0.5, 1e30])
@pytest.mark.parametrize("dtype,hq,hkv,width,nodes,cap,lengths", [
    # up to 128 rows per key/value head
    (DataType.BF16, 32, 4, 64, 1, 4096, [200]),
    (DataType.BF16, 4, 4, 64, 1, 4096, [130]),
    (DataType.F16, 8, 8, 128, 1, 4096, [255, 300]),
    (DataType.BF16, 2, 1, 64, 3, 3000, [1000]),
    (DataType.F16, 3, 1, 80, 7, 9000, [0, 700, 121]),
    # more of them
    (DataType.BF16, 8, 2, 64, 64, 4096, [100, 300]),
    (DataType.F16, 16, 1, 128, 32, 4096, [500]),
    (DataType.BF16, 4, 2, 16, 100, 3000, [0, 29, 1500]),
])
def test_unwritten_partials_are_not_read(gpu, dtype, hq, hkv, width, nodes, cap, lengths, value):
    device, queue = gpu
    case = Tree(device, dtype, hq, hkv, width, nodes, cap, lengths, seed=cap + width)
    give_workspace(device, queue, case, value)
    run(queue, case.issue(queue))
    case.check(nodes=sorted({0, nodes // 2, nodes - 1}), heads=sorted({0, hq // 2, hq - 1}))


@pytest.mark.parametrize("hq,hkv,width,nodes", [(8, 8, 64, 1), (16, 2, 64, 32), (4, 1, 128, 5)])
def test_one_workspace_while_the_lengths_grow_and_shrink(gpu, hq, hkv, width, nodes):
    """A decode that starts in an empty cache of its full capacity, eager and replayed in turn, and a
    shorter sequence in its place afterwards: the same bits as with a workspace of its own."""
    device, queue = gpu
    cap = 4096
    case = Tree(device, DataType.BF16, hq, hkv, width, nodes, cap, [1], seed=width)
    give_workspace(device, queue, case, 0.0)
    run(queue, case.issue(queue))
    with queue.capture() as step:
        case.issue(queue)
    lengths = list(range(1, cap - nodes, 128 if nodes == 1 else 384)) + [cap - nodes, 2433, 200, 1, 515, 0]
    heads = sorted({0, hq // 2, hq - 1})
    for turn, length in enumerate(lengths):
        case.lengths = [length]
        case.words["lengths"].copy_(device_words([length]))
        torch.cuda.synchronize()
        if turn % 2:
            queue.wait(step.replay())
        else:
            run(queue, case.issue(queue))
        case.check(nodes=sorted({0, nodes - 1}), heads=heads)
        bits = download(case.dev["out"]).copy()
        used, case.workspace = case.workspace, None
        give_workspace(device, queue, case, 0.0)
        run(queue, case.issue(queue))
        assert np.array_equal(bits, download(case.dev["out"]))
        case.workspace.close()
        case.workspace = used
    step.close()
