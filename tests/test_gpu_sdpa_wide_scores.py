"""Scores at both ends of binary32 under a scale that brings them close together: the differences
between scores overflow, the differences between scaled scores do not."""
import numpy as np
import pytest

from iom_b200.tensor import DataType
from gpu_support import download, gpu, run  # noqa: F401
from generation_support import UNIT, attend, check_rows, decode
from support import logical
from test_gpu_sdpa_packed import Packed
from test_gpu_sdpa_tree import Tree

pytestmark = pytest.mark.gpu

SCALE = 1.25e-38            # a normal binary32 value


def far_apart(v, cut):
    """Scores of -1.375 * 2^127 before `cut`, of +1.375 * 2^127 from there on: 5.8 apart when scaled."""
    v["q"][:] = 0
    v["q"][..., 0] = 2.0 ** 64
    v["k"][:] = 0
    v["k"][..., :cut, 0] = -1.375 * 2.0 ** 63
    v["k"][..., cut:, 0] = 1.375 * 2.0 ** 63
    v["v"][..., :cut, :] += 3.0


def test_packed(gpu):
    device, queue = gpu
    case = Packed(device, DataType.BF16, 4, 2, 32, [0, 700], seed=1, edit=lambda v: far_apart(v, 512))
    run(queue, case.issue(queue, SCALE))
    case.check(scale=SCALE, rows=[0, 100, 511, 512, 513, 600, 699])


@pytest.mark.parametrize("cap,length,nodes", [(400, 300, 1), (6000, 5000, 1), (6000, 5000, 70)])
def test_tree(gpu, cap, length, nodes):
    device, queue = gpu
    case = Tree(device, DataType.BF16, 4, 2, 32, nodes, cap, [length], seed=2, parents=None,
                edit=lambda v: far_apart(v, length - 40))
    run(queue, case.issue(queue, SCALE))
    assert int(case.words["status"].item()) == 0
    out = case.host["out"].clone()
    out.storage[:] = download(case.dev["out"])
    got = logical(out.view()).reshape(nodes, 4, 32)
    value = {n: decode(c, case.dtype) for n, c in case.codes.items()}
    scale = float(np.float32(SCALE))
    for i in sorted({0, nodes - 1}):
        rows = case.seen(0, i)
        for h in range(4):
            want, tolerance = attend(value["q"][0, h, i], value["k"][0, h // 2][rows], value["v"][0, h // 2][rows], scale,
                                     UNIT[case.dtype], False)
            check_rows(got[i, h], want, tolerance, case.dtype)
