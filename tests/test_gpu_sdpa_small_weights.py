"""F16 weights far below the largest one: many tokens of small weight add up to what the formula
gives.

Every token but the first has the weight 2^-26.5 of the first one's, in one pass over the row. The
kernel holds weights as F16 multiples of 2^-7 of the reference, where such a one is 2^-19.5: above
half of the smallest F16 value, 2^-25, and rounded to a multiple of 2^-24, so off by at most 2^-25,
which is 2^-32 of the reference. Over n tokens of value one, against a sum of at least one: n 2^-32.
The first token's value is zero, so nothing else of the result's size is rounded but the result."""
import numpy as np
import pytest

from iom_b200.tensor import DataType
from gpu_support import download, gpu, run  # noqa: F401
from generation_support import decode
from support import logical
from test_gpu_sdpa_packed import Packed
from test_gpu_sdpa_tree import Tree

pytestmark = pytest.mark.gpu

GAP = 26.5 * np.log(2.0)


def edit(v):
    v["q"][:] = 0
    v["q"][..., 0] = 1.0
    v["k"][:] = 0
    v["k"][..., 0, 0] = GAP         # rounded to F16: the test goes by the rounded one
    v["v"][:] = 1.0
    v["v"][..., 0, :] = 0.0


def wanted(gap, n):
    small = (n - 1) * np.exp(-gap)
    want = small / (1 + small)
    # weights, then the relative roundings: exponentials and sums (2^-18 covers them), the result (2^-11)
    return want, n * 2.0 ** -32 + want * (2.0 ** -11 + 2.0 ** -18 + n * 2.0 ** -24) + 2.0 ** -25


def test_packed(gpu):
    device, queue = gpu
    n = 60000
    case = Packed(device, DataType.F16, 2, 1, 16, [0, n], edit=edit)
    run(queue, case.issue(queue, 1.0))
    assert int(case.status.item()) == 0
    out = case.host["out"].clone()
    out.storage[:] = download(case.dev["out"])
    got = decode(logical(out.view()), DataType.F16)
    gap = float(decode(case.codes["k"], DataType.F16)[0, 0, 0])
    for r in (1, 2000, 30001, n - 1):
        want, tolerance = wanted(gap, r + 1)
        assert np.all(np.abs(got[r] - want) <= tolerance), (r, got[r].min(), got[r].max(), want, tolerance)


@pytest.mark.parametrize("nodes", [1, 130])
def test_tree(gpu, nodes):
    """Many sequences, so that a cache of 8 blocks stays whole; long ones are cut and joined."""
    device, queue = gpu
    for batch, length in ((48, 1000 - nodes), (1, 40000)):
        case = Tree(device, DataType.F16, 1, 1, 16, nodes, length + nodes, [length] * batch, parents=None, edit=edit)
        run(queue, case.issue(queue, 1.0))
        assert int(case.words["status"].item()) == 0
        out = case.host["out"].clone()
        out.storage[:] = download(case.dev["out"])
        got = decode(logical(out.view()), DataType.F16).reshape(batch, nodes, 16)
        gap = float(decode(case.codes["k"], DataType.F16)[0, 0, 0, 0])
        for i in {0, nodes - 1}:
            want, tolerance = wanted(gap, length + i + 1)
            assert np.all(np.abs(got[:, i] - want) <= tolerance), (length, i, got[:, i].min(), got[:, i].max(), want)
