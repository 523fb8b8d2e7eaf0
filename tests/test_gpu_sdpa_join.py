"""Ranges of a cut cache whose sums say less than their scores: a range with no weight left is
dropped from a row only when the row sees nothing in it."""
import numpy as np
import pytest

from iom_b200.tensor import DataType
from gpu_support import download, gpu, run  # noqa: F401
from support import logical
from test_gpu_sdpa_tree import Tree

pytestmark = pytest.mark.gpu


def codes(case):
    out = case.host["out"].clone()
    out.storage[:] = download(case.dev["out"])
    return logical(out.view()).reshape(case.batch, case.nodes, case.hq, case.width)


@pytest.mark.parametrize("hq,nodes", [(4, 1), (8, 40)])
@pytest.mark.parametrize("token", [0, 130, 3000, 4999])
def test_a_score_whose_product_with_log2e_overflows(gpu, hq, nodes, token):
    """One token's score is 1.5 * 2^127 (finite; times log2(e) it is not), all others are zero: it
    holds all the weight, and the result is its value, exactly."""
    device, queue = gpu

    def edit(v):
        v["q"][:] = 0
        v["q"][..., 0] = 2.0 ** 64
        v["k"][:] = 0
        v["k"][:, :, token, 0] = 1.5 * 2.0 ** 63
    case = Tree(device, DataType.BF16, hq, 2, 64, nodes, 6000, [5000], seed=token, parents=None, edit=edit)
    run(queue, case.issue(queue, 1.0))
    assert int(case.words["status"].item()) == 0
    got = codes(case)
    for h in range(hq):
        want = case.codes["v"][0, h // (hq // 2), token]
        want = np.where(want == 0x8000, 0, want)
        assert np.array_equal(got[0, :, h], np.broadcast_to(want, got[0, :, h].shape))


@pytest.mark.parametrize("hq,nodes", [(4, 1), (8, 40)])
def test_values_under_scores_of_minus_infinity(gpu, hq, nodes):
    """Visible tokens whose scores are -inf have weight zero, and zero times an infinite value is
    NaN, as in the formula, also where they fill ranges of their own."""
    device, queue = gpu

    def edit(v):
        v["q"][..., 0] = 1.0
        v["k"][:, :, 1000:4000, 0] = -np.inf
        v["v"][:, 0, 2000, 3] = np.inf
    case = Tree(device, DataType.BF16, hq, 2, 64, nodes, 6000, [5000], seed=1, parents=None, edit=edit)
    run(queue, case.issue(queue))
    case.check(nodes=sorted({0, nodes - 1}))
