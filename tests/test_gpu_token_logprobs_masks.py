"""Scores of rows whose tokens are ruled out by the leaf's lowest finite value, as attention and
grammar masks often do instead of -inf: such logits are ordinary values of weight zero, and the
entropy, the log probabilities and the best tokens are those of the formula."""
import numpy as np
import pytest

from iom_b200.tensor import DataType
from gpu_support import gpu, run  # noqa: F401
from test_gpu_token_logprobs import Scores

pytestmark = pytest.mark.gpu

LOWEST = {DataType.BF16: -3.3895313892515355e38, DataType.F16: -65504.0, DataType.F32: -3.4028234663852886e38}


@pytest.mark.parametrize("dtype", list(LOWEST))
@pytest.mark.parametrize("rows,vocab", [(1, 40), (18, 3000), (3, 32000), (40, 777)])
def test_the_lowest_value_as_a_mask(gpu, dtype, rows, vocab):
    device, queue = gpu
    low = LOWEST[dtype]
    rng = np.random.default_rng(vocab)
    at = np.arange(vocab)
    masks = {
        "first": np.broadcast_to(at < vocab // 2, (rows, vocab)),
        "last": np.broadcast_to(at >= vocab // 2, (rows, vocab)),
        "most": np.broadcast_to(at % 37 != 5, (rows, vocab)),
        "all but the last": np.broadcast_to(at != vocab - 1, (rows, vocab)),
        "all": np.ones((rows, vocab), dtype=bool),
        "here and there": rng.random((rows, vocab)) < 0.4,
        "pieces of 16": np.broadcast_to(at // 16 % 2 == 0, (rows, vocab)),
    }
    for name, mask in masks.items():
        values = np.where(mask, low, rng.normal(0, 2.5, (rows, vocab)))
        if name == "here and there":
            values[:, ::11] = -np.inf
        tokens = rng.integers(0, vocab, rows)
        case = Scores(device, values, dtype, tokens, min(12, vocab))
        run(queue, case.issue(queue))
        case.check()


@pytest.mark.parametrize("dtype", list(LOWEST))
def test_large_negative_values_of_every_size(gpu, dtype):
    """A running maximum that climbs from any of these to an ordinary logit."""
    device, queue = gpu
    rng = np.random.default_rng(1)
    sizes = [s for s in (1e2, 1e3, 6e4, 1e10, 1e30, 1e37, 3e38) if s <= -LOWEST[dtype]]
    values = rng.normal(0, 1, (len(sizes), 2000))
    for row, size in enumerate(sizes):
        values[row, :1700] -= size
    case = Scores(device, values, dtype, rng.integers(0, 2000, len(sizes)), 8)
    run(queue, case.issue(queue))
    case.check()
