"""The queue's generation calls return an error oid when an operand is missing, and never raise
(no GPU needed: nothing is issued)."""
import pytest

from iom_b200.device import OID_INVALID_ARGUMENT, B200Queue
from iom_b200.tensor import DataType
from support import HostTensor

WORD = 0x10000          # never dereferenced


class Device:
    """Stands in for the device that owns the views."""


@pytest.fixture
def queue():
    queue = object.__new__(B200Queue)
    queue._device = Device()
    queue._closed = True                # nothing to close

    def submit(*_args):
        pytest.fail("a call without its operands was issued")
    queue._submit = submit
    return queue


def tensor(queue, shape, dtype=DataType.BF16):
    owner = HostTensor(shape, dtype)
    owner.device = queue._device
    return owner.view()


@pytest.mark.parametrize("missing", range(4))
@pytest.mark.parametrize("scale", [None, 0.125])
def test_attention(queue, missing, scale):
    views = [tensor(queue, s) for s in ((4, 40, 64), (2, 40, 64), (2, 40, 64), (40, 256))]
    views[missing] = None
    assert queue.sdpa_packed(*views, WORD, 1, WORD, scale) == OID_INVALID_ARGUMENT
    views = [tensor(queue, s) for s in ((3, 4, 5, 64), (3, 2, 40, 64), (3, 2, 40, 64), (3, 5, 256))]
    views[missing] = None
    assert queue.sdpa_tree(*views, WORD, 0, 0, WORD, None, scale) == OID_INVALID_ARGUMENT


def test_workspace_requirements(queue):
    q, k = tensor(queue, (3, 4, 5, 64)), tensor(queue, (3, 2, 40, 64))
    for pair in ((None, k), (q, None)):
        with pytest.raises(ValueError):
            queue.sdpa_tree_workspace_requirements(*pair)


def test_compact(queue):
    cache = tensor(queue, (3, 2, 40, 64))
    assert queue.cache_compact(None, None, WORD, WORD, 4, WORD, WORD) == OID_INVALID_ARGUMENT
    assert queue.cache_compact(None, cache, WORD, WORD, 4, WORD, WORD) == OID_INVALID_ARGUMENT


@pytest.mark.parametrize("missing", range(3))
def test_scores(queue, missing):
    views = [tensor(queue, (5, 50)), tensor(queue, (1, 5), DataType.U32), tensor(queue, (1, 5), DataType.F32)]
    views[missing] = None
    assert queue.token_logprobs(*views, None, WORD) == OID_INVALID_ARGUMENT


def test_a_view_of_another_device(queue):
    views = [tensor(queue, s) for s in ((4, 40, 64), (2, 40, 64), (2, 40, 64), (40, 256))]
    views[1].owner.device = Device()
    assert queue.sdpa_packed(*views, WORD, 1, WORD) == OID_INVALID_ARGUMENT
