"""iomb_cache_compact on keys and values whose planes alternate inside one owner: distinct planes,
so one call takes both; planes in common are refused."""
import numpy as np
import pytest

from iom_b200.device import OID_INVALID_ARGUMENT
from iom_b200.tensor import DataType, TensorSpec, TensorView
from generation_support import device_words
from gpu_support import download, gpu, run, upload  # noqa: F401
from support import logical
from test_gpu_cache_compact import arrays, call, random_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,axis", [
    ((3, 2, 4, 40, 64), 1),         # [B, 2, H, C, D]
    ((2, 3, 4, 40, 64), 0),         # [2, B, H, C, D]
    ((3, 4, 2, 40, 64), 2),         # [B, H, 2, C, D]
    ((3, 5, 2, 2, 40, 64), 2),      # [B, layers, 2, H, C, D]
    ((1, 2, 1, 40, 64), 1),
])
def test_alternating_planes(gpu, shape, axis):
    device, queue = gpu
    rng = np.random.default_rng(axis)
    host = random_cache(rng, shape, DataType.BF16)
    dev = upload(device, host)
    k, v = dev.view().select(axis, 0), dev.view().select(axis, 1)
    batch = k.spec.shape[0]
    lengths, paths = [0, 7, 20][:batch], [[1, 3, 4, 8], [], [2, 9]][:batch]
    accepted, counts = arrays(paths, 10)
    status = device_words([9])
    run(queue, call(queue, k, v, device_words(lengths), accepted, 10, counts, status))
    assert int(status.item()) == 0
    values = logical(host.view())
    moved = values.copy()
    for which in range(2):
        source, target = np.take(values, which, axis), np.moveaxis(moved, axis, 0)[which]
        for b, (length, path) in enumerate(zip(lengths, paths)):
            for j, a in enumerate(path):
                target[b, ..., length + j, :] = source[b, ..., length + a, :]
    want = host.clone()
    want.view().copy_from_host(moved)
    assert np.array_equal(download(dev), want.storage)


def test_planes_in_common_are_refused(gpu):
    device, queue = gpu
    dev = upload(device, random_cache(np.random.default_rng(1), (20, 40, 64), DataType.BF16))
    accepted, counts = arrays([[1], [1], [1]], 4)
    lengths, status = device_words([0, 0, 0]), device_words([9])
    spec = TensorSpec((3, 2, 40, 64), DataType.BF16)

    def planes(offset, *strides):
        return TensorView(dev, spec, offset, strides)
    for k, v in ((planes(0, 2, 1), planes(0, 2, 1)), (planes(0, 4, 1), planes(1, 4, 1)), (planes(0, 4, 1), planes(4, 4, 1)),
                 (planes(3, 4, 1), planes(0, 4, 1)), (planes(0, 2, 1), planes(5, 2, 1)), (planes(0, 4, 1), planes(2, 3, 1))):
        assert call(queue, k, v, lengths, accepted, 4, counts, status) == OID_INVALID_ARGUMENT
    for k, v in ((planes(0, 4, 1), planes(2, 4, 1)), (planes(0, 2, 1), planes(6, 2, 1)), (planes(6, 2, 1), planes(0, 2, 1)),
                 (planes(1, 4, 2), planes(0, 4, 2))):
        run(queue, call(queue, k, v, lengths, accepted, 4, counts, status))
