"""In-place compaction of accepted cache rows (iomb_cache_compact), byte for byte: every leaf
width, odd feature widths, paths that overlap their targets, wrong paths, views."""
import numpy as np
import pytest
import torch

from iom_b200.device import OID_INVALID_ARGUMENT, OID_UNSUPPORTED
from iom_b200.tensor import DataType
from generation_support import device_words
from gpu_support import download, gpu, run, upload  # noqa: F401
from support import NUMPY_OF, HostTensor, logical

pytestmark = pytest.mark.gpu


def random_cache(rng, shape, dtype):
    host = HostTensor(shape, dtype).poison(0xA5)
    kind = np.dtype(NUMPY_OF[dtype])
    host.view().copy_from_host(rng.integers(0, 256, int(np.prod(shape)) * kind.itemsize).astype(np.uint8).view(kind)
                               .reshape(shape))
    return host


def compacted(host, lengths, paths):
    """The formula on the logical values; padding keeps its bytes."""
    want = host.clone()
    values = logical(host.view()).copy()
    moved = values.copy()
    for b, (length, path) in enumerate(zip(lengths, paths)):
        for j, a in enumerate(path):
            moved[b, ..., length + j, :] = values[b, ..., length + a, :]
    want.view().copy_from_host(moved)
    return want.storage


def arrays(paths, width):
    accepted = np.zeros((len(paths), width), dtype=np.int64)
    for b, path in enumerate(paths):
        accepted[b, :len(path)] = path
    return device_words(accepted), device_words([len(p) for p in paths])


def call(queue, k, v, lengths, accepted, width, counts, status):
    return queue.cache_compact(k, v, lengths.data_ptr(), accepted.data_ptr(), width, counts.data_ptr(),
                               status.data_ptr())


@pytest.mark.parametrize("dtype", [DataType.U8, DataType.F8_E4M3FN, DataType.BF16, DataType.F16, DataType.F32,
                                   DataType.F64])
@pytest.mark.parametrize("features", [1, 15, 16, 64, 69, 128])
def test_leaves_and_widths(gpu, dtype, features):
    device, queue = gpu
    rng = np.random.default_rng(features)
    lengths, width = [0, 7, 16, 33, 40], 9
    paths = [[0, 3, 4, 8], [], [8], [0, 1, 2], [1, 2, 3, 4, 5, 6, 7, 8]]
    hosts = [random_cache(rng, (5, 3, 50, features), dtype) for _ in range(2)]
    devs = [upload(device, h) for h in hosts]
    accepted, counts = arrays(paths, width)
    status = device_words([9])
    run(queue, call(queue, devs[0].view(), devs[1].view(), device_words(lengths), accepted, width, counts, status))
    assert int(status.item()) == 0
    for host, dev in zip(hosts, devs):
        assert np.array_equal(download(dev), compacted(host, lengths, paths))


def test_long_paths_overlap_their_targets(gpu):
    """Paths of hundreds of rows: what a row moves onto is read by an earlier step."""
    device, queue = gpu
    rng = np.random.default_rng(4)
    for width, keep in ((256, 200), (600, 599), (64, 40)):
        lengths = [3, 100]
        paths = [sorted(rng.choice(width, keep, replace=False).tolist()), list(range(1, width))]
        host = random_cache(rng, (2, 2, 100 + width, 96), DataType.BF16)
        dev = upload(device, host)
        accepted, counts = arrays(paths, width)
        status = device_words([9])
        run(queue, call(queue, dev.view(), None, device_words(lengths), accepted, width, counts, status))
        assert int(status.item()) == 0
        assert np.array_equal(download(dev), compacted(host, lengths, paths))


def test_wrong_paths_are_skipped_and_reported(gpu):
    device, queue = gpu
    rng = np.random.default_rng(5)
    lengths, width = [0, 0, 0, 45, 0, 0xFFFFFFF0, 10], 8
    paths = [[0, 2, 2], [3, 1], [0, 8], [1, 4, 7], [2, 4], [1], [0, 5]]
    good = [[], [], [], [], [2, 4], [], [0, 5]]
    host = random_cache(rng, (7, 2, 50, 32), DataType.BF16)
    dev = upload(device, host)
    accepted, counts = arrays(paths, width)
    status = device_words([9])
    words = torch.tensor(np.array(lengths, dtype=np.uint32).view(np.int32), device="cuda")
    run(queue, call(queue, dev.view(), None, words, accepted, width, counts, status))
    assert int(status.item()) == 1
    assert np.array_equal(download(dev), compacted(host, [0, 0, 0, 0, 0, 0, 10], good))
    dev = upload(device, host)
    counts[0] = 9           # more rows than a path holds
    run(queue, call(queue, dev.view(), None, words, accepted, width, counts, status))
    assert int(status.item()) == 1
    assert np.array_equal(download(dev), compacted(host, [0, 0, 0, 0, 0, 0, 10], good))


def test_layers_first_owner_and_interleaved_views(gpu):
    """[layers, B, heads, C, D] caches with the batch brought to the front."""
    device, queue = gpu
    rng = np.random.default_rng(6)
    hosts = [random_cache(rng, (3, 4, 2, 40, 48), DataType.BF16) for _ in range(2)]
    devs = [upload(device, h) for h in hosts]
    lengths, width = [0, 9, 20, 31], 8
    paths = [[1, 5], [0, 7], [], [2, 3, 4]]
    accepted, counts = arrays(paths, width)
    status = device_words([9])
    views = [d.view().slice(0, 0, 2, 2).permute([1, 0, 2]) for d in devs]       # layers 0 and 2
    run(queue, call(queue, views[0], views[1], device_words(lengths), accepted, width, counts, status))
    assert int(status.item()) == 0
    for host, dev in zip(hosts, devs):
        want = host.clone()
        values = logical(host.view()).copy()
        moved = values.copy()
        for b, path in enumerate(paths):
            for j, a in enumerate(path):
                moved[[0, 2], b, :, lengths[b] + j] = values[[0, 2], b, :, lengths[b] + a]
        want.view().copy_from_host(moved)
        assert np.array_equal(download(dev), want.storage)


def test_refusals(gpu):
    device, queue = gpu
    host = random_cache(np.random.default_rng(1), (2, 2, 20, 16), DataType.BF16)
    k, v = upload(device, host), upload(device, host)
    words = device_words([0, 0])
    accepted, counts = arrays([[0], [0]], 4)
    status = device_words([9])
    assert call(queue, k.view(), k.view(), words, accepted, 4, counts, status) == OID_INVALID_ARGUMENT
    assert call(queue, k.view(), v.view().select(0, 0), words, accepted, 4, counts, status) == OID_INVALID_ARGUMENT
    assert call(queue, k.view(), v.view(), words, accepted, 0, counts, status) == OID_INVALID_ARGUMENT
    assert queue.cache_compact(k.view(), v.view(), 0, accepted.data_ptr(), 4, counts.data_ptr(),
                               status.data_ptr()) == OID_INVALID_ARGUMENT
    narrow = upload(device, HostTensor((2, 2, 20, 16), DataType.U4))
    assert call(queue, narrow.view(), None, words, accepted, 4, counts, status) == OID_UNSUPPORTED
    assert np.array_equal(download(k), host.storage)
