"""Attention of drafted token trees over KV caches (iomb_sdpa_tree) against the formula in 64
bits: trees, chains and single tokens, head groups, caches from empty to long (ranges cut over
the SMs and joined), nodes not in use, stale and NaN rows behind the live ones, wrong arguments,
views, captured sequences."""
import numpy as np
import pytest
import torch

from iom_b200.device import OID_INVALID_ARGUMENT, OID_UNSUPPORTED
from iom_b200.tensor import DataType
from generation_support import UNIT, attend, check_rows, decode, device_words, encode, host_tensor
from gpu_support import download, gpu, run, upload  # noqa: F401
from support import HostTensor, logical

pytestmark = pytest.mark.gpu


def random_parents(rng, batch, nodes):
    return np.array([[int(rng.integers(-1, i)) if i else -1 for i in range(nodes)] for _ in range(batch)],
                    dtype=np.int32).reshape(batch, nodes)


class Tree:
    def __init__(self, device, dtype, hq, hkv, width, nodes, cap, lengths, counts=None, parents="random", seed=0,
                 edit=None):
        rng = np.random.default_rng(seed)
        self.batch = len(lengths)
        self.dtype, self.hq, self.hkv, self.width, self.nodes, self.cap = dtype, hq, hkv, width, nodes, cap
        self.lengths = list(lengths)
        self.counts = list(counts) if counts is not None else [nodes] * self.batch
        self.parents = random_parents(rng, self.batch, nodes) if isinstance(parents, str) else parents
        values = {"q": rng.normal(0, 1.5, (self.batch, hq, nodes, width)),
                  "k": rng.normal(0, 1, (self.batch, hkv, cap, width)),
                  "v": rng.normal(0, 1, (self.batch, hkv, cap, width))}
        if edit is not None:
            edit(values)
        self.codes = {n: encode(x, dtype) for n, x in values.items()}
        self.host = {n: host_tensor(c, dtype) for n, c in self.codes.items()}
        self.host["out"] = HostTensor((self.batch, nodes, hq * width), dtype).poison(0x3C)
        self.dev = {n: upload(device, h) for n, h in self.host.items()}
        self.words = {"lengths": device_words(self.lengths), "status": device_words([77])}
        if counts is not None:
            self.words["counts"] = device_words(self.counts)
        if self.parents is not None:
            self.words["parents"] = device_words(self.parents)
        self.device = device
        self.workspace = None

    def issue(self, queue, scale=None):
        d, w = self.dev, self.words
        need = queue.sdpa_tree_workspace_requirements(d["q"].view(), d["k"].view())
        if self.workspace is None and need.bytes:
            self.workspace = self.device.create_workspace(need.bytes)
            self.workspace.tensor().fill_(0xFF)         # whatever it holds does not matter

        def address(name):
            return w[name].data_ptr() if name in w else 0
        return queue.sdpa_tree(d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view(), address("lengths"),
                               address("parents"), address("counts"), address("status"),
                               self.workspace.view() if self.workspace is not None else None, scale)

    def seen(self, b, i):
        rows = list(range(self.lengths[b]))
        path, at = [], i
        while at >= 0:
            path.append(self.lengths[b] + at)
            if self.parents is None:
                at -= 1
            else:
                parent = int(self.parents[b][at])
                at = parent if parent < at else -1
        return rows + sorted(path)

    def check(self, nodes=None, heads=None, status=0, skipped=()):
        assert int(self.words["status"].item()) == status
        out = self.host["out"].clone()
        out.storage[:] = download(self.dev["out"])
        got = logical(out.view()).reshape(self.batch, self.nodes, self.hq, self.width)
        out.view().copy_from_host(np.full((self.batch, self.nodes, self.hq * self.width), 0x3C3C, dtype=np.uint16))
        assert np.all(out.storage == 0x3C), "padding of the output changed"
        value = {n: decode(c, self.dtype) for n, c in self.codes.items()}
        scale = float(np.float32(self.width ** -0.5))
        for b in range(self.batch):
            live = 0 if b in skipped else self.counts[b]
            assert np.all(got[b, live:] == 0x3C3C), "rows of nodes not in use changed"
            for i in range(live) if nodes is None else [i for i in nodes if i < live]:
                rows = self.seen(b, i)
                for h in range(self.hq) if heads is None else heads:
                    g = h // (self.hq // self.hkv)
                    want, tol = attend(value["q"][b, h, i], value["k"][b, g][rows], value["v"][b, g][rows], scale,
                                       UNIT[self.dtype], self.dtype == DataType.F16)
                    check_rows(got[b, i, h], want, tol, self.dtype)


@pytest.mark.parametrize("dtype", [DataType.BF16, DataType.F16])
@pytest.mark.parametrize("hq,hkv,width,nodes", [
    (4, 1, 64, 1), (32, 4, 64, 1), (8, 8, 128, 1), (6, 2, 80, 5), (4, 2, 64, 17), (8, 2, 32, 33), (16, 2, 64, 16),
    (24, 8, 96, 3), (2, 2, 128, 64), (32, 8, 128, 64), (3, 1, 16, 100), (12, 1, 64, 31), (5, 1, 48, 256),
    (4, 2, 20, 7), (2, 1, 256, 3),
])
def test_head_groups_and_nodes(gpu, dtype, hq, hkv, width, nodes):
    device, queue = gpu
    lengths = [0, 1, 16, 100, 130]
    case = Tree(device, dtype, hq, hkv, width, nodes, 130 + nodes, lengths, seed=nodes + width)
    run(queue, case.issue(queue))
    case.check(nodes=range(0, nodes, max(1, nodes // 6)), heads=range(0, hq, max(1, hq // 4)))


@pytest.mark.parametrize("lengths,cap,nodes", [
    ([0], 1, 1), ([0], 200, 1), ([126], 127, 1), ([127], 128, 1), ([128], 129, 1), ([255, 256, 257], 300, 2),
    ([0, 0, 0], 20, 4), ([5, 300, 0, 1, 77, 1023], 1040, 8), ([2047], 2048, 1), ([120], 256, 136),
])
def test_cache_borders(gpu, lengths, cap, nodes):
    device, queue = gpu
    for parents in ("random", None):
        case = Tree(device, DataType.BF16, 4, 2, 64, nodes, cap, lengths, seed=cap, parents=parents)
        run(queue, case.issue(queue))
        case.check(nodes=range(0, nodes, max(1, nodes // 9)))


@pytest.mark.parametrize("dtype,hq,hkv,width,nodes,lengths,cap", [
    (DataType.BF16, 8, 1, 64, 1, [20000], 20011),
    (DataType.F16, 24, 8, 80, 5, [9000, 4097], 9100),
    (DataType.BF16, 32, 4, 64, 1, [int(x) for x in np.random.default_rng(1).integers(0, 2047, 40)], 2048),
    (DataType.BF16, 8, 2, 128, 64, [3000, 17, 0], 3100),
    (DataType.F16, 4, 2, 128, 160, [1500, 900], 1700),
])
def test_long_caches(gpu, dtype, hq, hkv, width, nodes, lengths, cap):
    device, queue = gpu
    case = Tree(device, dtype, hq, hkv, width, nodes, cap, lengths, seed=cap)
    run(queue, case.issue(queue))
    case.check(nodes=sorted({0, 1, 2, nodes // 2, nodes - 1}), heads=sorted({0, 1, hq - 1}))


def test_nodes_not_in_use_and_ragged_counts(gpu):
    device, queue = gpu
    for dtype, hq, hkv, width in ((DataType.BF16, 4, 2, 64), (DataType.F16, 8, 1, 128), (DataType.BF16, 2, 2, 24)):
        case = Tree(device, dtype, hq, hkv, width, 20, 400, [10, 380, 0, 200, 33], counts=[0, 20, 1, 7, 0], seed=5)
        run(queue, case.issue(queue))
        case.check()


def test_stale_rows_behind_the_tree_and_masked_nodes(gpu):
    """NaN and infinities in rows no node sees, and in nodes that only their descendants see."""
    device, queue = gpu
    parents = np.array([[-1, 0, 0, 1, 2, 3, -1, 6]], dtype=np.int32).repeat(2, axis=0)

    def edit(v):
        v["k"][0, :, 60 + 8:] = np.nan
        v["v"][0, :, 60 + 8:] = np.inf
        v["v"][1, :, 130 + 2] = np.nan      # node 2: its child 4 only
        v["k"][1, 0, 130 + 6] = np.nan      # node 6 (a root): itself and 7
        v["v"][1, 1, 130 + 1] = -np.inf     # node 1: 3 and 5
    for width in (64, 40):
        for heads in ((4, 2), (32, 2)):
            case = Tree(device, DataType.BF16, *heads, width, 8, 200, [60, 130], parents=parents, seed=8, edit=edit)
            run(queue, case.issue(queue))
            case.check()


def test_nan_inside_a_long_prefix(gpu):
    device, queue = gpu

    def edit(v):
        v["v"][0, 0, 3000, 5] = np.nan
        v["k"][0, 1, 100] = np.inf      # mixed signs: NaN scores
        v["q"][1, 0, 0] = np.nan
    case = Tree(device, DataType.BF16, 4, 2, 64, 3, 6000, [5000, 4000], seed=8, edit=edit)
    run(queue, case.issue(queue))
    case.check()


@pytest.mark.parametrize("width", [64, 24])
def test_wrong_arguments_are_reported(gpu, width):
    device, queue = gpu
    # a sequence that does not fit is skipped, the others are served
    case = Tree(device, DataType.BF16, 4, 2, width, 6, 300, [10, 297, 0xFFFFFFFF - 2, 250], counts=[6, 6, 6, 6], seed=1)
    run(queue, case.issue(queue))
    case.check(status=1, skipped=(1, 2))
    case = Tree(device, DataType.BF16, 4, 2, width, 6, 300, [10, 20, 30], counts=[6, 7, 0xFFFFFFFF], seed=1)
    run(queue, case.issue(queue))
    case.check(status=1, skipped=(1, 2))
    # a parent that is not before its node makes a root
    parents = np.array([[-1, 1, 5, 0, 3, 2]], dtype=np.int32)
    case = Tree(device, DataType.BF16, 4, 2, width, 6, 300, [100], parents=parents, seed=1)
    run(queue, case.issue(queue))
    case.check(status=1)
    parents = np.array([[-1, -2, -5, 0, 3, 2]], dtype=np.int32)
    case = Tree(device, DataType.BF16, 4, 2, width, 6, 300, [100], parents=parents, seed=1)
    run(queue, case.issue(queue))
    case.check(status=1)
    # nodes not in use may hold anything
    parents = np.array([[-1, 0, 99, 77, -9, 5]], dtype=np.int32)
    case = Tree(device, DataType.BF16, 4, 2, width, 6, 300, [100], counts=[2], parents=parents, seed=1)
    run(queue, case.issue(queue))
    case.check()


def test_strided_caches_and_batches(gpu):
    """Caches as one layer of [layers, B, 2, Hkv, C, D] owners; queries head-major."""
    device, queue = gpu
    rng = np.random.default_rng(3)
    owner = host_tensor(rng.normal(0, 1, (2, 3, 2, 2, 90, 64)), DataType.BF16)
    queries = host_tensor(rng.normal(0, 1, (4, 3, 5, 64)), DataType.BF16)       # [Hq, B, N, D]
    dev, dq = upload(device, owner), upload(device, queries)
    out = upload(device, HostTensor((3, 5, 256), DataType.BF16).poison(0x3C))
    layer = dev.view().select(0, 1)
    k, v = layer.select(1, 0), layer.select(1, 1)
    q = dq.view().permute([1, 0])
    lengths = [80, 0, 33]
    words = [device_words(lengths), device_words([9])]
    need = queue.sdpa_tree_workspace_requirements(q, k)
    ws = device.create_workspace(need.bytes) if need.bytes else None
    run(queue, queue.sdpa_tree(q, k, v, out.view(), words[0].data_ptr(), 0, 0, words[1].data_ptr(),
                               ws.view() if ws else None))
    values = decode(logical(owner.view()), DataType.BF16)[1]
    qv = decode(logical(queries.view()), DataType.BF16)
    host = HostTensor((3, 5, 256), DataType.BF16)
    host.storage[:] = download(out)
    got = logical(host.view()).reshape(3, 5, 4, 64)
    for b in range(3):
        for i in range(5):
            for h in range(4):
                end = lengths[b] + i + 1
                want, tol = attend(qv[h, b, i], values[b, 0, h // 2, :end], values[b, 1, h // 2, :end], 0.125,
                                   UNIT[DataType.BF16], False)
                check_rows(got[b, i, h], want, tol, DataType.BF16)


def test_refusals(gpu):
    device, queue = gpu
    case = Tree(device, DataType.BF16, 4, 2, 64, 6, 300, [10])
    run(queue, case.issue(queue))
    d, w = case.dev, case.words
    views = (d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view())
    ws = case.workspace.view() if case.workspace is not None else None
    assert queue.sdpa_tree(*views, 0, 0, 0, w["status"].data_ptr(), ws) == OID_INVALID_ARGUMENT
    if ws is not None:
        assert queue.sdpa_tree(*views, w["lengths"].data_ptr(), 0, 0, w["status"].data_ptr()) == OID_INVALID_ARGUMENT
        assert queue.sdpa_tree(*views, w["lengths"].data_ptr(), 0, 0, w["status"].data_ptr(),
                               ws.subrange(0, 64)) == OID_INVALID_ARGUMENT
    big = Tree(device, DataType.BF16, 1, 1, 16, 257, 300, [10])
    d = big.dev
    assert queue.sdpa_tree(d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view(), big.words["lengths"].data_ptr(),
                           0, 0, big.words["status"].data_ptr(), ws) == OID_UNSUPPORTED


def test_captured_decode_follows_the_lengths(gpu):
    device, queue = gpu
    case = Tree(device, DataType.BF16, 32, 4, 64, 1, 1000, [0, 0, 0], parents=None, seed=2)
    run(queue, case.issue(queue))
    with queue.capture() as step:
        case.issue(queue)
    for lengths in ([5, 999, 128], [700, 0, 300], [999, 999, 999]):
        case.lengths = lengths
        case.words["lengths"].copy_(device_words(lengths))
        torch.cuda.synchronize()
        queue.wait(step.replay())
        case.check(heads=(0, 9, 31))
    step.close()


def test_two_queues_at_once_and_the_same_bits(gpu):
    device, queue = gpu
    other = device.create_ops()
    try:
        a = Tree(device, DataType.BF16, 8, 2, 128, 8, 9000, [8900, 5000], seed=1)
        b = Tree(device, DataType.F16, 8, 1, 64, 3, 9000, [8000, 100], seed=2)
        run(queue, a.issue(queue))
        run(other, b.issue(other))
        first = [download(x.dev["out"]).copy() for x in (a, b)]
        for _ in range(5):
            tokens = [a.issue(queue), b.issue(other), a.issue(queue), b.issue(other)]
            queue.wait(tokens[2])
            other.wait(tokens[3])
            for x, bits in zip((a, b), first):
                assert np.array_equal(download(x.dev["out"]), bits)
        a.check(nodes=(0, 7), heads=(0, 7))
        b.check(nodes=(0, 2), heads=(0, 7))
    finally:
        other.close()


@pytest.mark.parametrize("width,nodes,hq", [(16, 1, 2), (64, 3, 8), (128, 2, 4), (80, 150, 2)])
def test_every_end_inside_a_tile(gpu, width, nodes, hq):
    """The last tile of every sequence, shared with NaN rows behind it, at every offset."""
    device, queue = gpu
    lengths = [n if n % 2 else 120 + n for n in range(32)] + [600, 1100, 1301]

    def edit(v):
        for b, n in enumerate(lengths):
            v["k"][b, :, n + nodes:] = np.nan
            v["v"][b, :, n + nodes:] = np.nan
    case = Tree(device, DataType.BF16, hq, 1, width, nodes, 1500, lengths, seed=width, edit=edit)
    run(queue, case.issue(queue))
    case.check(nodes=[0, nodes - 1])
