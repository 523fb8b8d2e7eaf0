"""Attention over packed prompts (iomb_sdpa_packed) against the formula in 64 bits, row by row:
head groups, widths on and off the tensor cores, sequences of every length around the tiles
(16), the row blocks and the token blocks (128), rows outside every sequence, special values,
views, other streams and captured sequences."""
import numpy as np
import pytest
import torch

from iom_b200.device import OID_INVALID_ARGUMENT
from iom_b200.tensor import DataType
from generation_support import UNIT, attend, check_rows, decode, device_words, encode, host_tensor
from gpu_support import download, gpu, run, upload  # noqa: F401
from support import HostTensor, logical

pytestmark = pytest.mark.gpu


class Packed:
    """One call's operands on both sides."""

    def __init__(self, device, dtype, hq, hkv, width, borders, rows=None, seed=0, edit=None):
        rng = np.random.default_rng(seed)
        self.dtype, self.hq, self.hkv, self.width, self.borders = dtype, hq, hkv, width, list(borders)
        self.rows = rows if rows is not None else borders[-1]
        self.values = {"q": rng.normal(0, 1.5, (hq, self.rows, width)), "k": rng.normal(0, 1, (hkv, self.rows, width)),
                       "v": rng.normal(0, 1, (hkv, self.rows, width))}
        if edit is not None:
            edit(self.values)
        self.codes = {n: encode(x, dtype) for n, x in self.values.items()}
        self.host = {n: host_tensor(c, dtype) for n, c in self.codes.items()}
        self.host["out"] = HostTensor((self.rows, hq * width), dtype).poison(0x3C)
        self.dev = {n: upload(device, h) for n, h in self.host.items()}
        self.offsets = device_words(self.borders)
        self.status = device_words([77])

    def issue(self, queue, scale=None):
        d = self.dev
        return queue.sdpa_packed(d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view(), self.offsets.data_ptr(),
                                 len(self.borders) - 1, self.status.data_ptr(), scale)

    def check(self, scale=None, rows=None, heads=None):
        """`rows` / `heads`: the ones compared (all by default); bytes outside the sequences always."""
        scale = np.float32(self.width ** -0.5 if scale is None else scale).astype(np.float64)
        assert int(self.status.item()) == 0
        got_host = self.host["out"].clone()
        got_host.storage[:] = download(self.dev["out"])
        got = logical(got_host.view()).reshape(self.rows, self.hq, self.width)
        inside = np.zeros(self.rows, dtype=bool)
        inside[self.borders[0]:self.borders[-1]] = True
        assert np.all(got[~inside] == 0x3C3C), "rows outside every sequence changed"
        # padding of the output keeps its bytes: put the poison back over the logical cells
        got_host.view().copy_from_host(np.full((self.rows, self.hq * self.width), 0x3C3C, dtype=np.uint16))
        assert np.all(got_host.storage == 0x3C), "padding of the output changed"
        value = {n: decode(c, self.dtype) for n, c in self.codes.items()}
        half = self.dtype == DataType.F16
        for a, e in zip(self.borders, self.borders[1:]):
            for r in range(a, e) if rows is None else [r for r in rows if a <= r < e]:
                for h in range(self.hq) if heads is None else heads:
                    g = h // (self.hq // self.hkv)
                    want, tolerance = attend(value["q"][h, r], value["k"][g, a:r + 1], value["v"][g, a:r + 1], scale,
                                             UNIT[self.dtype], half)
                    check_rows(got[r, h], want, tolerance, self.dtype)


HEADS = [(1, 1), (4, 1), (8, 8), (6, 2), (10, 2), (16, 1), (24, 8)]


@pytest.mark.parametrize("dtype", [DataType.BF16, DataType.F16])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_head_groups(gpu, dtype, hq, hkv):
    device, queue = gpu
    case = Packed(device, dtype, hq, hkv, 64, [0, 5, 5, 48, 49, 95], seed=hq)
    run(queue, case.issue(queue))
    case.check()


@pytest.mark.parametrize("width", [1, 5, 16, 17, 32, 48, 64, 80, 96, 112, 128, 129, 144, 200, 256])
def test_head_widths(gpu, width):
    device, queue = gpu
    for dtype in (DataType.BF16, DataType.F16):
        case = Packed(device, dtype, 4, 2, width, [0, 33, 50, 70], seed=width)
        run(queue, case.issue(queue))
        case.check()


@pytest.mark.parametrize("borders,rows", [
    ([0, 1], 1), ([0, 1], 40), ([7, 8], 9), ([0, 15, 31, 48], 48), ([3, 19, 20, 36, 53], 60),
    ([0, 127], 127), ([0, 128], 128), ([0, 129], 129), ([1, 129], 131), ([15, 143, 272], 300),
    ([0, 16, 16, 16, 32], 32), ([31, 31], 64), ([64, 64, 65], 65), ([17, 270], 288),
    ([0] + list(range(1, 41)), 41),
])
def test_borders(gpu, borders, rows):
    device, queue = gpu
    case = Packed(device, DataType.BF16, 4, 2, 64, borders, rows=rows, seed=rows)
    run(queue, case.issue(queue))
    case.check()
    case = Packed(device, DataType.F16, 2, 2, 128, borders, rows=rows, seed=rows)
    run(queue, case.issue(queue))
    case.check()


@pytest.mark.parametrize("dtype,hq,hkv,width,borders", [
    (DataType.BF16, 32, 4, 64, [0, 700, 705, 1333]),
    (DataType.BF16, 8, 2, 128, [5, 1030, 1500]),
    (DataType.F16, 3, 3, 96, [0, 900]),
    (DataType.F16, 12, 4, 80, [0, 17, 1100]),
    (DataType.BF16, 2, 1, 16, [0, 2100]),
])
def test_long_sequences(gpu, dtype, hq, hkv, width, borders):
    device, queue = gpu
    case = Packed(device, dtype, hq, hkv, width, borders, seed=width)
    run(queue, case.issue(queue))
    last = borders[-1]
    rows = sorted({r for r in (0, 1, 15, 16, 127, 128, 129, 255, 256, 257, 511, 640, 699, 700, 704, 705, 833,
                               1023, 1024, 1029, 1030, last - 2, last - 1) if borders[0] <= r < last})
    case.check(rows=rows)


def test_peaked_scores_and_growing_maxima(gpu):
    """Scores that grow along the sequence (every block raises the running maximum) and fall
    (none does), far beyond the exponent range of one block to the next."""
    device, queue = gpu
    for sign in (1.0, -1.0):
        def edit(v):
            n = v["k"].shape[1]
            v["q"][:] = 1.0
            v["k"][:] = (sign * np.arange(n) / 4.0)[None, :, None] / 8.0
        case = Packed(device, DataType.BF16, 2, 1, 64, [0, 600], seed=3, edit=edit)
        run(queue, case.issue(queue))
        case.check()
        case = Packed(device, DataType.F16, 2, 1, 64, [0, 300], seed=3, edit=edit)
        run(queue, case.issue(queue, scale=1.0))
        case.check(scale=1.0)


def test_special_values(gpu):
    """NaN and infinities in q, k and v: visible ones follow the formula, ones under the mask or
    in another sequence have no influence."""
    device, queue = gpu

    def edit(v):
        v["v"][0, 40, 3] = np.nan           # rows >= 40 of the second sequence see it
        v["v"][0, 100, 5] = np.inf
        v["v"][0, 120, 5] = -np.inf         # from 120 on: inf - inf
        v["k"][1, 180, 7] = np.nan
        v["q"][3, 60, 0] = np.nan
        v["k"][1, 70, :] = np.inf           # +inf or -inf scores, NaN where signs mix
        v["q"][2, 75, :] = 1.0              # +inf score at 70
        v["q"][2, 76, :] = -1.0             # -inf score at 70: weight zero
        v["k"][0, 200, :] = np.inf          # the third sequence's first row
        v["q"][0, 200:204, :] = -1.0        # row 200 sees only -inf
        v["v"][1, 20, 0] = 3e38             # large but finite values
        v["v"][1, 21, 0] = 3e38
    for dtype in (DataType.BF16, DataType.F16):
        case = Packed(device, dtype, 4, 2, 64, [0, 30, 200, 330], rows=340, seed=9, edit=edit)
        run(queue, case.issue(queue))
        case.check()


def test_poisoned_rows_outside(gpu):
    """Rows that belong to no sequence hold NaN."""
    device, queue = gpu

    def edit(v):
        for x in v.values():
            x[:, :5] = np.nan
            x[:, 150:] = np.nan
    case = Packed(device, DataType.BF16, 2, 1, 64, [5, 60, 150], rows=200, seed=4, edit=edit)
    run(queue, case.issue(queue))
    case.check()


@pytest.mark.parametrize("borders", [[0, 20, 10, 40], [0, 41], [5, 4], [0, 0xFFFFFFFF], [0, 20, 0xFFFFFFF0, 40]])
@pytest.mark.parametrize("width", [64, 40])
def test_wrong_borders_write_nothing(gpu, borders, width):
    device, queue = gpu
    case = Packed(device, DataType.BF16, 2, 1, width, [0, 40], rows=40)
    case.borders = borders
    case.offsets = torch.tensor(np.array(borders, dtype=np.uint32).view(np.int32), device="cuda")
    run(queue, case.issue(queue))
    assert int(case.status.item()) == 1
    assert np.all(download(case.dev["out"]) == 0x3C)
    case.offsets = device_words([0, 40])
    case.borders = [0, 40]
    run(queue, case.issue(queue))       # and a good call clears the word
    case.check()


def test_views_of_wider_owners(gpu):
    """Heads strided through wider owners: q, k and v as slices of one fused [heads, T, D] owner,
    heads in another order."""
    device, queue = gpu
    rng = np.random.default_rng(12)
    fused = host_tensor(rng.normal(0, 1, (12, 50, 64)), DataType.BF16)
    dev = upload(device, fused)
    out = upload(device, HostTensor((3, 50, 4 * 64), DataType.BF16).poison(0x3C))
    q = dev.view().slice(0, 1, 4, 2)        # planes 1, 3, 5, 7
    k, v = dev.view().slice(0, 8, 2), dev.view().slice(0, 10, 2)
    offsets, status = device_words([0, 20, 50]), device_words([5])
    run(queue, queue.sdpa_packed(q, k, v, out.view().select(0, 1), offsets.data_ptr(), 2, status.data_ptr()))
    values = decode(logical(fused.view()), DataType.BF16)
    host = HostTensor((3, 50, 256), DataType.BF16)
    host.storage[:] = download(out)
    got = logical(host.view())
    assert np.all(got[[0, 2]] == 0x3C3C)
    for a, e in ((0, 20), (20, 50)):
        for r in range(a, e):
            for h in range(4):
                want, tol = attend(values[1 + 2 * h, r], values[8 + h // 2, a:r + 1], values[10 + h // 2, a:r + 1],
                                   0.125, UNIT[DataType.BF16], False)
                check_rows(got[1, r, 64 * h:64 * h + 64], want, tol, DataType.BF16)


def test_refusals_leave_the_output(gpu):
    device, queue = gpu
    case = Packed(device, DataType.BF16, 4, 2, 64, [0, 20])
    d = case.dev
    assert queue.sdpa_packed(d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view(), 0, 1,
                             case.status.data_ptr()) == OID_INVALID_ARGUMENT
    assert queue.sdpa_packed(d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view(),
                             case.offsets.data_ptr(), 0, case.status.data_ptr()) == OID_INVALID_ARGUMENT
    other = device.create_ops()
    try:
        run(other, case.issue(other))       # a second queue of the device
    finally:
        other.close()
    case.check()


def test_captured_and_replayed_with_new_borders(gpu):
    """The borders are read when the operation runs: a replay follows them."""
    device, queue = gpu
    case = Packed(device, DataType.BF16, 8, 2, 64, [0, 100, 160], rows=200, seed=2)
    run(queue, case.issue(queue))
    with queue.capture() as step:
        case.issue(queue)
    for borders in ([0, 40, 160], [10, 10, 200], [0, 199, 200]):
        case.borders = borders
        case.offsets.copy_(device_words(borders))
        case.dev["out"].storage().fill_(0x3C)
        torch.cuda.synchronize()
        queue.wait(step.replay())
        case.check()
    step.close()


def test_same_call_gives_the_same_bits(gpu):
    device, queue = gpu
    case = Packed(device, DataType.BF16, 8, 2, 128, [0, 333, 800], seed=6)
    run(queue, case.issue(queue))
    first = download(case.dev["out"]).copy()
    for _ in range(3):
        run(queue, case.issue(queue))
        assert np.array_equal(first, download(case.dev["out"]))


@pytest.mark.parametrize("width", [16, 64, 80, 128])
@pytest.mark.parametrize("first", range(0, 18, 3))
def test_every_start_and_end_inside_a_tile(gpu, width, first):
    """The tiles that a sequence shares with NaN rows beside it, at every offset."""
    device, queue = gpu
    borders = [first]
    for n in range(1, 18):
        borders.append(borders[-1] + 16 + n)

    def edit(v):
        for x in v.values():
            x[:, :first] = np.nan
            x[:, borders[-1]:] = np.nan
    case = Packed(device, DataType.BF16, 2, 1, width, borders, rows=borders[-1] + 40, seed=first, edit=edit)
    run(queue, case.issue(queue))
    case.check()
