"""Scores of given tokens (iomb_token_logprobs) against 64 bits: leaves, vocabularies around the
tiles, rows around the bands, ties, tokens ruled out, special rows, wrong tokens, views.

Tolerance: x - m and the results are binary32 (2^-24 of the value each, a few steps), a term's
exponential is off by 2^-21 and by |x - m| 2^-23 from its rounded argument (|x - m| < 90 where the
term counts), sums over V terms add V 2^-24 at the very most; all enter log z and t / z relative
to a value of the size of the logits' range."""
import numpy as np
import pytest
import torch

from iom_b200.device import OID_INVALID_ARGUMENT, OID_UNSUPPORTED
from iom_b200.tensor import DataType
from generation_support import decode, device_words, encode, host_tensor
from gpu_support import download, gpu, run, upload  # noqa: F401
from support import HostTensor, logical

pytestmark = pytest.mark.gpu


def best(values, k):
    """Indices of the k best of a row: NaN above everything, -0 as +0, ties by the lower index."""
    x = np.where(values == 0, 0.0, values)
    order = sorted(range(len(x)), key=lambda i: (not np.isnan(x[i]), -x[i] if not np.isnan(x[i]) else 0.0, i))
    return order[:k]


def fast_best(values, k):
    if np.isnan(values).any():
        return best(values, k)
    return np.argsort(-np.where(values == 0, 0.0, values), kind="stable")[:k].tolist()


class Scores:
    def __init__(self, device, values, dtype, tokens, top, entropy=True, token_type=DataType.U32):
        self.codes = values if values.dtype == np.uint16 else encode(values, dtype)
        self.value = decode(self.codes, dtype)
        *lead, rows, vocab = self.codes.shape
        self.lead, self.rows, self.vocab, self.top = lead, rows, vocab, top
        self.tokens = np.asarray(tokens).reshape(*lead, 1, rows)
        kind = {DataType.U32: np.uint32, DataType.I32: np.int32, DataType.I64: np.int64, DataType.U64: np.uint64}[token_type]
        self.logits = upload(device, host_tensor(self.codes if dtype != DataType.F32 else self.codes.astype(np.float32), dtype))
        self.dev_tokens = upload(device, host_tensor(self.tokens.astype(np.int64).astype(kind), token_type, poison=0xFF))
        self.host = {"logprob": HostTensor((*lead, 1, rows), DataType.F32).poison(0x3C)}
        if entropy:
            self.host["entropy"] = HostTensor((*lead, 1, rows), DataType.F32).poison(0x3C)
        if top:
            self.host["top_logprobs"] = HostTensor((*lead, rows, top), DataType.F32).poison(0x3C)
            self.host["top_tokens"] = HostTensor((*lead, rows, top), DataType.U32).poison(0x3C)
        self.dev = {n: upload(device, h) for n, h in self.host.items()}
        self.status = device_words([9])

    def issue(self, queue):
        d = {n: t.view() for n, t in self.dev.items()}
        return queue.token_logprobs(self.logits.view(), self.dev_tokens.view(), d["logprob"], d.get("entropy"),
                                    self.status.data_ptr(), d.get("top_logprobs"), d.get("top_tokens"))

    def result(self, name):
        host = self.host[name].clone()
        host.storage[:] = download(self.dev[name])
        got = logical(host.view())
        fill = np.full(got.shape, 0x3C3C3C3C, dtype=np.uint32)
        host.view().copy_from_host(fill.view(got.dtype))
        assert np.all(host.storage == 0x3C), f"padding of {name} changed"
        return got

    def check(self, bad=()):
        assert int(self.status.item()) == (1 if bad else 0)
        got = {n: self.result(n) for n in self.host}
        flat = self.value.reshape(-1, self.rows, self.vocab)
        for p in range(flat.shape[0]):
            where = np.unravel_index(p, self.lead) if self.lead else ()
            for r in range(self.rows):
                x = flat[p, r]
                m = x.max()
                odd = np.isnan(x).any() or np.isinf(m)
                token = int(self.tokens.reshape(-1, self.rows)[p, r])
                logprob = got["logprob"][where + (0, r)]
                order = fast_best(x, self.top)
                if self.top:
                    assert got["top_tokens"][where + (r,)].tolist() == order
                if (p, r) in bad:
                    assert logprob.view(np.uint32) == 0x3C3C3C3C
                if odd:
                    assert (p, r) in bad or np.isnan(logprob)
                    if "entropy" in got:
                        assert np.isnan(got["entropy"][where + (0, r)])
                    if self.top:
                        assert np.isnan(got["top_logprobs"][where + (r,)]).all()
                    continue
                y = x - m
                e = np.exp(y)
                z = e.sum()
                weight = e / z
                entropy = np.log(z) - (weight[e > 0] * y[e > 0]).sum()
                span = 2.0 ** -20 + self.vocab * 2.0 ** -24 + (weight[e > 0] * np.abs(y[e > 0])).sum() * 2.0 ** -22
                if (p, r) not in bad:
                    want = y[token] - np.log(z)
                    if np.isinf(want):
                        assert logprob == want
                    else:
                        assert abs(logprob - want) <= span + (abs(want) + abs(y[token])) * 2.0 ** -23, (logprob, want)
                if "entropy" in got:
                    slack = span * (1 + (weight[e > 0] * np.abs(y[e > 0])).sum()) + np.log(z) * 2.0 ** -22 + 2.0 ** -22
                    assert abs(got["entropy"][where + (0, r)] - entropy) <= 2 * slack
                if self.top:
                    want = y[order] - np.log(z)
                    have = got["top_logprobs"][where + (r,)]
                    assert np.array_equal(np.isinf(want), np.isinf(have))
                    fine = np.isfinite(want)
                    assert np.all(np.abs(have[fine] - want[fine]) <= span + (np.abs(want[fine]) + np.abs(y[order][fine])) * 2.0 ** -23)


DTYPES = [DataType.BF16, DataType.F16, DataType.F32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 0), (3, 15, 15), (16, 16, 5), (17, 17, 17), (1, 40, 32), (33, 100, 32), (2, 4097, 20),
    (15, 1000, 1), (1, 32000, 20), (5, 32000, 32), (18, 5003, 8), (1, 130001, 32),
])
def test_shapes(gpu, dtype, rows, vocab, top):
    device, queue = gpu
    rng = np.random.default_rng(vocab + rows)
    case = Scores(device, rng.normal(0, 2.5, (rows, vocab)), dtype, rng.integers(0, vocab, rows), top)
    run(queue, case.issue(queue))
    case.check()


@pytest.mark.parametrize("token_type", [DataType.U32, DataType.I32, DataType.I64, DataType.U64])
def test_leading_axes_optional_results_and_token_leaves(gpu, token_type):
    device, queue = gpu
    rng = np.random.default_rng(1)
    for entropy, top in ((True, 4), (False, 4), (True, 0), (False, 0)):
        case = Scores(device, rng.normal(0, 3, (2, 3, 21, 333)), DataType.BF16, rng.integers(0, 333, (2, 3, 21)), top,
                      entropy, token_type)
        run(queue, case.issue(queue))
        case.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lower_token(gpu, dtype):
    device, queue = gpu
    rng = np.random.default_rng(2)
    for values in (np.zeros((3, 5000)),                                           # all equal
                   rng.integers(-2, 3, (20, 3000)).astype(np.float64),            # few values
                   np.where(rng.random((18, 2000)) < 0.5, 0.0, -0.0),             # signed zeros are equal
                   np.where(rng.random((4, 9000)) < 0.999, -np.inf, 1.0)):        # nearly all ruled out
        values[:, 7] = 1.0
        tokens = rng.integers(0, values.shape[1], values.shape[0])
        case = Scores(device, values, dtype, tokens, 32)
        run(queue, case.issue(queue))
        case.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_ordered_rows(gpu, dtype):
    """Ascending and descending logits: the worst order for a running list of the best."""
    device, queue = gpu
    ramp = np.linspace(-30, 30, 40000)
    values = np.stack([ramp, ramp[::-1], np.roll(ramp, 20000), np.repeat(ramp[::100], 100)])
    case = Scores(device, values, dtype, [0, 5, 39999, 777], 32)
    run(queue, case.issue(queue))
    case.check()


def test_special_rows(gpu):
    device, queue = gpu
    rng = np.random.default_rng(3)
    for dtype in DTYPES:
        values = rng.normal(0, 2, (20, 3000))
        values[0, 5] = np.nan
        values[1, 2999] = np.inf
        values[2] = -np.inf
        values[3, :2990] = -np.inf
        values[4, [7, 9]] = np.inf
        values[5, [0, 1]] = np.nan, np.inf
        values[6] = -np.inf
        values[6, 1234] = 5.0
        values[7, 10] = 6e4                 # everything else has weight zero
        values[8] = -6e4
        tokens = rng.integers(0, 3000, 20)
        tokens[3] = 0                       # a ruled-out token: -inf
        tokens[6] = 1234
        case = Scores(device, values, dtype, tokens, 12)
        run(queue, case.issue(queue))
        case.check()


def test_wrong_tokens_are_reported(gpu):
    device, queue = gpu
    rng = np.random.default_rng(4)
    tokens = rng.integers(0, 500, (2, 19))
    tokens[0, 3], tokens[1, 18], tokens[1, 0] = -1, 500, 2 ** 31 - 1
    case = Scores(device, rng.normal(0, 2, (2, 19, 500)), DataType.F32, tokens, 3, token_type=DataType.I32)
    run(queue, case.issue(queue))
    case.check(bad={(0, 3), (1, 18), (1, 0)})
    tokens[0, 3], tokens[1, 18], tokens[1, 0] = 2 ** 32, 2 ** 40 + 3, -(2 ** 40)
    case = Scores(device, rng.normal(0, 2, (2, 19, 500)), DataType.F16, tokens, 0, token_type=DataType.I64)
    run(queue, case.issue(queue))
    case.check(bad={(0, 3), (1, 18), (1, 0)})


def test_views_and_captured_sequences(gpu):
    device, queue = gpu
    rng = np.random.default_rng(5)
    case = Scores(device, rng.normal(0, 2, (4, 18, 700)), DataType.BF16, rng.integers(0, 700, (4, 18)), 5)
    run(queue, case.issue(queue))
    case.check()
    d = {n: t.view().permute([0]).slice(0, 1, 2, 2) for n, t in case.dev.items()}      # planes 1 and 3
    for t in case.dev.values():
        t.storage().fill_(0x3C)
    torch.cuda.synchronize()
    with queue.capture() as step:
        queue.token_logprobs(case.logits.view().slice(0, 1, 2, 2), case.dev_tokens.view().slice(0, 1, 2, 2), d["logprob"],
                             d["entropy"], case.status.data_ptr(), d["top_logprobs"], d["top_tokens"])
    queue.wait(step.replay())
    got = case.result("top_tokens")
    assert np.all(got[[0, 2]] == 0x3C3C3C3C)
    for p in (1, 3):
        for r in range(18):
            assert got[p, r].tolist() == fast_best(case.value[p, r], 5)
    step.close()


def test_many_rows_and_the_same_bits(gpu):
    device, queue = gpu
    rng = np.random.default_rng(6)
    case = Scores(device, rng.normal(0, 2.5, (3000, 600)), DataType.BF16, rng.integers(0, 600, 3000), 7)
    run(queue, case.issue(queue))
    case.check()
    first = {n: download(t).copy() for n, t in case.dev.items()}
    for _ in range(3):
        run(queue, case.issue(queue))
        for n, t in case.dev.items():
            assert np.array_equal(first[n], download(t))


def test_refusals(gpu):
    device, queue = gpu
    rng = np.random.default_rng(7)
    case = Scores(device, rng.normal(0, 2, (4, 50)), DataType.F32, [0, 1, 2, 3], 5)
    d = {n: t.view() for n, t in case.dev.items()}
    x, t, s = case.logits.view(), case.dev_tokens.view(), case.status.data_ptr()
    assert queue.token_logprobs(x, t, d["logprob"], d["entropy"], 0) == OID_INVALID_ARGUMENT
    assert queue.token_logprobs(x, t, d["logprob"], d["entropy"], s, d["top_logprobs"]) == OID_INVALID_ARGUMENT
    assert queue.token_logprobs(x, t, d["logprob"], d["logprob"], s) == OID_INVALID_ARGUMENT
    assert queue.token_logprobs(x, d["logprob"], d["logprob"], None, s) == OID_UNSUPPORTED
    wide = [device.create_tensor(HostTensor((4, 33), k).spec) for k in (DataType.F32, DataType.U32)]
    assert queue.token_logprobs(x, t, d["logprob"], None, s, wide[0].view(), wide[1].view()) == OID_UNSUPPORTED
