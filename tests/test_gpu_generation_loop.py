"""The generation operators together, as a serving loop uses them: prompts answered in one packed
call and appended to their caches, drafted trees appended, attended, scored and compacted, step
after step, eagerly and from captured sequences; and random shapes of each operator."""
import ctypes

import numpy as np
import pytest
import torch

from iom_b200.tensor import DataType, TensorSpec
from generation_support import UNIT, attend, check_rows, decode, device_words, encode, host_tensor
from gpu_support import download, gpu, run, upload  # noqa: F401
from support import HostTensor, logical
from test_gpu_sdpa_packed import Packed
from test_gpu_sdpa_tree import Tree, random_parents
from test_gpu_token_logprobs import Scores

pytestmark = pytest.mark.gpu

B, HQ, HKV, D, CAP, NODES, VOCAB = 3, 8, 2, 64, 320, 12, 700


class Loop:
    """Device state of three sequences and the host's own account of their caches."""

    def __init__(self, device, queue):
        self.device, self.queue = device, queue
        self.dev = {n: device.create_tensor(HostTensor(s, DataType.BF16).spec) for n, s in {
            "k": (B, HKV, CAP, D), "v": (B, HKV, CAP, D), "q": (B, HQ, NODES, D), "kn": (B, HKV, NODES, D),
            "vn": (B, HKV, NODES, D), "out": (B, NODES, HQ * D), "logits": (B, NODES, VOCAB)}.items()}
        self.dev["tokens"] = device.create_tensor(HostTensor((B, 1, NODES), DataType.U32).spec)
        self.dev["logprob"] = device.create_tensor(HostTensor((B, 1, NODES), DataType.F32).spec)
        self.dev["best"] = device.create_tensor(HostTensor((B, NODES, 4), DataType.F32).spec)
        self.dev["best_tokens"] = device.create_tensor(HostTensor((B, NODES, 4), DataType.U32).spec)
        self.words = {"lengths": device_words([0] * B), "parents": device_words(np.zeros((B, NODES))),
                      "counts": device_words([NODES] * B), "accepted": device_words(np.zeros((B, NODES))),
                      "kept": device_words([0] * B), "status": device_words([0] * 5)}
        need = queue.sdpa_tree_workspace_requirements(self.dev["q"].view(), self.dev["k"].view())
        self.workspace = device.create_workspace(max(32, need.bytes))
        self.host = {n: np.zeros((B, HKV, CAP, D)) for n in ("k", "v")}
        self.lengths = [0] * B

    def put(self, name, values, dtype=DataType.BF16):
        host = host_tensor(values, dtype)
        self.dev[name].storage().copy_(torch.from_numpy(host.storage.copy()))

    def get(self, name):
        spec = self.dev[name].spec
        host = HostTensor(spec.shape, spec.data_type)
        host.storage[:] = download(self.dev[name])
        return logical(host.view())

    def step_operations(self):
        d, w, q = self.dev, self.words, self.queue
        status = w["status"].data_ptr()
        return [
            q.cache_append_batched(d["kn"].view(), d["k"].view(), w["lengths"].data_ptr(), status),
            q.cache_append_batched(d["vn"].view(), d["v"].view(), w["lengths"].data_ptr(), status + 4),
            q.sdpa_tree(d["q"].view(), d["k"].view(), d["v"].view(), d["out"].view(), w["lengths"].data_ptr(),
                        w["parents"].data_ptr(), w["counts"].data_ptr(), status + 8, self.workspace.view()),
            q.token_logprobs(d["logits"].view(), d["tokens"].view(), d["logprob"].view(), None, status + 12,
                             d["best"].view(), d["best_tokens"].view()),
            q.cache_compact(d["k"].view(), d["v"].view(), w["lengths"].data_ptr(), w["accepted"].data_ptr(), NODES,
                            w["kept"].data_ptr(), status + 16),
        ]


def draft(loop, rng):
    """A step's inputs: drafted nodes, and the path that will be kept."""
    parents = random_parents(rng, B, NODES)
    paths = []
    for b in range(B):
        path, at = [], int(rng.integers(0, NODES))
        while at >= 0:
            path.append(at)
            at = int(parents[b][at])
        paths.append(path[::-1])
    values = {n: decode(encode(rng.normal(0, 1, s), DataType.BF16), DataType.BF16)
              for n, s in (("q", (B, HQ, NODES, D)), ("kn", (B, HKV, NODES, D)), ("vn", (B, HKV, NODES, D)),
                           ("logits", (B, NODES, VOCAB)))}
    for n, x in values.items():
        loop.put(n, x)
    tokens = rng.integers(0, VOCAB, (B, 1, NODES)).astype(np.uint32)
    loop.put("tokens", tokens, DataType.U32)
    accepted = np.zeros((B, NODES))
    for b, path in enumerate(paths):
        accepted[b, :len(path)] = path
    loop.words["lengths"].copy_(device_words(loop.lengths))
    loop.words["parents"].copy_(device_words(parents))
    loop.words["accepted"].copy_(device_words(accepted))
    loop.words["kept"].copy_(device_words([len(p) for p in paths]))
    torch.cuda.synchronize()
    return parents, paths, values, tokens


def check_step(loop, parents, paths, values, tokens):
    assert loop.words["status"].tolist() == [0] * 5
    out = loop.get("out").reshape(B, NODES, HQ, D)
    logprob, best = loop.get("logprob"), loop.get("best_tokens")
    for b in range(B):
        at = loop.lengths[b]
        for n, new in (("k", "kn"), ("v", "vn")):
            loop.host[n][b][:, at:at + NODES] = values[new][b]
        for i in range(0, NODES, 3):
            seen, j = list(range(at)), i
            path = []
            while j >= 0:
                path.append(at + j)
                j = int(parents[b][j])
            seen += sorted(path)
            for h in (0, 5, 7):
                g = h // (HQ // HKV)
                want, tol = attend(values["q"][b, h, i], loop.host["k"][b, g][seen], loop.host["v"][b, g][seen], D ** -0.5,
                                   UNIT[DataType.BF16], False)
                check_rows(out[b, i, h], want, tol, DataType.BF16)
            x = values["logits"][b, i]
            lse = np.log(np.exp(x - x.max()).sum()) + x.max()
            assert abs(logprob[b, 0, i] - (x[tokens[b, 0, i]] - lse)) < 1e-5
            assert best[b, i].tolist() == np.argsort(-x, kind="stable")[:4].tolist()
        for n in ("k", "v"):        # the accepted path moves to the front of the tree
            loop.host[n][b][:, at:at + len(paths[b])] = loop.host[n][b][:, [at + a for a in paths[b]]]
        loop.lengths[b] += len(paths[b])
    for n in ("k", "v"):
        got = decode(loop.get(n), DataType.BF16)
        for b in range(B):
            assert np.array_equal(got[b, :, :loop.lengths[b]], loop.host[n][b][:, :loop.lengths[b]])


def prefill(loop, rng):
    """Three prompts in one packed call; their keys and values go to the caches."""
    borders = [0, 70, 71, 200]
    case = Packed(loop.device, DataType.BF16, HQ, HKV, D, borders, rows=210, seed=int(rng.integers(1 << 30)))
    run(loop.queue, case.issue(loop.queue))
    case.check(rows=(0, 69, 70, 71, 150, 199), heads=(0, 7))
    for n in ("k", "v"):
        values = decode(case.codes[n], DataType.BF16)
        for b in range(B):
            loop.host[n][b][:, :borders[b + 1] - borders[b]] = values[:, borders[b]:borders[b + 1]]
        loop.put(n, loop.host[n])
    loop.lengths = [borders[b + 1] - borders[b] for b in range(B)]


def test_serving_loop(gpu):
    device, queue = gpu
    rng = np.random.default_rng(11)
    loop = Loop(device, queue)
    prefill(loop, rng)
    for _ in range(4):
        step = draft(loop, rng)
        tokens = loop.step_operations()
        assert all(t > 0 for t in tokens)
        queue.wait(tokens[-1])
        check_step(loop, *step)
    with queue.capture() as sequence:
        loop.step_operations()
    for _ in range(5):
        step = draft(loop, rng)
        queue.wait(sequence.replay())
        check_step(loop, *step)
    sequence.close()
    count = ctypes.c_uint(99)
    assert device._lib.iomb_sdpa_wait_timeouts(ctypes.byref(count)) == 0 and count.value == 0


@pytest.mark.parametrize("seed", range(12))
def test_random_packed_shapes(gpu, seed):
    device, queue = gpu
    rng = np.random.default_rng(seed)
    hkv = int(rng.integers(1, 6))
    hq = hkv * int(rng.integers(1, 10))
    rows = int(rng.integers(1, 900))
    cuts = sorted(int(x) for x in rng.integers(0, rows + 1, int(rng.integers(2, 12))))
    dtype = (DataType.BF16, DataType.F16)[seed % 2]
    case = Packed(device, dtype, hq, hkv, 16 * int(rng.integers(1, 9)), cuts, rows=rows, seed=seed)
    run(queue, case.issue(queue))
    inside = list(range(cuts[0], cuts[-1]))
    picked = set(rng.choice(inside, min(25, len(inside)), replace=False).tolist()) if inside else set()
    picked |= {r for c in cuts for r in (c - 1, c, c + 1)}
    case.check(rows=sorted(picked), heads=sorted({0, hq // 2, hq - 1}))


@pytest.mark.parametrize("seed", range(16))
def test_random_tree_shapes(gpu, seed):
    device, queue = gpu
    rng = np.random.default_rng(100 + seed)
    hkv = int(rng.integers(1, 5))
    hq = hkv * int(rng.integers(1, 9))
    nodes = int(rng.choice([1, 1, 2, 5, 16, 33, 64]))
    cap = nodes + int(rng.integers(1, 1500))
    batch = int(rng.integers(1, 9))
    lengths = [int(x) for x in rng.integers(0, cap - nodes + 1, batch)]
    counts = [int(x) for x in rng.integers(0, nodes + 1, batch)] if seed % 3 == 0 else None
    dtype = (DataType.BF16, DataType.F16)[seed % 2]
    case = Tree(device, dtype, hq, hkv, 16 * int(rng.integers(1, 9)), nodes, cap, lengths, counts=counts,
                parents=None if seed % 4 == 1 else "random", seed=seed)
    run(queue, case.issue(queue))
    case.check(nodes=sorted({0, nodes // 3, nodes - 1}), heads=sorted({0, hq // 2, hq - 1}))


def test_many_sequences(gpu):
    """More sequences than one pass of the planning warp takes."""
    device, queue = gpu
    rng = np.random.default_rng(5)
    lengths = [int(x) for x in rng.integers(0, 290, 300)]
    case = Tree(device, DataType.BF16, 4, 2, 32, 2, 292, lengths, seed=1)
    run(queue, case.issue(queue))
    case.check(heads=(0, 3))
    cuts = sorted(int(x) for x in rng.integers(0, 1500, 301))
    packed = Packed(device, DataType.BF16, 4, 2, 32, cuts, rows=1500, seed=2)
    run(queue, packed.issue(queue))
    packed.check(rows=range(cuts[0], cuts[-1], 7), heads=(0, 3))


def test_caches_beyond_32_bits(gpu):
    """The last plane of a five-gigabyte owner, rows near the end of a plane of two million: the rows
    before them are zero, so each has score zero and adds nothing but its weight."""
    from iom_b200.device import DeviceMemoryConfig, make_b200_device
    device = make_b200_device(0, DeviceMemoryConfig(12 << 30))
    queue = device.create_ops()
    try:
        rows, planes, width = 1 << 21, 9, 128
        rng = np.random.default_rng(9)
        owners = [device.create_tensor(TensorSpec((planes, 1, rows, width), DataType.BF16))
                  for _ in range(2)]
        live = {n: decode(encode(rng.normal(0, 1, (16, width)), DataType.BF16), DataType.BF16) for n in ("k", "v")}
        for owner, n in zip(owners, ("k", "v")):
            tile = HostTensor((16, width), DataType.BF16)
            tile.view().copy_from_host(encode(live[n], DataType.BF16))
            owner.storage()[-tile.storage_nbytes:].copy_(torch.from_numpy(tile.storage.copy()))
        q = host_tensor(rng.normal(0, 2, (1, 4, 1, width)), DataType.BF16)
        out = upload(device, HostTensor((1, 1, 4 * width), DataType.BF16))
        dq = upload(device, q)
        views = [o.view().slice(0, planes - 1, 1) for o in owners]
        words = [device_words([rows - 1]), device_words([7])]
        need = queue.sdpa_tree_workspace_requirements(dq.view(), views[0])
        ws = device.create_workspace(need.bytes)
        run(queue, queue.sdpa_tree(dq.view(), *views, out.view(), words[0].data_ptr(), 0, 0, words[1].data_ptr(), ws.view(), 1.0))
        assert int(words[1].item()) == 0
        host = HostTensor((1, 1, 4 * width), DataType.BF16)
        host.storage[:] = download(out)
        got = decode(logical(host.view()), DataType.BF16).reshape(4, width)
        qv = decode(logical(q.view()), DataType.BF16)[0, :, 0]
        for h in range(4):
            s = live["k"] @ qv[h]
            top = max(s.max(), 0.0)
            z = np.exp(s - top).sum() + (rows - 16) * np.exp(-top)
            want = np.exp(s - top) @ live["v"] / z
            # weights rounded to BF16 and the result again; two million terms of the sum
            assert np.all(np.abs(got[h] - want) <= (2.0 ** -7 + rows * 2.0 ** -24) * (np.exp(s - top) @ np.abs(live["v"]) / z) + 1e-30)
        # and compaction there: the tree's second row becomes its first
        words = [device_words([rows - 2]), device_words([[1, 0]]), device_words([1]), device_words([7])]
        run(queue, queue.cache_compact(*views, words[0].data_ptr(), words[1].data_ptr(), 2, words[2].data_ptr(), words[3].data_ptr()))
        assert int(words[3].item()) == 0
        for owner, n in zip(owners, ("k", "v")):
            tile = HostTensor((16, width), DataType.BF16)
            tile.storage[:] = owner.storage()[-tile.storage_nbytes:].cpu().numpy()
            rows_now = decode(logical(tile.view()), DataType.BF16)
            assert np.array_equal(rows_now[14], live[n][15]) and np.array_equal(rows_now[13], live[n][13])
    finally:
        queue.close()


@pytest.mark.parametrize("seed", range(20))
def test_random_score_shapes(gpu, seed):
    """Few distinct values make ties at the border of the K best likely."""
    device, queue = gpu
    rng = np.random.default_rng(200 + seed)
    rows = int(rng.integers(1, 70))
    vocab = int(np.exp(rng.uniform(np.log(33), np.log(20000))))
    dtype = (DataType.BF16, DataType.F16, DataType.F32)[seed % 3]
    values = rng.normal(0, 3, (rows, vocab))
    if seed % 2:
        values = np.round(values * 2) / 2
    if seed % 5 == 0:
        values[rng.random(values.shape) < 0.7] = -np.inf
    case = Scores(device, values, dtype, rng.integers(0, vocab, rows), int(rng.integers(1, 33)))
    run(queue, case.issue(queue))
    case.check()
