"""Measured cases of the generation operators: attention over packed prompts, attention of drafted
token trees over a KV cache, compaction of the accepted rows, and scoring of tokens.

Every tensor is held as the library holds it: the last two axes cut into 16x16 tiles (tile rows,
tile columns, row in tile, column in tile), both padded to multiples of 16. `run` either computes
the operators in plain 32-bit torch operations on these bytes, or calls the library on them.
"""
import math
import random

import torch

own = False

BF16, F16, F32 = "bf16", "f16", "f32"
TYPES = {BF16: torch.bfloat16, F16: torch.float16, F32: torch.float32}


def listed():
    return [
        # A few short chat turns answered together: a launch-bound call.
        dict(name="packed_short_f16", op="packed", dtype=F16, rows=333, seqs=9, hq=32, hkv=4, d=64, mix=1),
        # One prompt of the full context of the benchmark's decoder geometry.
        dict(name="packed_context", op="packed", dtype=BF16, rows=2048, seqs=1, hq=32, hkv=4, d=64, mix=2),
        # Prompts of very different lengths in one batch, wide heads.
        dict(name="packed_ragged", op="packed", dtype=BF16, rows=6007, seqs=17, hq=32, hkv=8, d=128, mix=3),
        # One long document.
        dict(name="packed_long", op="packed", dtype=BF16, rows=8192, seqs=1, hq=32, hkv=8, d=128, mix=4),
        # One sequence decoding one token: latency.
        dict(name="tree_one_token", op="tree", dtype=BF16, batch=1, nodes=1, hq=32, hkv=4, d=64, cap=2048, chain=True, mix=5),
        # The benchmark's decode step: 64 sequences, one token each, anywhere in their context.
        dict(name="tree_decode_batch", op="tree", dtype=BF16, batch=64, nodes=1, hq=32, hkv=4, d=64, cap=2048, chain=True, mix=6),
        # Trees of 64 drafted tokens for eight sequences over longer caches.
        dict(name="tree_drafts", op="tree", dtype=BF16, batch=8, nodes=64, hq=32, hkv=8, d=128, cap=8192, chain=False, mix=7),
        # Few sequences with very long caches, an odd number of nodes, head groups of three.
        dict(name="tree_long_cache_f16", op="tree", dtype=F16, batch=2, nodes=5, hq=24, hkv=8, d=80, cap=100001, chain=False, mix=8),
        # Accepted rows of the decode batch move to the front of the drafted rows: one layer.
        dict(name="compact_layer", op="compact", dtype=BF16, batch=64, layers=1, heads=4, cap=2048, d=64, nodes=16, mix=9),
        # The same for eight layers held together and larger trees.
        dict(name="compact_layers", op="compact", dtype=BF16, batch=32, layers=8, heads=8, cap=1024, d=128, nodes=64, mix=10),
        # Scores of the decode batch over the benchmark's vocabulary.
        dict(name="logprobs_decode", op="logprobs", dtype=BF16, rows=64, vocab=32000, top=20, masked=False, mix=11),
        # Scores of every token of a prompt, 32-bit logits of an odd vocabulary, some tokens ruled out.
        dict(name="logprobs_prompt_f32", op="logprobs", dtype=F32, rows=2045, vocab=50021, top=8, masked=True, mix=12),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "tree", "tree", "compact", "logprobs"])
    mix = rng.randrange(1 << 20)
    hkv = rng.choice([1, 2, 4, 5, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 8] if hkv <= 4 else [1, 2, 3, 4])
    d = rng.choice([16, 32, 64, 64, 80, 96, 112, 128, 128])
    if op == "packed":
        rows = _spread(rng, 1, 8000)
        return dict(op=op, dtype=rng.choice([BF16, F16]), rows=rows, seqs=_spread(rng, 1, min(96, rows)),
                    hq=hq, hkv=hkv, d=d, mix=mix)
    if op == "tree":
        nodes = rng.choice([1, 1, _spread(rng, 2, 64)])
        cap = _spread(rng, nodes + 1, 60000)
        batch = _spread(rng, 1, max(1, min(96, 2000000 // (cap * hkv))))
        return dict(op=op, dtype=rng.choice([BF16, F16]), batch=batch, nodes=nodes, hq=hq, hkv=hkv, d=d,
                    cap=cap, chain=nodes == 1 or rng.random() < 0.3, mix=mix)
    if op == "compact":
        nodes = _spread(rng, 2, 64)
        return dict(op=op, dtype=rng.choice([BF16, F16, F32]), batch=_spread(rng, 1, 64), layers=rng.randint(1, 4),
                    heads=hkv, cap=_spread(rng, nodes + 1, 1500), d=rng.choice([d, d + 5]), nodes=nodes, mix=mix)
    vocab = _spread(rng, 40, 120000)
    return dict(op=op, dtype=rng.choice([BF16, F16, F32]), rows=_spread(rng, 1, max(1, min(4000, 80000000 // vocab))),
                vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]), masked=rng.random() < 0.3, mix=mix)


# ---- the geometry a case fixes -------------------------------------------------------------------

def _offsets(case):
    """Borders of the packed sequences: uneven, some of one row, the last rows sometimes unused."""
    rng = random.Random(case["mix"])
    rows, seqs = case["rows"], case["seqs"]
    last = rows - (rng.randrange(16) if seqs > 1 and rows > 64 else 0)
    if seqs == 1:
        return [0, last]
    weights = [math.exp(rng.uniform(0, 4)) for _ in range(seqs)]
    cuts, at = [0], 0.0
    for w in weights[:-1]:
        at += w / sum(weights)
        cuts.append(min(last, int(at * last)))
    return cuts + [last]


def _lengths(case):
    """Live rows before the tree, and nodes in use, for every sequence."""
    rng = random.Random(case["mix"])
    cap, nodes, batch = case["cap"], case["nodes"], case["batch"]
    room = cap - nodes
    if batch == 1:
        return [room], [nodes]
    if case["op"] == "tree" and batch == 2:
        return [room, max(0, room * 2 // 3)], [nodes, max(1, nodes - 1)]
    lengths = [rng.randint(0, room) for _ in range(batch)]
    counts = [nodes if nodes <= 2 or rng.random() < 0.7 else rng.randint(1, nodes) for _ in range(batch)]
    return lengths, counts


def _accepted(case):
    """Accepted nodes of every tree, ascending: the path one verification keeps."""
    rng = random.Random(case["mix"] + 1)
    _, counts = _lengths(case)
    paths = []
    for count in counts:
        keep = rng.randint(1, max(1, min(8, count)))
        paths.append(sorted(rng.sample(range(count), keep)))
    return paths


def work(case):
    size = {BF16: 2, F16: 2, F32: 4}[case["dtype"]]
    if case["op"] == "packed":
        cuts = _offsets(case)
        pairs = sum((b - a) * (b - a + 1) // 2 for a, b in zip(cuts, cuts[1:]))
        rows = cuts[-1] - cuts[0]
        return {"bytes": rows * case["d"] * size * 2 * (case["hq"] + case["hkv"]),
                "flops": 4 * case["d"] * case["hq"] * pairs}
    if case["op"] == "tree":
        lengths, counts = _lengths(case)
        live = sum(a + n for a, n in zip(lengths, counts))
        nodes = sum(counts)
        seen = sum(n * (a + (n + 1) / 2) for a, n in zip(lengths, counts))
        return {"bytes": case["d"] * size * 2 * (live * case["hkv"] + nodes * case["hq"]),
                "flops": 4 * case["d"] * case["hq"] * seen}
    if case["op"] == "compact":
        moved = sum(len(p) for p in _accepted(case))
        return {"bytes": 2 * 2 * moved * case["layers"] * case["heads"] * case["d"] * size, "flops": 0}
    cells = case["rows"] * case["vocab"]
    return {"bytes": cells * size + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * cells}


# ---- tiled storage --------------------------------------------------------------------------------

def _up(n):
    return (n + 15) // 16 * 16


def _tile(x):
    """Logical [..., R, C] -> its tiled storage, flat, padding zero."""
    r, c = x.shape[-2:]
    if (r, c) != (_up(r), _up(c)):
        x = torch.nn.functional.pad(x, (0, _up(c) - c, 0, _up(r) - r))
    return x.reshape(*x.shape[:-2], _up(r) // 16, 16, _up(c) // 16, 16).transpose(-3, -2).reshape(-1)


def _untile(flat, shape):
    r, c = shape[-2:]
    x = flat.view(*shape[:-2], _up(r) // 16, _up(c) // 16, 16, 16).transpose(-3, -2)
    return x.reshape(*shape[:-2], _up(r), _up(c))[..., :r, :c]


# ---- inputs ---------------------------------------------------------------------------------------

def _logical_inputs(case, seed):
    """Logical inputs by name, on the GPU; the integer arrays beside the tensors."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + case["mix"])
    t = TYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * by).to(t)

    def whole(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["op"] == "packed":
        # Queries a little larger than the keys: some heads look at few tokens.
        return ({"q": normal(case["hq"], case["rows"], case["d"], by=1.5),
                 "k": normal(case["hkv"], case["rows"], case["d"]), "v": normal(case["hkv"], case["rows"], case["d"])},
                {"offsets": whole(_offsets(case))})
    if case["op"] == "tree":
        b, n = case["batch"], case["nodes"]
        lengths, counts = _lengths(case)
        # Parents lie before their children; -1 hangs a node on the last token of the prefix.
        draws = torch.rand(b, n, generator=gen, device="cuda")
        at = torch.arange(n, device="cuda")
        parents = (draws.sqrt() * (at + 1)).floor().clamp(max=at).to(torch.int32) - 1
        if case["chain"]:
            parents = (at - 1).to(torch.int32).expand(b, n).contiguous()
        caches = {"k": normal(b, case["hkv"], case["cap"], case["d"]), "v": normal(b, case["hkv"], case["cap"], case["d"])}
        return ({"q": normal(b, case["hq"], n, case["d"], by=1.5), **caches},
                {"lengths": whole(lengths), "counts": whole(counts), "parents": parents.contiguous()})
    if case["op"] == "compact":
        lengths, _ = _lengths(case)
        paths = _accepted(case)
        n = case["nodes"]
        shape = (case["batch"], case["layers"], case["heads"], case["cap"], case["d"])
        return ({"k": normal(*shape), "v": normal(*shape)},
                {"lengths": whole(lengths), "counts": whole([len(p) for p in paths]),
                 "accepted": whole([p + [0] * (n - len(p)) for p in paths])})
    r, v = case["rows"], case["vocab"]
    logits = normal(r, v, by=2.5)
    if case["masked"]:  # tokens that a grammar rules out, other ones in every row
        logits.masked_fill_(torch.rand(r, v, generator=gen, device="cuda") < 0.4, float("-inf"))
    # Mostly likely tokens, as a model's own text has them.
    tokens = torch.rand(r, 64, generator=gen, device="cuda").mul(v).long().clamp(max=v - 1)
    tokens = tokens.gather(1, logits.float().gather(1, tokens).argmax(1, keepdim=True)).view(1, r)
    return {"logits": logits, "tokens": tokens.to(torch.int32)}, {}


def _result_shapes(case):
    """Name -> (shape, type) of the tensors that the operator writes."""
    if case["op"] == "packed":
        return {"out": ((case["rows"], case["hq"] * case["d"]), TYPES[case["dtype"]])}
    if case["op"] == "tree":
        return {"out": ((case["batch"], case["nodes"], case["hq"] * case["d"]), TYPES[case["dtype"]])}
    if case["op"] == "compact":
        return {}
    r, k = case["rows"], case["top"]
    shapes = {"logprob": ((1, r), torch.float32), "entropy": ((1, r), torch.float32)}
    if k:
        shapes["top_logprobs"] = ((r, k), torch.float32)
        shapes["top_tokens"] = ((r, k), torch.int32)
    return shapes


def prepare(case, seed):
    tensors, arrays = _logical_inputs(case, seed)
    state = {"case": case, "arrays": arrays, "shapes": {n: tuple(x.shape) for n, x in tensors.items()}}
    state["data"] = {n: _tile(x) for n, x in tensors.items()}
    results = _result_shapes(case)
    if own:
        # The same bytes in tensors of the library, with the queue and the small arrays that a
        # generation loop keeps from call to call.
        from iom_b200.device import DeviceMemoryConfig, make_b200_device
        from iom_b200.tensor import DataType, TensorSpec
        leaf = {torch.bfloat16: DataType.BF16, torch.float16: DataType.F16, torch.float32: DataType.F32,
                torch.int32: DataType.U32}
        specs = {n: TensorSpec(x.shape, leaf[x.dtype]) for n, x in tensors.items()}
        specs |= {n: TensorSpec(shape, leaf[t]) for n, (shape, t) in results.items()}
        need = sum(s.tiled_storage_nbytes() + 256 for s in specs.values())
        scratch = 96 << 20 if case["op"] == "tree" else 0
        device = make_b200_device(0, DeviceMemoryConfig((need + scratch + (1 << 20)) // 32 * 32))
        queue = device.create_ops()
        held = {n: device.create_tensor(s) for n, s in specs.items()}
        for n, flat in state["data"].items():
            held[n].storage().copy_(flat.view(torch.uint8))
        state["data"] = {n: t.storage().view(tensors[n].dtype if n in tensors else results[n][1]) for n, t in held.items()}
        views = {n: t.view() for n, t in held.items()}
        state |= {"device": device, "queue": queue, "held": held, "views": views,
                  "status": torch.zeros(1, dtype=torch.int32, device="cuda")}
        if case["op"] == "tree":
            need = queue.sdpa_tree_workspace_requirements(views["q"], views["k"])
            state["workspace"] = device.create_workspace(need.bytes) if need.bytes else None
        torch.cuda.synchronize()
    return state


# ---- the operators ----------------------------------------------------------------------------------

def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the seen cells; rows that see nothing are not defined."""
    s = torch.matmul(q * scale, k.transpose(-1, -2)).masked_fill_(~seen, float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    return torch.matmul(s, v) / s.sum(-1, keepdim=True)


def _plain_packed(case, data, shapes, arrays):
    hq, hkv, t, d = case["hq"], case["hkv"], case["rows"], case["d"]
    q = _untile(data["q"], shapes["q"]).float().view(hkv, hq // hkv, t, d)
    k, v = (_untile(data[n], shapes[n]).float().view(hkv, 1, t, d) for n in ("k", "v"))
    at = torch.arange(t, device=q.device)
    owner = (arrays["offsets"][None, :] <= at[:, None]).sum(1)
    live = (owner >= 1) & (owner <= case["seqs"])
    seen = (owner[:, None] == owner[None, :]) & (at[None, :] <= at[:, None])
    out = _attend(q, k, v, seen, 1.0 / math.sqrt(d)).view(hq, t, d).permute(1, 0, 2).reshape(t, hq * d)
    return {"out": _tile(torch.where(live[:, None], out, 0.0).to(TYPES[case["dtype"]]))}


def _plain_tree(case, data, shapes, arrays):
    b, n, hq, hkv, c, d = (case[x] for x in ("batch", "nodes", "hq", "hkv", "cap", "d"))
    q = _untile(data["q"], shapes["q"]).float().view(b, hkv, hq // hkv, n, d)
    k, v = (_untile(data[x], shapes[x]).float().view(b, hkv, 1, c, d) for x in ("k", "v"))
    node = torch.arange(n, device=q.device)
    up = (arrays["parents"][:, :, None] == node[None, None, :]).float() + torch.eye(n, device=q.device)
    for _ in range(max(1, (n - 1).bit_length())):  # 2^k steps up the tree
        up = (torch.matmul(up, up) > 0).float()
    at = torch.arange(c, device=q.device)
    rel = at[None, :] - arrays["lengths"][:, None]
    kin = up.gather(2, rel.clamp(0, n - 1)[:, None, :].expand(b, n, c)) > 0
    seen = (rel < 0)[:, None, :] | (kin & ((rel >= 0) & (rel < n))[:, None, :])
    live = node[None, :] < arrays["counts"][:, None]
    out = _attend(q, k, v, seen[:, None, None], 1.0 / math.sqrt(d))
    out = out.view(b, hq, n, d).permute(0, 2, 1, 3).reshape(b, n, hq * d)
    return {"out": _tile(torch.where(live[:, :, None], out, 0.0).to(TYPES[case["dtype"]]))}


def _plain_compact(case, data, shapes, arrays):
    n = case["nodes"]
    node = torch.arange(n, device="cuda")
    moved = node[None, :] < arrays["counts"][:, None]
    who, j = moved.nonzero(as_tuple=True)
    to = arrays["lengths"][who].long() + j
    start = arrays["lengths"][who].long() + arrays["accepted"][who, j].long()
    for name in ("k", "v"):
        flat, shape = data[name], shapes[name]
        rows, cols = shape[-2:]
        # [batch, layers, heads, tile row, tile column, row in tile, column in tile]
        x = flat.view(*shape[:-2], _up(rows) // 16, _up(cols) // 16, 16, 16)
        x[who, :, :, to // 16, :, to % 16] = x[who, :, :, start // 16, :, start % 16]
    return {"k": data["k"], "v": data["v"]}


def _plain_logprobs(case, data, shapes, arrays):
    x = _untile(data["logits"], shapes["logits"]).float()
    token = _untile(data["tokens"], shapes["tokens"]).view(-1, 1).long()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    p = e / z
    entropy = -torch.where(p > 0, p * (x - lse), 0.0).sum(-1)
    out = {"logprob": _tile((x.gather(1, token) - lse).view(1, -1)), "entropy": _tile(entropy.view(1, -1))}
    if case["top"]:
        best, token = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_logprobs"] = _tile(best[:, :case["top"]] - lse)
        out["top_tokens"] = _tile(token[:, :case["top"]].to(torch.int32))
    return out


def run(state):
    case, data = state["case"], state["data"]
    if own:
        queue, v, a = state["queue"], state["views"], state["arrays"]
        status = state["status"].data_ptr()
        if case["op"] == "packed":
            token = queue.sdpa_packed(v["q"], v["k"], v["v"], v["out"], a["offsets"].data_ptr(), case["seqs"], status)
        elif case["op"] == "tree":
            space = state["workspace"].view() if state["workspace"] is not None else None
            token = queue.sdpa_tree(v["q"], v["k"], v["v"], v["out"], a["lengths"].data_ptr(),
                                    0 if case["chain"] else a["parents"].data_ptr(), a["counts"].data_ptr(), status, space)
        elif case["op"] == "compact":
            token = queue.cache_compact(v["k"], v["v"], a["lengths"].data_ptr(), a["accepted"].data_ptr(), case["nodes"],
                                        a["counts"].data_ptr(), status)
        else:
            token = queue.token_logprobs(v["logits"], v["tokens"], v["logprob"], v["entropy"], status,
                                         v.get("top_logprobs"), v.get("top_tokens"))
        if token <= 0:
            raise RuntimeError("the call was refused: oid %d" % token)
        names = _result_shapes(case) or {"k": 0, "v": 0}
        return {n: data[n] for n in names}
    plain = {"packed": _plain_packed, "tree": _plain_tree, "compact": _plain_compact, "logprobs": _plain_logprobs}
    return plain[case["op"]](case, data, state["shapes"], state["arrays"])


# ---- the definitions in 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "compact":
        return None  # moved bits, nothing is computed
    tensors, arrays = _logical_inputs(case, seed)
    if case["op"] == "packed":
        q, k, v = (tensors[n].double() for n in ("q", "k", "v"))
        group = case["hq"] // case["hkv"]
        out = torch.zeros(case["rows"], case["hq"], case["d"], dtype=torch.float64, device="cuda")
        cuts = _offsets(case)
        for a, b in zip(cuts, cuts[1:]):
            if a == b:
                continue
            past = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
            for h in range(case["hq"]):
                score = q[h, a:b] @ k[h // group, a:b].T / math.sqrt(case["d"])
                weight = torch.softmax(score.masked_fill(~past, float("-inf")), -1)
                out[a:b, h] = weight @ v[h // group, a:b]
        return {"out": _tile(out.view(case["rows"], -1))}
    if case["op"] == "tree":
        lengths, counts = _lengths(case)
        parents = arrays["parents"].tolist()
        group = case["hq"] // case["hkv"]
        out = torch.zeros(case["batch"], case["nodes"], case["hq"], case["d"], dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            base, n = lengths[b], counts[b]
            seen = torch.zeros(n, base + n, dtype=torch.bool)
            seen[:, :base] = True
            for i in range(n):
                j = i
                while j >= 0:
                    seen[i, base + j] = True
                    j = parents[b][j]
            seen = seen.to("cuda")
            q = tensors["q"][b, :, :n].double().view(case["hkv"], group, n, case["d"])
            k = tensors["k"][b, :, None, :base + n].double()
            v = tensors["v"][b, :, None, :base + n].double()
            score = q @ k.transpose(-1, -2) / math.sqrt(case["d"])
            weight = torch.softmax(score.masked_fill(~seen, float("-inf")), -1)
            out[b, :n] = (weight @ v).view(case["hq"], n, case["d"]).transpose(0, 1)
        return {"out": _tile(out.view(case["batch"], case["nodes"], -1))}
    x = tensors["logits"].double()
    pick = tensors["tokens"].view(-1).long()
    lse = torch.logsumexp(x, -1)
    p = torch.softmax(x, -1)
    entropy = torch.special.entr(p).sum(-1)
    result = {"logprob": _tile((x[torch.arange(case["rows"], device="cuda"), pick] - lse).view(1, -1)),
              "entropy": _tile(entropy.view(1, -1))}
    if case["top"]:
        result["top_logprobs"] = _tile(torch.topk(x, case["top"]).values - lse[:, None])
        result["top_tokens"] = None
    return result
