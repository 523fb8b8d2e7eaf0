"""Refusals of the generation operators at the C ABI, before any device work (no GPU needed)."""
import ctypes

import pytest

from iom_b200 import _abi
from iom_b200.tensor import DataType, TensorView
from support import HostTensor

WORD = 0x10000          # never dereferenced on the host; every call below is refused


def ref(view):
    return None if view is None else ctypes.byref(view.as_abi())


def tensor(shape, dtype=DataType.BF16):
    return HostTensor(shape, dtype).view()


def packed(q=None, k=None, v=None, out=None, offsets=WORD, sequences=2, scale=0.125, status=WORD):
    q = q or tensor((4, 40, 64))
    k, v = k or tensor((2, 40, 64)), v or tensor((2, 40, 64))
    out = out or tensor((40, 256))
    return _abi.load_library().iomb_sdpa_packed(ref(q), ref(k), ref(v), ref(out), offsets, sequences, scale, status, None)


@pytest.mark.parametrize("change,code", [
    (dict(q=tensor((1, 4, 40, 64))), 1), (dict(out=tensor((1, 40, 256))), 1),           # ranks
    (dict(k=tensor((2, 40, 32))), 1), (dict(v=tensor((2, 40, 32))), 1),                 # widths
    (dict(k=tensor((2, 41, 64)), v=tensor((2, 41, 64))), 1),                            # rows
    (dict(k=tensor((3, 40, 64)), v=tensor((3, 40, 64))), 1),                            # heads do not group
    (dict(k=tensor((2, 40, 64), DataType.F16)), 1),                                     # encodings
    (dict(out=tensor((40, 255))), 1), (dict(out=tensor((39, 256))), 1),
    (dict(q=tensor((4, 40, 272)), k=tensor((2, 40, 272)), v=tensor((2, 40, 272)), out=tensor((40, 1088))), 2),
    (dict(q=tensor((4, 40, 64), DataType.F32), k=tensor((2, 40, 64), DataType.F32), v=tensor((2, 40, 64), DataType.F32),
          out=tensor((40, 256), DataType.F32)), 2),
    (dict(offsets=None), 1), (dict(offsets=WORD + 2), 1), (dict(sequences=0), 1), (dict(sequences=1 << 21), 2),
    (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
    (dict(status=None), 1), (dict(status=WORD + 1), 1),
])
def test_packed(change, code):
    assert packed(**change) == code
    assert _abi.last_error()


def test_packed_output_overlaps_an_input():
    owner = HostTensor((4, 40, 64), DataType.BF16)
    out = TensorView(owner, tensor((40, 256)).spec, 0, ())
    assert packed(q=owner.view(), out=out) == 1
    assert "overlaps" in _abi.last_error()


def tree(q=None, k=None, v=None, out=None, lengths=WORD, parents=None, counts=None, scale=0.125, workspace=WORD,
         nbytes=1 << 40, status=WORD):
    q = q or tensor((3, 4, 5, 64))
    k, v = k or tensor((3, 2, 400, 64)), v or tensor((3, 2, 400, 64))
    out = out or tensor((3, 5, 256))
    return _abi.load_library().iomb_sdpa_tree(ref(q), ref(k), ref(v), ref(out), lengths, parents, counts, scale, workspace,
                                              nbytes, status, None)


@pytest.mark.parametrize("change,code", [
    (dict(q=tensor((4, 5, 64))), 1), (dict(q=tensor((2, 4, 5, 64))), 1), (dict(out=tensor((2, 5, 256))), 1),
    (dict(k=tensor((3, 3, 400, 64)), v=tensor((3, 3, 400, 64))), 1), (dict(v=tensor((3, 2, 401, 64))), 1),
    (dict(q=tensor((3, 4, 257, 64)), out=tensor((3, 257, 256))), 2),
    (dict(lengths=None), 1), (dict(lengths=WORD + 1), 1), (dict(parents=WORD + 2), 1), (dict(counts=WORD + 3), 1),
    (dict(scale=0.0), 1), (dict(status=None), 1),
])
def test_tree(change, code):
    assert tree(**change) == code
    assert _abi.last_error()


def test_tree_workspace_is_checked():
    lib = _abi.load_library()
    nbytes = ctypes.c_uint64()
    long = tensor((3, 2, 4000, 64))
    assert lib.iomb_sdpa_tree_workspace_bytes(ref(tensor((3, 4, 5, 64))), ref(long), ctypes.byref(nbytes)) == 0
    assert nbytes.value > 0 and nbytes.value % 32 == 0
    for change in (dict(workspace=None), dict(nbytes=nbytes.value - 1), dict(workspace=WORD + 16, nbytes=nbytes.value)):
        assert tree(k=long, v=tensor((3, 2, 4000, 64)), **change) == 1
        assert "workspace" in _abi.last_error()
    # a short cache is never cut, a width off the tensor cores has no partial sums
    for k, q in ((tensor((3, 2, 128, 64)), tensor((3, 4, 5, 64))), (tensor((3, 2, 4000, 40)), tensor((3, 4, 5, 40)))):
        assert lib.iomb_sdpa_tree_workspace_bytes(ref(q), ref(k), ctypes.byref(nbytes)) == 0 and nbytes.value == 0


def test_tree_workspace_bytes():
    lib = _abi.load_library()
    nbytes = ctypes.c_uint64()
    q, k = tensor((3, 4, 5, 64)), tensor((3, 2, 400, 64))
    assert lib.iomb_sdpa_tree_workspace_bytes(ref(q), ref(k), ctypes.byref(nbytes)) == 0
    assert lib.iomb_sdpa_tree_workspace_bytes(ref(q), ref(k), None) == 1
    assert lib.iomb_sdpa_tree_workspace_bytes(None, ref(k), ctypes.byref(nbytes)) == 1
    assert lib.iomb_sdpa_tree_workspace_bytes(ref(tensor((3, 4, 5, 32))), ref(k), ctypes.byref(nbytes)) == 1
    assert lib.iomb_sdpa_tree_workspace_bytes(ref(tensor((3, 5, 5, 64))), ref(k), ctypes.byref(nbytes)) == 1
    assert lib.iomb_sdpa_tree_workspace_bytes(ref(tensor((3, 4, 257, 64))), ref(k), ctypes.byref(nbytes)) == 2


def compact(k=None, v=None, lengths=WORD, accepted=WORD, width=8, counts=WORD, status=WORD):
    k = k or tensor((3, 2, 40, 64))
    return _abi.load_library().iomb_cache_compact(ref(k), ref(v), lengths, accepted, width, counts, status, None)


@pytest.mark.parametrize("change,code", [
    (dict(k=tensor((40, 64))), 1), (dict(v=tensor((3, 2, 41, 64))), 1), (dict(v=tensor((3, 2, 40, 64), DataType.F16)), 1),
    (dict(lengths=None), 1), (dict(accepted=None), 1), (dict(counts=None), 1), (dict(status=None), 1),
    (dict(accepted=WORD + 1), 1), (dict(width=0), 1), (dict(k=tensor((3, 2, 40, 64), DataType.U4)), 2),
])
def test_compact(change, code):
    assert compact(**change) == code
    assert _abi.last_error()


def test_compact_planes_must_be_distinct():
    owner = HostTensor((6, 40, 64), DataType.BF16)
    twice = TensorView(owner, tensor((3, 2, 40, 64)).spec, 0, (1, 1))     # [3, 2] planes over four
    assert compact(k=twice) == 1
    assert "overlap" in _abi.last_error()
    assert compact(k=owner.view(), v=TensorView(owner, owner.spec, 0, (1,))) == 1


def scores(logits=None, tokens=None, logprob=None, entropy=None, values=None, best=None, status=WORD):
    logits = logits or tensor((2, 5, 50))
    tokens = tokens or tensor((2, 1, 5), DataType.U32)
    logprob = logprob or tensor((2, 1, 5), DataType.F32)
    return _abi.load_library().iomb_token_logprobs(ref(logits), ref(tokens), ref(logprob), ref(entropy), ref(values),
                                                   ref(best), status, None)


@pytest.mark.parametrize("change,code", [
    (dict(logits=tensor((2, 5, 50), DataType.I32)), 2), (dict(tokens=tensor((2, 1, 5), DataType.U8)), 2),
    (dict(tokens=tensor((2, 5, 1), DataType.U32)), 1), (dict(tokens=tensor((1, 1, 5), DataType.U32)), 1),
    (dict(logprob=tensor((2, 1, 5))), 1), (dict(entropy=tensor((2, 1, 6), DataType.F32)), 1),
    (dict(values=tensor((2, 5, 4), DataType.F32)), 1),
    (dict(values=tensor((2, 5, 4), DataType.F32), best=tensor((2, 5, 3), DataType.U32)), 1),
    (dict(values=tensor((2, 5, 33), DataType.F32), best=tensor((2, 5, 33), DataType.U32)), 2),
    (dict(logits=tensor((2, 5, 3)), values=tensor((2, 5, 4), DataType.F32), best=tensor((2, 5, 4), DataType.U32)), 1),
    (dict(values=tensor((2, 5, 4), DataType.F32), best=tensor((2, 5, 4), DataType.U64)), 1),
    (dict(status=None), 1),
])
def test_scores(change, code):
    assert scores(**change) == code
    assert _abi.last_error()


def test_scores_results_do_not_overlap():
    shared = tensor((2, 1, 5), DataType.F32)
    assert scores(logprob=shared, entropy=shared) == 1
