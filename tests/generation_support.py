"""Plain 64-bit forms of the generation operators, and their device fixtures.

Tolerances are derived from the kernels' rounding, with u = eps / 2 of the leaf:
* a weight is rounded to the leaf once (relative u, or for F16 at most 2^-25 absolute below its
  normal range; the largest weight of a row is at least one before the division by the sum);
* a score is a binary32 dot product of D terms, each addition off by at most 2^-23 relative to
  the sum of magnitudes (an accumulator that truncates), so a weight is off by the factor
  exp(2 ds) with ds = (D + 4) 2^-23 scale sum|q k| and the exponential's own 2^-21;
* the sums over n tokens add n 2^-23;
* the result is rounded to the leaf once (relative u; F16 below its normal range 2^-25 absolute).
"""
from __future__ import annotations

import numpy as np
import torch

from iom_b200.tensor import DataType
from support import HostTensor, bf16_bits_to_f32, f32_to_bf16_bits, logical

UNIT = {DataType.BF16: 2.0 ** -8, DataType.F16: 2.0 ** -11}
NAN_CODE = {DataType.BF16: 0x7FC0, DataType.F16: 0x7E00}


def encode(values, data_type):
    values = np.asarray(values, dtype=np.float32)
    if data_type == DataType.BF16:
        return f32_to_bf16_bits(values).reshape(values.shape)
    if data_type == DataType.F16:
        with np.errstate(over="ignore"):
            return values.astype(np.float16).view(np.uint16)
    return values


def decode(codes, data_type):
    if data_type == DataType.BF16:
        return bf16_bits_to_f32(codes).reshape(codes.shape).astype(np.float64)
    if data_type == DataType.F16:
        return codes.view(np.float16).astype(np.float64)
    return codes.astype(np.float64)


def host_tensor(values, data_type, poison=0xA5):
    """A host owner of these logical values (any float array, or codes of the leaf), every
    padding byte poisoned."""
    values = np.asarray(values)
    host = HostTensor(values.shape, data_type).poison(poison)
    codes = values if values.dtype in (np.uint16, np.uint32, np.int32, np.int64, np.uint64) else \
        encode(values, data_type)
    host.view().copy_from_host(np.ascontiguousarray(codes))
    return host


def device_words(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values).astype(np.int64), dtype=dtype, device="cuda").contiguous()


def attend(q, k, v, scale, unit, half):
    """(out, tolerance) of one row: q [D], the visible k and v [n, D], in 64 bits. Special rows as
    the operators define them."""
    width = q.shape[0]
    if k.shape[0] == 0:
        return np.zeros(v.shape[1]), np.zeros(v.shape[1])
    with np.errstate(all="ignore"):
        s = (k @ q) * scale
        magnitude = (np.abs(k) @ np.abs(q)) * scale
    if np.isnan(s).any() or np.all(s == -np.inf):
        return np.full(v.shape[1], np.nan), np.zeros(v.shape[1])
    infinite = s == np.inf
    if infinite.any():
        w = infinite / infinite.sum()
        magnitude = np.zeros_like(s)
    else:
        w = np.exp(s - s.max())
        w /= w.sum()
    with np.errstate(all="ignore"):
        out = w @ v
        spread = w @ np.abs(v)
        finite = magnitude[np.isfinite(magnitude)]
        ds = (width + 4) * 2.0 ** -23 * (finite.max() if finite.size else 0.0)
        relative = unit + np.expm1(2 * ds) + 2.0 ** -20 + k.shape[0] * 2.0 ** -23
        tolerance = relative * spread + unit * np.abs(out) + 1e-37
        if half:
            tolerance = tolerance + 2.0 ** -25 * np.abs(v).sum(0) + 2.0 ** -25
    return out, tolerance


def check_rows(got_codes, want, tolerance, data_type):
    """Codes of the leaf against 64-bit rows: classes equal, finite values within tolerance,
    stored zeros and NaN canonical."""
    got = decode(got_codes, data_type)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    assert np.all(got_codes[nan] == NAN_CODE[data_type])
    assert not np.any(got_codes == 0x8000), "-0 was stored"
    infinite = np.isinf(want)
    assert np.array_equal(got[infinite], want[infinite])
    fine = ~nan & ~infinite
    limit = 3.3895313892515355e38 if data_type == DataType.BF16 else 65504.0
    inside = fine & (np.abs(want) < limit * 0.99)
    off = np.abs(got[inside] - want[inside])
    bad = off > tolerance[inside]
    assert not bad.any(), (off[bad].max(), tolerance[inside][bad].max(), int(bad.sum()), int(inside.sum()))


def live(view):
    return logical(view)
