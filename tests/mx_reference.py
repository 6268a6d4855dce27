"""Plain 64-bit implementations of the block-scaled ("microscaled") operations, for the tests: the element types
as tables of their values, nearest by search, everything else in float64."""
import math

import numpy as np

import helpers  # noqa: F401
from synaptik_b200 import program
from synaptik_b200.program import BF16, F16, F32

helpers.NP_DTYPES.setdefault(program.U8, np.uint8)
STORAGE = {"f32": F32, "bf16": BF16, "f16": F16}
EPS = {"f32": 2.0 ** -23, "bf16": 2.0 ** -7, "f16": 2.0 ** -10}


def levels(fmt):
    """The non-negative values of E2M1 / E4M3 by code."""
    mantissa, bias, count = (1, 1, 8) if fmt == "mx4" else (3, 7, 127)
    out = []
    for code in range(count):
        e, m = code >> mantissa, code & ((1 << mantissa) - 1)
        out.append(math.ldexp(m, 1 - bias - mantissa) if e == 0 else math.ldexp(1 + m / (1 << mantissa), e - bias))
    return np.array(out)


def blocked(x):
    x = np.asarray(x, dtype=np.float64)
    pad = -x.shape[-1] % 32
    return np.pad(x, [(0, 0)] * (x.ndim - 1) + [(0, pad)]).reshape(x.shape[:-1] + (-(-x.shape[-1] // 32), 32))


def quantize(x, fmt):
    """(codes, scales) bytes of float values x [.., K]."""
    table = levels(fmt)
    b = blocked(x)
    finite = np.isfinite(b).all(-1)
    largest = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0)).max(-1), 0)
    exponent = np.full(largest.shape, -127)
    for e in range(-127, 128):                  # the least scale that holds the block
        exponent = np.where(largest > table[-1] * math.ldexp(1.0, e), e + 1, exponent)
    under = np.where(finite[..., None], np.abs(np.where(np.isfinite(b), b, 0)), 0) / np.exp2(exponent.astype(np.float64))[..., None]
    above = np.minimum(np.searchsorted(table, under), len(table) - 1)
    below = np.maximum(above - 1, 0)
    up, down = table[above] - under, under - table[below]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    sign = np.signbit(b) & finite[..., None]
    lead = b.shape[:-2]
    scales = np.where(finite, exponent + 127, 255).astype(np.uint8)
    scales = np.pad(scales, [(0, 0)] * len(lead) + [(0, -scales.shape[-1] % 4)])
    if fmt == "mx8":
        return (code + 128 * sign).astype(np.uint8).reshape(lead + (32 * b.shape[-2],)), scales
    nibbles = (code + 8 * sign).astype(np.uint8).reshape(lead + (32 * b.shape[-2],))
    return nibbles[..., 0::2] | (nibbles[..., 1::2] << 4), scales


def values(codes, scales, fmt, features):
    """float64 values of a block-scaled tensor [.., features]."""
    table = np.append(levels(fmt), np.nan) if fmt == "mx8" else levels(fmt)
    codes = np.asarray(codes)
    if fmt == "mx4":
        codes = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (2 * codes.shape[-1],))
        value = table[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    else:
        value = table[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    blocks = value.shape[-1] // 32
    scale = np.exp2(scales[..., :blocks].astype(np.float64) - 127)
    scale = np.where(scales[..., :blocks] == 255, np.nan, scale)
    return (value.reshape(value.shape[:-1] + (blocks, 32)) * scale[..., None]).reshape(value.shape)[..., :features]


def sigmoid(x):
    return 1 / (1 + np.exp(-np.clip(x, -700, 700)))


_erf = np.vectorize(math.erf, otypes=[np.float64])
_erfc = np.vectorize(math.erfc, otypes=[np.float64])
C = math.sqrt(2 / math.pi)


def activate(act, z):
    if act is None:
        return z
    with np.errstate(over="ignore", invalid="ignore"):
        return {"relu": lambda: np.maximum(z, 0), "tanh": lambda: np.tanh(z), "sigmoid": lambda: sigmoid(z), "silu": lambda: z * sigmoid(z),
                "gelu_tanh": lambda: z * sigmoid(2 * C * (z + 0.044715 * z ** 3)), "gelu": lambda: 0.5 * z * _erfc(-z / math.sqrt(2))}[act]()


def slope(act, z):
    if act == "relu":
        return np.where(np.isnan(z), z, (z > 0) * 1.0)
    z = np.clip(z, -1e4, 1e4)
    if act == "tanh":
        return 1 / np.cosh(np.clip(z, -300, 300)) ** 2
    if act == "sigmoid":
        return sigmoid(z) * sigmoid(-z)
    if act == "silu":
        return sigmoid(z) * (1 + z * sigmoid(-z))
    if act == "gelu_tanh":
        u = 2 * C * (z + 0.044715 * z ** 3)
        return sigmoid(u) + z * sigmoid(u) * sigmoid(-u) * 2 * C * (1 + 3 * 0.044715 * z * z)
    return 0.5 * _erfc(-z / math.sqrt(2)) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def stored(kind, x):
    """x as the storage type holds it: (what is fed, its exact float64 values)."""
    with np.errstate(over="ignore"):
        bits = program.to_storage(kind, np.asarray(x, dtype=np.float32))
    return bits, program.from_storage(kind, bits).astype(np.float64)


def read(kind, bits):
    return program.from_storage(kind, bits).astype(np.float64)
