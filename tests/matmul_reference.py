"""The floating point products in numpy: 8-bit floating point numbers, the block quantisation, products in 64 bits and the rows
of each group."""
import numpy as np

LARGEST = {"Fp8E4M3FN": 448.0, "Fp8E5M2": 57344.0}
# Mantissa bits and the exponent of the smallest normal number.
FIELDS = {"Fp8E4M3FN": (3, -6), "Fp8E5M2": (2, -14)}
HALF_STEP = {"Bf16": 2.0 ** -8, "F16": 2.0 ** -11, "F32": 2.0 ** -24}
INDEX = {"I32": np.int32, "I64": np.int64}


def decoded(codes: np.ndarray, kind: str) -> np.ndarray:
    """The numbers that bytes of an 8-bit type are."""
    bits, low = FIELDS[kind]
    c = codes.astype(np.int64)
    e, f = (c >> bits) & ((1 << (7 - bits)) - 1), c & ((1 << bits) - 1)
    v = np.where(e == 0, f * 2.0 ** (low - bits), (f + (1 << bits)) * np.exp2(e + float(low - 1 - bits)))
    if kind == "Fp8E4M3FN":
        v = np.where((c & 127) == 127, np.nan, v)
    else:
        v = np.where((c & 127) == 124, np.inf, np.where((c & 127) > 124, np.nan, v))
    return np.where(c & 128, -v, v)


def encoded(x: np.ndarray, kind: str) -> np.ndarray:
    """The bytes of the nearest numbers of an 8-bit type, ties to the even one; |x| no more than rounds to the largest."""
    bits, low = FIELDS[kind]
    x = np.asarray(x, np.float64)
    _, e = np.frexp(np.abs(x))
    step = np.ldexp(1.0, np.maximum(e - 1, low) - bits)
    n = np.rint(np.abs(x) / step) * step  # the number itself
    assert (n <= LARGEST[kind]).all()
    _, e = np.frexp(n)
    small = n < 2.0 ** low
    exponent = np.where(small, 0, e - 1 - low + 1).astype(np.int64)
    fraction = np.where(small, n / 2.0 ** (low - bits), n / np.ldexp(1.0, np.where(small, 0, e - 1)) * (1 << bits) - (1 << bits))
    return (exponent << bits | fraction.astype(np.int64) | np.signbit(x).astype(np.int64) << 7).astype(np.uint8)


def quantised(x: np.ndarray, kind: str, block_rows: int, transpose: bool):
    """Codes (bytes) and F32 scales of a matrix of numbers (float64 that are exact in 32 bits)."""
    y = (x.T if transpose else x).astype(np.float32)
    r, c = y.shape
    rb, cb = -(-r // block_rows), -(-c // 128)
    codes, scales = np.zeros((r, c), np.uint8), np.zeros((rb, cb), np.float32)
    with np.errstate(all="ignore"):
        for i in range(rb):
            for j in range(cb):
                at = np.s_[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
                most = np.abs(y[at]).max()
                if not np.isfinite(most):
                    scales[i, j] = np.nan
                    continue
                scales[i, j] = most * np.float32(1.0 / LARGEST[kind])
                unit = scales[i, j] if scales[i, j] > 0 else np.float32(1)
                codes[at] = encoded(y[at] / unit, kind)
    return codes, scales


def product8(a, sa, b, sb, b_rows, sizes=True):
    """a [m, k] and b [n, k] as numbers, their scales: the product in 64 bits, the sum of its terms' magnitudes, and that of the
    largest term of each 16 neighbours (both 0 without `sizes`)."""
    k = a.shape[1]
    out, size, tops = (np.zeros((a.shape[0], b.shape[0])) for _ in range(3))
    for c in range(-(-k // 128)):
        at = slice(128 * c, 128 * (c + 1))
        s = sa[:, c, None].astype(np.float64) * np.repeat(sb[:, c].astype(np.float64), b_rows)[None, :b.shape[0]]
        out += s * (a[:, at] @ b[:, at].T)
        if not sizes:
            continue
        size += np.abs(s) * (np.abs(a[:, at]) @ np.abs(b[:, at]).T)
        for i in range(128 * c, min(k, 128 * (c + 1)), 16):
            tops += np.abs(s) * (np.abs(a[:, None, i:i + 16]) * np.abs(b[None, :, i:i + 16])).max(-1)
    return out, size, tops


def bounds(starts, rows):
    """Each group's rows, as the kernels read starts that do not decrease."""
    s = np.clip(np.asarray(starts, np.int64), 0, rows)
    return [(int(s[g]), int(max(s[g], s[g + 1]))) for g in range(len(s) - 1)]


def group_rows(ids, per, groups):
    ids = np.asarray(ids).astype(np.int64)
    inside = (ids >= 0) & (ids < groups)
    order = np.argsort(np.where(inside, ids, groups), kind="stable")[:inside.sum()]
    starts = np.concatenate([[0], np.cumsum(np.bincount(ids[inside], minlength=groups))])
    rows, place = np.full(len(ids), -1), np.full(len(ids), -1)
    rows[:len(order)] = order // per
    place[order] = np.arange(len(order))
    return starts.astype(np.int32), rows.astype(np.int32), place.astype(np.int32)
