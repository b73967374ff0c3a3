"""The floating point products on the GPU at the ends of their numbers' ranges, and where elements are missing or named twice."""
import numpy as np
import pytest

import unpopped_amd as u
from tests import matmul_reference as ref
from tests.test_gpu_matmul import dev, executor, held, run

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -149  # the smallest step of f32


# ---------------------------------------------------------------------------------------
# Quantisation
# ---------------------------------------------------------------------------------------
def quantised(y, kind, block_rows):
    """Codes and F32 scales of y [rows, cols] in whole blocks: no quotient is past the largest code."""
    top = ref.LARGEST[kind]
    z = y.astype(np.float32).reshape(y.shape[0] // block_rows, block_rows, y.shape[1] // 128, 128)
    scales = np.abs(z).max((1, 3)) * np.float32(1.0 / top)
    unit = np.where(scales > 0, scales, np.float32(1))
    return ref.encoded(np.clip(z / unit[:, None, :, None], -top, top), kind).reshape(y.shape), scales


def quantise_blocks(dtype, kind, block_rows, transpose, y):
    """Compares every code and scale of y, whole blocks of 128 columns."""
    codes, scales = quantised(y, kind, block_rows)
    x = y.T if transpose else y
    xb, cb, sb = dev(held(x, dtype)), u.DeviceBuffer(y.size), u.DeviceBuffer(4 * scales.size)
    run(executor("lower_quant8", dtype=dtype, kind=kind, block_rows=block_rows, transpose=transpose), xb, cb, sb, *x.shape, x.shape[1],
        y.shape[1], scales.shape[1])
    assert np.array_equal(sb.download(np.float32, scales.size).reshape(scales.shape), scales)
    got = cb.download(np.uint8, y.size).reshape(y.shape)
    assert np.isfinite(ref.decoded(got, kind)).all()
    assert np.array_equal(got, codes), (np.argwhere(got != codes)[:5], got[got != codes][:5], codes[got != codes][:5])


# Block maxima, in steps of 2^-149, about the places where the scale rounds to another number of steps, and between them.
SMALL = {
    ("Bf16", "Fp8E5M2"): [k << 16 for k in range(1, 40)],
    ("Bf16", "Fp8E4M3FN"): [k << 16 for k in range(1, 40)],
    ("F32", "Fp8E4M3FN"): sorted({1, 600} | {max(1, j * 224 + d) for j in range(40) for d in (-1, 0, 1, 16, 17, 100)}),
    ("F32", "Fp8E5M2"): sorted({1, 600} | {max(1, j * 28672 + d) for j in range(20) for d in (-1, 0, 1, 4095, 4097, 20000)}),
}


@pytest.mark.parametrize("block_rows, transpose", [(1, False), (128, False), (1, True), (128, True)])
@pytest.mark.parametrize("dtype, kind", list(SMALL))
def test_blocks_whose_scale_is_subnormal(hip_device, dtype, kind, block_rows, transpose):
    rng = np.random.default_rng(1)
    blocks = []
    for most in SMALL[dtype, kind]:
        step = 1 << 16 if dtype == "Bf16" else 1
        y = rng.integers(-(most // step), most // step + 1, (block_rows, 128)) * step
        y[rng.integers(0, block_rows), rng.permutation(128)[:2]] = most, -most
        y[0, rng.integers(0, 128)] = 0
        y[-1, rng.integers(0, 128)] = -most
        blocks.append(y)
    quantise_blocks(dtype, kind, block_rows, transpose, np.concatenate(blocks) * UNIT)


@pytest.mark.parametrize("block_rows, transpose", [(1, False), (1, True), (128, False)])
@pytest.mark.parametrize("kind", ["Fp8E4M3FN", "Fp8E5M2"])
def test_quotients_beside_the_smallest_ties(hip_device, kind, block_rows, transpose):
    """A quotient next to a tie is on its side of it, for scales about those from which on they are not divided; the rows of one wave have
    scales of both sorts."""
    bits, low = ref.FIELDS[kind]
    top, ties = np.float32(ref.LARGEST[kind]), np.ldexp(np.arange(1, 16, 2), low - bits - 1).astype(np.float32)
    rng, rows = np.random.default_rng(3), []
    for e in range(-96, -76):
        for f in (1.0, 2.0 - 2.0 ** -23, 2.0 - 7 * 2.0 ** -22, *(1.0 + rng.integers(0, 1 << 23, 5) * 2.0 ** -23)):
            most = np.float32(np.ldexp(f, e)) * top
            unit = most * np.float32(1.0 / top)
            y = [ties * unit]
            for _ in range(3):
                y = [np.nextafter(y[0], np.float32(0)), *y, np.nextafter(y[-1], top)]
            y = np.concatenate(y)[:127]
            rows.append(np.concatenate([[most], y, np.zeros(127 - len(y), np.float32)]))
    for most, other in (("0x1.bffff2p-74", "0x1.fffff4p-107"), ("0x1.bffffap-73", "0x1.fffffcp-106")):
        rows.append(np.array([float.fromhex(most), float.fromhex(other)] + [0.0] * 126))
        rows += [np.zeros(128)] * 7  # no scale that divides beside it
    y = np.array(rows)
    y = np.concatenate([y, rng.permutation(y)])
    y = np.concatenate([y, np.zeros((-len(y) % 128, 128))]) if block_rows == 1 else np.repeat(y[-60:], 128, 0) * (rng.random((60 * 128, 1)) < 0.5)
    quantise_blocks("F32", kind, block_rows, transpose, y)
