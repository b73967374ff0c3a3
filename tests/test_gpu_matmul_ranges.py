"""The floating point products on the GPU at the ends of their numbers' ranges, and where elements are missing or named twice."""
import numpy as np
import pytest

import unpopped_amd as u
from tests import matmul_reference as ref
from tests.test_gpu_matmul import JUNK, dev, executor, grouped_case, held, laid, matmul8_case, read, run, starts_of

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


# ---------------------------------------------------------------------------------------
# Products of codes whose scales are far from 1
# ---------------------------------------------------------------------------------------
def launch_codes(a, sa, b, sb, a_kind, b_kind, out, b_rows, pad, starts, workspace=None):
    """The product of numbers that are codes: [m][n] in 64 bits, and the launch."""
    (m, k), (g, n, _) = a.shape, b.shape
    aa, a_row, _ = laid(ref.encoded(a, a_kind), pad, 0, JUNK[a_kind])
    ba, b_row, b_group = laid(ref.encoded(b, b_kind), pad, 0, JUNK[b_kind])
    sab, as_row, _ = laid(sa, 0, 0, np.float32(np.nan))
    sbb, bs_row, bs_group = laid(sb, 0, 0, np.float32(np.nan))
    ex = executor("lower_matmul8", a_kind=a_kind, b_kind=b_kind, out=out, b_rows=b_rows, grouped=starts is not None)
    shape = (m, n, k) if starts is None else (m, n, k, g)
    ws = ex.workspace_bytes(*shape) if workspace is None else workspace
    ob = dev(held(np.full((m, n), 9.0), out))
    run(ex, dev(aa), dev(sab), dev(ba), dev(sbb), *([] if starts is None else [dev(starts.astype(np.int32))]), ob,
        dev(np.full(ws + 16, 0xFF, np.uint8)), *shape, a_row, as_row, b_row, bs_row, *([] if starts is None else [b_group, bs_group]), n, ws)
    return read(ob, m * n, out).reshape(m, n), ex.last_launch()


FAR = [
    (16, 33, 1040, dict(), "_one"), (16, 33, 1040, dict(b_rows=1), "_one"), (1, 300, 2048, dict(b_kind="Fp8E5M2"), "_one"),
    (32, 2100, 272, dict(), "_slim"), (65, 4100, 272, dict(b_rows=1), "_few"), (600, 2100, 272, dict(b_rows=1), "_some"),
    (1000, 2100, 16, dict(), "_tile"), (2817, 2561, 143, dict(b_rows=1, pad=1), "_tile"), (130, 300, 200, dict(pad=1), "_any"),
    (70, 300, 200, dict(pad=1, b_rows=1), "_any"), (4000, 2561, 272, dict(), "_wide"), (4000, 2561, 272, dict(a_kind="Fp8E5M2"), "_wide"),
    (4000, 2100, 143, dict(pad=1, b_rows=1), "_wide"), (2817, 4100, 257, dict(pad=15), "_wide"), (2817, 2820, 400, dict(b_rows=1), "_wide"),
    (60, 300, 28000, dict(), "_join"), (3500, 2561, 272, dict(groups=2), "_wide"), (900, 1300, 272, dict(groups=6), "_some"),
]


def far_inputs(m, n, k, a_kind, b_kind, b_rows, groups):
    rng = np.random.default_rng(6)
    nb, nr, g = -(-k // 128), -(-n // b_rows), max(1, groups)
    a, b = (ref.decoded(ref.encoded(32 + 64 * np.minimum(np.abs(rng.normal(size=s)), 4), kind), kind) for s, kind in (((m, k), a_kind), ((g, n, k), b_kind)))
    sa, sb = (np.exp(rng.normal(size=s) / 2) for s in ((m, nb), (g, nr, nb)))
    starts = starts_of(rng, m, groups, "all") if groups else None
    return rng, a, sa, b, sb, starts


@pytest.mark.parametrize("m, n, k, kw, entry", FAR)
def test_scales_whose_product_is_no_number(hip_device, m, n, k, kw, entry):
    """Products of scales far below f32 and past its end, whose products with the sums of codes are ordinary numbers or 0."""
    kinds = [kw.get(s, "Fp8E4M3FN") for s in ("a_kind", "b_kind")]
    b_rows, groups = kw.get("b_rows", 128), kw.get("groups", 0)
    rng, a, sa, b, sb, starts = far_inputs(m, n, k, *kinds, b_rows, groups)
    nb, nr = sa.shape[1], sb.shape[1]
    some = rng.permutation(m)
    # Columns of 2^-60, of 2^-110 and, in one block, of 2^40.
    sb[:, 0] *= 2.0 ** -60
    if nr > 2:
        sb[:, nr // 2] *= 2.0 ** -110
        sb[:, -1, nb - 1] *= 2.0 ** 40
    # Rows of 2^-84, of subnormal scales, of 2^120, and of 2^100 where all codes are 0.
    sa[some[:2]] *= 2.0 ** -84
    if m > 6:
        sa[some[2:3]] *= 2.0 ** -143
        sa[some[3:4]] *= 2.0 ** 120
        sa[some[4:5], nb - 1], a[some[4], 128 * (nb - 1):] = 2.0 ** 100, 0
    sa, sb = sa.astype(np.float32), sb.astype(np.float32)
    got, launch = launch_codes(a, sa, b, sb, *kinds, "Bf16", b_rows, kw.get("pad", 0), starts)
    assert launch["entry"].endswith(entry), launch
    assert not np.isnan(got).any()
    for i in {*some[:5], *some[-20:], 0, m - 1}:
        w = 0 if starts is None else int(np.searchsorted(starts, i, "right")) - 1
        want, size, tops = (v[0] for v in ref.product8(a[i:i + 1], sa[i:i + 1], b[w], sb[w], b_rows))
        # As for scales near 1: the matrix unit's 2^-13 of the largest of 16 products, 2^-23 of the magnitudes for each sum and product.
        # A sum that takes exponents below f32's keeps steps of 2^-149 times 4 of the fractions.  Then the type's rounding.
        tol = tops * 15 * 2.0 ** -13 + size * (8 + 3 * nb) * 2.0 ** -23 + nb * 2.0 ** -147
        tol += (np.abs(want) + tol) * 2.0 ** -8 + 2.0 ** -134
        over = want > 2.0 ** 130
        assert (over | (want < 2.0 ** 127)).all()
        with np.errstate(invalid="ignore"):
            bad = np.where(over, got[i] != np.inf, ~(np.abs(got[i] - want) <= tol))
        assert not bad.any(), (launch, i, np.flatnonzero(bad)[:5], got[i][bad][:5], want[bad][:5])


@pytest.mark.parametrize("m, n, k, kw, entry", [c for c in FAR if c[0] > 6])
def test_far_scales_leave_other_rows_as_they_were(hip_device, m, n, k, kw, entry):
    """Bit for bit: rows beside one of a tiny scale, columns beside some of a large one."""
    kinds = [kw.get(s, "Fp8E4M3FN") for s in ("a_kind", "b_kind")]
    b_rows, groups = kw.get("b_rows", 128), kw.get("groups", 0)
    _, a, sa, b, sb, starts = far_inputs(m, n, k, *kinds, b_rows, groups)
    args = (b, sb.astype(np.float32), *kinds, "F16", b_rows, kw.get("pad", 0), starts)
    sa /= 2.0 ** 20
    plain, _ = launch_codes(a, sa.astype(np.float32), *args)
    sa[m // 2] *= 2.0 ** -90
    got, launch = launch_codes(a, sa.astype(np.float32), *args)
    assert launch["entry"].endswith(entry) and np.isfinite(plain).all()
    keep = np.arange(m) != m // 2
    assert np.array_equal(got[keep], plain[keep]) and (got[m // 2] == 0).all()


# ---------------------------------------------------------------------------------------
# 16-bit products
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("direction, rows, n, k, entry", [
    ("input", 4000, 129, 2304, "_wide"), ("input", 4000, 143, 2304, "_wide"), ("input", 900, 71, 304, "_few"), ("input", 40, 257, 48, "_slim"),
    ("input", 2000, 71, 2104, "_tile"), ("input", 33, 17, 64, "_slim"), ("input", 40, 1041, 48, "_one"), ("forward", 4000, 2304, 129, "_wide"), ("forward", 900, 304, 71, "_few"),
    ("forward", 40, 48, 1041, "_one"),
])
def test_infinities_in_a_depths_last_elements(hip_device, direction, rows, n, k, entry):
    """A weight that is infinite makes infinities of the sums that it is in, also where a depth ends inside 16 bytes, and nothing else."""
    rng = np.random.default_rng(9)
    forward, groups = direction == "forward", 3
    depth, wide = (k, n) if forward else (n, k)
    x = rng.integers(1, 4, (rows, depth)).astype(float)
    w = rng.integers(-3, 4, (groups, wide, depth)).astype(float)  # of each column of out
    w[0, 3, depth - 1], w[1, wide - 1, depth // 8 * 8], w[2, 5, 0], w[2, 8, depth - 1] = np.inf, -np.inf, np.inf, -np.inf
    starts = np.array([0, rows // 3, rows // 2, rows])
    want = np.concatenate([x[r0:r1] @ w[g].T for g, (r0, r1) in enumerate(ref.bounds(starts, rows))])
    xa, x_row, _ = laid(held(x, "Bf16"), -depth % 8, 0, held(np.array([np.nan]), "Bf16")[0])
    wa = held(w if forward else w.transpose(0, 2, 1), "Bf16")
    wa, w_row, w_group = laid(np.ascontiguousarray(wa), -wa.shape[-1] % 8, 0, held(np.array([np.nan]), "Bf16")[0])
    ex, ob = executor("lower_grouped_matmul", dtype="Bf16", out="F32", direction=direction), u.DeviceBuffer(4 * want.size)
    run(ex, dev(xa), dev(wa), dev(starts.astype(np.int32)), ob, u.DeviceBuffer(16), rows, n, k, groups, x_row, w_group, w_row, wide, 0)
    assert ex.last_launch()["entry"].endswith(entry), ex.last_launch()
    got = ob.download(np.float32, want.size).reshape(want.shape)
    assert np.array_equal(got, want), (np.argwhere(got != want)[:5], got[got != want][:5], want[got != want][:5])


@pytest.mark.parametrize("how", ["forward", "input", "codes"])
@pytest.mark.parametrize("rows, groups, depth, lists", [
    (40, 5, 96, [[0, 39, 0, 39, 0, 40], [40, 0, 40, 0, 40, 0], [5, 3, 1, 0, 2, 4], [2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1, 0, -1], [3, -7, 20, 10, 30, 25]]),
    (60, 5, 16384, [[0, 39, 0, 39, 0, 40], [0, 59, 0, 59, 0, 60], [50, 10, 55, 20, 57, 3], [40, 0, 0, 0, 0, 0], [-4, 20, 19, 70, 0, 1]]),
    (500, 200, 128, ["steps", "drop", "any"]),
])
def test_a_start_below_an_earlier_one_counts_as_that_one(hip_device, how, rows, groups, depth, lists):
    """Every row from the first start to the largest is one group's, whatever the workspace held before; the others stay."""
    rng = np.random.default_rng(11)
    wide = 136
    x, w = rng.integers(-1, 2, (rows, depth)).astype(float), rng.integers(-1, 2, (groups, wide, depth)).astype(float)
    blocks = -(-depth // 128)
    if how == "codes":
        ex = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="F16", b_rows=128, grouped=True)
        ones = dev(np.ones(max(rows, groups * 2) * blocks, np.float32))
        ins = [dev(ref.encoded(x, "Fp8E4M3FN")), ones, dev(ref.encoded(w, "Fp8E4M3FN")), ones]
        shape, strides = (rows, wide, depth, groups), (depth, blocks, depth, blocks, wide * depth, 2 * blocks, wide)
    else:
        ex = executor("lower_grouped_matmul", dtype="F16", out="F16", direction=how)
        n, k = (wide, depth) if how == "forward" else (depth, wide)
        ins = [dev(held(x, "F16")), dev(held(w if how == "forward" else np.ascontiguousarray(w.transpose(0, 2, 1)), "F16"))]
        shape, strides = (rows, n, k, groups), (depth, n * k, k, wide)
    need = ex.workspace_bytes(*shape)
    for starts in lists:
        if starts == "steps":
            starts = np.arange(groups + 1) * 2 + rng.integers(-9, 10, groups + 1)
        elif starts == "drop":  # a large start in the first 64 groups, ones below it in the others
            starts = np.sort(rng.integers(0, rows, groups + 1))
            starts[30] = starts[-1] - 20
        elif starts == "any":
            starts = rng.integers(-50, rows + 50, groups + 1)
        want = np.full((rows, wide), 9.0)
        for g, (r0, r1) in enumerate(ref.bounds(np.maximum.accumulate(np.clip(starts, 0, rows)), rows)):
            want[r0:r1] = x[r0:r1] @ w[g].T
        for junk in (0xFF, 0x3F):
            ob = dev(held(np.full((rows, wide), 9.0), "F16"))
            run(ex, *ins, dev(np.array(starts, np.int32)), ob, dev(np.full(need + 16, junk, np.uint8)), *shape, *strides, need)
            got = read(ob, rows * wide, "F16").reshape(rows, wide)
            assert np.array_equal(got, want), (list(starts), junk, np.argwhere(got != want)[:5])
    assert depth < 1000 or ex.last_launch()["chunks"] > 1


# ---------------------------------------------------------------------------------------
# Split depths of every kernel, and long ones of the largest
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind, m, n, k, groups, kw, parts", [
    ("codes", 300, 264, 12297, 0, dict(pad=7), 12),                # 64 x 128
    ("codes", 1030, 2056, 12297, 0, dict(pad=7), 4),               # 256 x 256
    ("codes", 1030, 2056, 12297, 0, dict(pad=7, b_rows=1), 4),     # 256 x 256
    ("codes", 1030, 520, 32777, 2, dict(pad=7, way="gaps"), 16),   # 256 x 256
    ("codes", 1500, 520, 12304, 5, dict(way="gaps"), 3),           # 128 x 128
    ("codes", 260, 264, 12297, 3, dict(pad=7, out_pad=1), 12),     # 64 x 128
    ("codes", 24, 72, 12304, 2, dict(b_rows=1), 12),               # 32 x 64
    ("forward", 1500, 520, 8201, 5, dict(pad=7, way="gaps"), 8),   # 256 x 256
    ("forward", 1500, 520, 8201, 5, dict(pad=7, out="F32"), 8),    # 256 x 256
    ("forward", 520, 1544, 8200, 5, dict(way="gaps"), 3),          # 128 x 128
    ("forward", 260, 264, 8201, 3, dict(pad=7), 12),               # 64 x 128
    ("forward", 24, 136, 12296, 5, dict(way="gaps"), 16),          # 32 x 64
    ("input", 1500, 8201, 520, 5, dict(pad=8, x_pad=7, way="gaps"), 8),
    ("input", 520, 8200, 1544, 5, dict(way="gaps"), 3),
    ("input", 260, 8201, 264, 3, dict(pad=8, x_pad=7, out_pad=1), 12),
    ("input", 24, 12296, 136, 5, dict(way="gaps"), 16),
    ("weight", 24584, 264, 1032, 5, dict(way="gaps"), 4),          # 256 x 256
    ("weight", 24584, 264, 1032, 5, dict(out="F32", out_pad=4), 4),
    ("weight", 2320, 104, 264, 2, dict(way="gaps"), 4),            # 128 x 128
])
def test_a_split_depth_of_each_kernel(hip_device, kind, m, n, k, groups, kw, parts):
    """Whole numbers, exactly, by each shape of tile; lengths that end inside 16 bytes, which the last part alone takes up."""
    if kind == "codes":
        launch = matmul8_case(m, n, k, groups=groups, top=1, **kw)
    else:
        launch = grouped_case(kind, m, n, k, groups, **kw)
    assert launch["chunks"] == parts, launch


@pytest.mark.parametrize("kw", [
    dict(m=4000, n=2561, k=1175, pad=9), dict(m=4000, n=2561, k=1175, pad=9, b_rows=1), dict(m=4000, n=2561, k=2208, b_rows=1, a_kind="Fp8E5M2", top=2),
    dict(m=3500, n=2561, k=1303, pad=9, groups=2, starts=[0, 1100, 3500]), dict(m=3500, n=2561, k=1312, groups=2, starts=[0, 1100, 3500], b_rows=1),
])
def test_codes_of_more_steps_than_their_scales_have_places(hip_device, kw):
    """256 x 256 tiles of whole and half height, from 10 steps on."""
    assert matmul8_case(**kw)["entry"].endswith("_wide")
