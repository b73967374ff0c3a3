"""The floating point products on the GPU against their numpy reference: values, odd and empty sizes, strides, groups, refusals."""
import ctypes as C

import numpy as np
import pytest

import unpopped_amd as u
from unpopped_amd import _lib
from tests import matmul_reference as ref
from tests.cache4_reference import loaded, rounded, stored

pytestmark = pytest.mark.gpu
B = u.HipBackend()
_execs: dict = {}
DIRECTIONS = ["forward", "input", "weight"]
# A NaN of each type: what lies where nothing may be read, or may not count.
JUNK = {"Fp8E4M3FN": 0x7F, "Fp8E5M2": 0x7E}


def executor(how, **form):
    key = (how, *sorted(form.items()))
    if key not in _execs:
        _execs[key] = u.Executor(getattr(B, how)(**form))
    return _execs[key]


def dev(a):
    return u.DeviceBuffer.from_array(np.ascontiguousarray(a))


def run(ex, *args):
    print(ex.kernel.name, [a for a in args if not isinstance(a, u.DeviceBuffer)], flush=True)
    ex.launch(*args)
    u.synchronize()


def invalid(ex, *args):
    with pytest.raises(u.UnpError) as e:
        ex.launch(*args)
    assert e.value.kind == "InvalidArgument" and e.value.detail


def held(a, dtype):
    """Numbers as their type holds them: the array to upload."""
    return a.astype(np.float32) if dtype == "F32" else stored(a, dtype)


def read(buf, n, dtype):
    return buf.download(np.float32, n).astype(np.float64) if dtype == "F32" else loaded(buf.download(held(np.zeros(1), dtype).dtype, n), dtype)


def once(a, dtype):
    """64-bit numbers rounded once to a type."""
    return a.astype(np.float32).astype(np.float64) if dtype == "F32" else rounded(a, dtype)


def laid(a, pad, first, junk):
    """[..., rows, cols] with rows of cols + pad elements after `first` of them, junk between and around: a flat array and the
    row's and matrix's strides."""
    r, c = a.shape[-2:]
    wide = np.full((*a.shape[:-1], c + pad), junk, a.dtype)
    wide[..., :c] = a
    return np.concatenate([np.full(first, junk, a.dtype), wide.ravel(), np.full(32, junk, a.dtype)]), c + pad, r * (c + pad)


# ---------------------------------------------------------------------------------------
# Quantisation
# ---------------------------------------------------------------------------------------
def quantise_case(dtype, kind, block_rows, transpose, rows, cols, pad, first=0, seed=0, special=True):
    rng = np.random.default_rng(seed)
    x = once(rng.normal(size=(rows, cols)) * np.exp2(rng.integers(-12, 8, (rows, 1))), dtype)
    if special and rows > 2 and cols > 3:
        x[rows // 2, : min(cols, 128)] = 0.0
        x[0, cols - 1] = np.inf
        x[rows - 1, 0] = np.nan
        x[1, 2] = -0.0
    want, scales = ref.quantised(x, kind, block_rows, transpose)
    xa, x_row, _ = laid(held(x, dtype), pad, first, held(np.array([np.nan]), dtype)[0])
    r, c = want.shape
    ca, code_row, _ = laid(np.full((r, c), 0xAA, np.uint8), pad, first, 0xAA)
    sa, scale_row, _ = laid(np.full(scales.shape, 7, np.float32), pad, 0, np.float32(7))
    xb, cb, sb = dev(xa), dev(ca), dev(sa)
    size = held(np.zeros(1), dtype).itemsize
    run(executor("lower_quant8", dtype=dtype, kind=kind, block_rows=block_rows, transpose=transpose), xb.at(first * size), cb.at(first), sb,
        rows, cols, x_row, code_row, scale_row)
    gs, gc = sb.download(np.float32, len(sa)), cb.download(np.uint8, len(ca))
    at = np.arange(scales.shape[0])[:, None] * scale_row + np.arange(scales.shape[1])
    assert np.array_equal(gs[at], scales, equal_nan=True)
    gs[at] = 7
    assert (gs == 7).all()
    at = first + np.arange(r)[:, None] * code_row + np.arange(c)
    assert np.array_equal(gc[at], want)
    gc[at] = 0xAA
    assert (gc == 0xAA).all()


@pytest.mark.parametrize("block_rows, transpose", [(1, False), (128, False), (1, True), (128, True)])
@pytest.mark.parametrize("dtype, kind, rows, cols, pad, first", [
    ("Bf16", "Fp8E4M3FN", 1, 1, 0, 0), ("Bf16", "Fp8E4M3FN", 130, 256, 0, 0), ("F32", "Fp8E4M3FN", 128, 128, 16, 16),
    ("F16", "Fp8E5M2", 5, 400, 0, 0), ("Bf16", "Fp8E5M2", 257, 129, 3, 1), ("F32", "Fp8E4M3FN", 300, 17, 0, 3),
    ("F16", "Fp8E4M3FN", 64, 136, 8, 0),
])
def test_quantisation_is_bit_exact(hip_device, dtype, kind, rows, cols, pad, first, block_rows, transpose):
    quantise_case(dtype, kind, block_rows, transpose, rows, cols, pad, first)


@pytest.mark.parametrize("kind", ["Fp8E4M3FN", "Fp8E5M2"])
def test_quantisation_near_its_borders(hip_device, kind):
    """Quotients on and beside the ties of the codes; scales from the smallest to the largest of 32 bits."""
    grid = ref.decoded(np.arange(0x7C if kind == "Fp8E5M2" else 0x7F, dtype=np.uint8), kind)
    ties = ((grid[1:] + grid[:-1]) / 2).astype(np.float32)
    rows = []
    for e in (-149, -140, -126, -100, -90, -89, -60, 0, 31, 100, 110):
        unit = np.float32(np.ldexp(1.0 + 0.37 * (e > -126), e))
        with np.errstate(all="ignore"):
            y = np.concatenate([ties * unit, np.nextafter(ties * unit, np.float32(0)), np.nextafter(ties * unit, np.float32(np.inf))])
        y = y[np.isfinite(y)]
        for i in range(0, len(y), 127):
            rows.append(np.concatenate([[np.float32(ref.LARGEST[kind]) * unit], y[i:i + 127], np.zeros(max(0, 127 - len(y[i:i + 127])))]))
    x = np.array(rows, np.float32).astype(np.float64)
    want, scales = ref.quantised(x, kind, 1, False)
    xb, cb, sb = dev(x.astype(np.float32)), u.DeviceBuffer(x.size), u.DeviceBuffer(4 * len(x))
    run(executor("lower_quant8", dtype="F32", kind=kind, block_rows=1, transpose=False), xb, cb, sb, len(x), 128, 128, 128, 1)
    assert np.array_equal(sb.download(np.float32, len(x)), scales[:, 0], equal_nan=True)
    assert np.array_equal(cb.download(np.uint8, x.size).reshape(x.shape), want)


def test_quantisation_refuses(hip_device):
    ex = executor("lower_quant8", dtype="F32", kind="Fp8E4M3FN", block_rows=1, transpose=False)
    x, c, s = dev(np.zeros(256, np.float32)), u.DeviceBuffer(256), u.DeviceBuffer(64)
    invalid(ex, x, c, s, 2, 128, 128, 128)
    invalid(ex, x, c, 0, 2, 128, 128, 128, 1)
    invalid(ex, x, c, s, -1, 128, 128, 128, 1)
    invalid(ex, x, c, s, 2, 128, -128, 128, 1)
    invalid(ex, x, c, s, 2, 128, 128, 127, 1)   # codes named twice
    invalid(ex, x, c, s, 2, 128, 128, 128, 0)   # scales too
    invalid(ex, x, c, s, 2, (1 << 28) + 1, 1 << 29, 1 << 29, 1 << 22)
    invalid(ex, x.at(2), c, s, 2, 64, 64, 64, 1)
    invalid(ex, u.DeviceBuffer.held(0, 0, None), c, s, 2, 128, 128, 128, 1)
    with pytest.raises(u.UnpError):
        ex.launch_views([(x, (2, 128), None, 0), (c, (2, 128), None, 0), (s, (2, 1), None, 0)], [2, 128, 128, 128, 1])
    ex.launch(x, c, s, 0, 128, 128, 128, 1)  # nothing to do
    ex.launch(x, c, s, 2, 0, 128, 128, 1)


# ---------------------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------------------
def starts_of(rng, rows, groups, way):
    """Where the groups of `rows` rows begin."""
    if way == "gaps":  # rows that no group names ahead of the first and behind the last, groups without rows
        cut = np.sort(rng.integers(rows // 8, rows - rows // 8 + 1, groups + 1))
        return cut
    if way == "one":   # one group has them all
        at = groups // 2
        return np.array([0] * (at + 1) + [rows] * (groups - at))
    return np.concatenate([[0], np.sort(rng.integers(0, rows + 1, groups - 1)), [rows]])


def matmul8_case(m, n, k, a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="Bf16", b_rows=128, groups=0, way="all", pad=0, first=0, seed=0,
                 whole=True, workspace=None, nan_scale=False, starts=None, out_pad=0, top=4):
    """whole: numbers and scales whose products and sums are exact in 32 bits, so that the result has to be."""
    rng = np.random.default_rng(seed)
    nb, nr = -(-k // 128), -(-n // b_rows)
    g = max(1, groups)
    if whole:
        a, b = (rng.integers(-top, top + 1, s).astype(float) for s in ((m, k), (g, n, k)))
        sa, sb = (np.exp2(rng.integers(-2, 3, s)).astype(np.float32) for s in ((m, nb), (g, nr, nb)))
        assert top * top * k * 16 * 16 <= 1 << 24  # in units of 2^-4
    else:
        a, b = (ref.decoded(ref.encoded(rng.normal(size=s), kind), kind) for s, kind in (((m, k), a_kind), ((g, n, k), b_kind)))
        sa, sb = (np.exp(rng.normal(size=s)).astype(np.float32) for s in ((m, nb), (g, nr, nb)))
    if nan_scale and nb:
        sa[m // 2, 0] = np.nan
    aa, a_row, _ = laid(ref.encoded(a, a_kind), pad, first, JUNK[a_kind])
    ba, b_row, b_group = laid(ref.encoded(b, b_kind), pad, first, JUNK[b_kind])
    spad = pad // 4
    sab, as_row, _ = laid(sa, spad, 0, np.float32(np.nan))
    sbb, bs_row, bs_group = laid(sb, spad, 0, np.float32(np.nan))
    fill = 9.0
    oa, out_row, _ = laid(held(np.full((m, n), fill), out), out_pad, 4 * (out_pad > 0), held(np.array([fill]), out)[0])
    size = held(np.zeros(1), out).itemsize
    ob = dev(oa)
    if groups:
        starts = starts_of(rng, m, groups, way) if starts is None else np.asarray(starts)
    ex = executor("lower_matmul8", a_kind=a_kind, b_kind=b_kind, out=out, b_rows=b_rows, grouped=groups > 0)
    shape = (m, n, k) + ((groups,) if groups else ())
    need = ex.workspace_bytes(*shape)
    ws = need if workspace is None else workspace
    args = [dev(aa).at(first), dev(sab), dev(ba).at(first), dev(sbb)] + ([dev(starts.astype(np.int32))] if groups else [])
    args += [ob.at(4 * (out_pad > 0) * size), dev(np.full(ws + 16, 0xFF, np.uint8)), *shape, a_row, as_row, b_row, bs_row]
    args += ([b_group, bs_group] if groups else []) + [out_row, ws]
    run(ex, *args)
    got = read(ob, len(oa), out)
    at = 4 * (out_pad > 0) + np.arange(m)[:, None] * out_row + np.arange(n)
    want = np.full((m, n), fill)
    tol = np.zeros((m, n))
    for i, (r0, r1) in enumerate(ref.bounds(starts, m) if groups else [(0, m)]):
        if groups and r1 <= r0:
            continue
        y, s, tops = ref.product8(a[r0:r1], sa[r0:r1], b[i], sb[i], b_rows, not whole)
        want[r0:r1] = once(y, out)
        if not whole:
            # The matrix unit takes 15 of 16 products to 2^-13 of the largest; it adds 8 sums of 16, then there are two products
            # and a sum a block, each to 2^-23 of the terms' magnitudes.  Then the type's rounding.
            want[r0:r1] = y
            t = tops * 15 * 2.0 ** -13 + s * (8 + 3 * nb) * 2.0 ** -23
            tol[r0:r1] = t + (np.abs(y) + t) * ref.HALF_STEP[out]
    if nan_scale and nb:
        assert np.isnan(got[at][m // 2]).all()
        got[at[m // 2]], want[m // 2], tol[m // 2] = 0, 0, 0
    off = np.abs(got[at] - want)
    assert (off <= tol).all(), (ex.last_launch(), np.argwhere(~(off <= tol))[:5], got[at][~(off <= tol)][:5], want[~(off <= tol)][:5])
    got[at] = fill
    assert (got == fill).all()
    return ex.last_launch()


@pytest.mark.parametrize("m, n, k", [
    (1, 1, 1), (1, 1, 128), (1, 300, 144), (17, 5, 15), (3, 16, 16), (128, 128, 256), (130, 129, 400), (16, 129, 1000), (64, 40, 1024),
    (257, 260, 128), (65, 257, 768), (5, 7, 0),
])
def test_product_of_codes(hip_device, m, n, k):
    matmul8_case(m, n, k)


@pytest.mark.parametrize("kw", [
    dict(a_kind="Fp8E5M2"), dict(b_kind="Fp8E5M2"), dict(a_kind="Fp8E5M2", b_kind="Fp8E5M2", out="F16"), dict(), dict(b_rows=1),
    dict(b_rows=1, out="F16", pad=16), dict(pad=16, out_pad=4), dict(pad=1, first=1), dict(pad=3, first=16, out_pad=1), dict(nan_scale=True),
    dict(workspace=0), dict(out="F16", out_pad=3),
])
def test_product_of_codes_types_and_strides(hip_device, kw):
    matmul8_case(70, 150, 400, **kw)
    matmul8_case(7, 150, 384, **kw)


@pytest.mark.parametrize("out", ["Bf16", "F16"])
@pytest.mark.parametrize("b_rows", [1, 128])
def test_product_of_codes_of_real_numbers(hip_device, out, b_rows):
    matmul8_case(33, 140, 1111, out=out, b_rows=b_rows, whole=False, pad=9)
    matmul8_case(140, 260, 1024, out=out, b_rows=b_rows, whole=False, b_kind="Fp8E5M2")


@pytest.mark.parametrize("m, n, k, groups, way", [
    (1, 20, 128, 1, "all"), (64, 130, 256, 64, "all"), (300, 40, 144, 5, "all"), (300, 129, 256, 7, "gaps"), (200, 64, 128, 130, "all"),
    (129, 256, 272, 3, "one"), (2, 17, 128, 300, "all"), (5, 16, 0, 2, "gaps"), (700, 40, 128, 3, "gaps"),
])
@pytest.mark.parametrize("pad", [0, 16, 1])
def test_product_of_codes_by_group(hip_device, m, n, k, groups, way, pad):
    matmul8_case(m, n, k, groups=groups, way=way, pad=pad)


@pytest.mark.parametrize("starts", [[-5, 3, 40, 1000], [0, 0, 0, 0], [40, 40, 40, 40], [50, 50, 60, 70]])
def test_starts_outside_the_rows(hip_device, starts):
    matmul8_case(40, 30, 128, groups=3, starts=starts)
    grouped_case("forward", 40, 30, 64, 3, starts=starts)
    grouped_case("weight", 40, 32, 64, 3, starts=starts)


def test_starts_that_decrease_stay_inside(hip_device):
    """Which group takes a row is not said; the rows that are written, and nothing else, may hold anything."""
    for starts in ([0, 40, 0, 40, 0, 40], [40, 0, 40, 0, 40, 0], [2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1, 0, -1]):
        for direction in DIRECTIONS:
            m, n, k, groups = 40, 24, 64, 5
            x = dev(held(np.ones((m, 64)), "Bf16"))
            w = dev(held(np.ones((groups, 64, 64)), "Bf16"))
            out = dev(np.full(groups * 64 * 64 + 64, 7, np.uint16))
            ex = executor("lower_grouped_matmul", dtype="Bf16", out="Bf16", direction=direction)
            strides = (64, 64, 64 * 64, 64) if direction == "weight" else (64, 64 * 64, 64, 64)
            run(ex, x, w, dev(np.array(starts, np.int32)), out, u.DeviceBuffer(16), m, n, k, groups, *strides, 0)
            got = out.download(np.uint16, groups * 64 * 64 + 64)
            last = groups * 64 * 64 if direction == "weight" else m * 64
            assert (got[last:] == 7).all()


def grouped_case(direction, rows, n, k, groups, dtype="Bf16", out=None, way="all", pad=0, first=0, seed=0, whole=True, workspace=None,
                 starts=None, out_pad=0, x_pad=None):
    rng = np.random.default_rng(seed)
    out = dtype if out is None else out
    weight, wide = direction == "weight", k if direction == "forward" else n
    starts = starts_of(rng, rows, groups, way) if starts is None else np.asarray(starts)
    draw = (lambda s: rng.integers(-3, 4, s).astype(float)) if whole else (lambda s: rounded(rng.normal(size=s), dtype))
    x, w = draw((rows, wide)), draw((rows, k) if weight else (groups, n, k))
    if whole:
        assert 9 * max(rows, n, k) < 1 << 24
    nan = held(np.array([np.nan]), dtype)[0]
    # Rows that no group names hold NaN.
    named = np.zeros(rows, bool)
    for r0, r1 in ref.bounds(starts, rows):
        named[r0:r1] = True
    xs = np.where(named[:, None], x, np.nan)
    xa, x_row, _ = laid(held(xs, dtype), pad if x_pad is None else x_pad, first, nan)
    wa, w_row, w_group = laid(held(np.where(named[:, None], w, np.nan) if weight else w, dtype), pad, first, nan)
    shape = (groups, n, k) if weight else (rows, n if direction == "forward" else k)
    fill = 9.0
    oa, out_row, out_group = laid(held(np.full(shape, fill), out), out_pad, 4 * (out_pad > 0), held(np.array([fill]), out)[0])
    ob, size, osize = dev(oa), held(np.zeros(1), dtype).itemsize, held(np.zeros(1), out).itemsize
    ex = executor("lower_grouped_matmul", dtype=dtype, out=out, direction=direction)
    need = ex.workspace_bytes(rows, n, k, groups)
    ws = need if workspace is None else workspace
    strides = (x_row, w_row, out_group, out_row) if weight else (x_row, w_group, w_row, out_row)
    run(ex, dev(xa).at(first * size), dev(wa).at(first * size), dev(starts.astype(np.int32)), ob.at(4 * (out_pad > 0) * osize),
        dev(np.full(ws + 16, 0xFF, np.uint8)), rows, n, k, groups, *strides, ws)
    got = read(ob, len(oa), out)
    want, size_of = np.full(shape, fill), np.zeros(shape)
    for g, (r0, r1) in enumerate(ref.bounds(starts, rows)):
        if weight:
            want[g], size_of[g] = x[r0:r1].T @ w[r0:r1], np.abs(x[r0:r1]).T @ np.abs(w[r0:r1])
        elif r1 > r0:
            m = w[g].T if direction == "forward" else w[g]
            want[r0:r1], size_of[r0:r1] = x[r0:r1] @ m, np.abs(x[r0:r1]) @ np.abs(m)
    depth = rows if weight else wide
    # An instruction adds 32 products to a sum, each to 2^-23 of the terms' magnitudes; parts of a split depth are added after.
    # Below 2^-14 F16 counts in steps of 2^-24, so that a rounding there is off by 2^-25 whatever the value.
    step = np.maximum(np.abs(want) * ref.HALF_STEP[out], 2.0 ** -25 if out == "F16" else 0)
    tol = 0 if whole else size_of * (depth / 32 + 32) * 2.0 ** -23 * (1 + ref.HALF_STEP[out]) + step
    lead = np.arange(int(np.prod(shape[:-1])))[:, None] * out_row + np.arange(shape[-1])
    at = 4 * (out_pad > 0) + lead.reshape(shape)
    off = np.abs(got[at] - (once(want, out) if whole else want))
    assert (off <= tol).all(), (ex.last_launch(), np.argwhere(~(off <= tol))[:5], got[at][~(off <= tol)][:5], want[~(off <= tol)][:5])
    got[at] = fill
    assert (got == fill).all()
    return ex.last_launch()


@pytest.mark.parametrize("direction", DIRECTIONS)
@pytest.mark.parametrize("rows, n, k, groups, way", [
    (1, 8, 8, 1, "all"), (1, 1, 1, 1, "all"), (64, 136, 72, 64, "all"), (300, 40, 200, 5, "gaps"), (200, 264, 64, 130, "all"),
    (129, 64, 264, 3, "one"), (2, 16, 520, 300, "all"), (33, 17, 65, 2, "all"), (700, 40, 128, 3, "gaps"), (1030, 130, 136, 2, "one"),
])
def test_grouped_product(hip_device, direction, rows, n, k, groups, way):
    grouped_case(direction, rows, n, k, groups, way=way)


@pytest.mark.parametrize("direction", DIRECTIONS)
@pytest.mark.parametrize("kw", [
    dict(dtype="F16"), dict(dtype="F16", out="F32"), dict(out="F32", pad=8, out_pad=4), dict(pad=1, first=1), dict(pad=3, first=8, out_pad=1),
    dict(workspace=0), dict(out="F32", out_pad=2),
])
def test_grouped_product_types_and_strides(hip_device, direction, kw):
    grouped_case(direction, 150, 72, 200, 3, way="gaps", **kw)
    grouped_case(direction, 9, 72, 200, 4, way="all", **kw)


@pytest.mark.parametrize("direction", DIRECTIONS)
@pytest.mark.parametrize("dtype, out", [("Bf16", "Bf16"), ("F16", "F16"), ("Bf16", "F32")])
def test_grouped_product_of_real_numbers(hip_device, direction, dtype, out):
    grouped_case(direction, 333, 264, 520, 3, dtype, out, whole=False)
    grouped_case(direction, 40, 1000, 264, 7, dtype, out, whole=False)


@pytest.mark.parametrize("direction", DIRECTIONS)
def test_grouped_product_without_depth_or_rows(hip_device, direction):
    """A sum of nothing is 0; no rows, no groups and no columns are nothing to do."""
    ex = executor("lower_grouped_matmul", dtype="F16", out="F16", direction=direction)
    x, w, st, ws = dev(np.zeros(4096, np.float16)), dev(np.zeros(4096, np.float16)), dev(np.array([0, 3, 3], np.int32)), u.DeviceBuffer(16)
    out = dev(np.full(4096, 9, np.float16))
    sizes = {"forward": (3, 16, 0), "input": (3, 0, 16), "weight": (0, 8, 16)}[direction]
    strides = (16, 16, 128, 16) if direction == "weight" else (16, 256, 16, 16)
    run(ex, x, w, st, out, ws, *sizes, 2, *strides, 0)
    got = out.download(np.float16, 4096)
    live = 2 * 128 if direction == "weight" else 48
    assert (got[:live] == 0).all() and (got[live:] == 9).all()
    for sizes in ((0, 16, 16), (3, 0, 0)) if direction != "weight" else ((3, 0, 16), (3, 16, 0)):
        ex.launch(x, w, st, out, ws, *sizes, 2, *strides, 0)
    ex.launch(x, w, st, out, ws, 3, 16, 16, 0, *strides, 0)


def test_products_refuse(hip_device):
    ex = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="F16", b_rows=128, grouped=False)
    a, s, out, ws, null = u.DeviceBuffer(4096), dev(np.ones(64, np.float32)), u.DeviceBuffer(4096), u.DeviceBuffer(64), u.DeviceBuffer.held(0, 0, None)
    good = [a, s, a, s, out, ws, 4, 8, 128, 128, 1, 128, 1, 8, 0]
    ex.launch(*good)

    def bad(**at):
        args = list(good)
        for i, v in at.items():
            args[int(i[1:])] = v
        invalid(ex, *args)

    invalid(ex, *good[:-1])
    bad(_0=null), bad(_1=null), bad(_2=null), bad(_3=null), bad(_4=null), bad(_6=-1), bad(_7=-1), bad(_8=-1)
    bad(_6=(1 << 28) + 1), bad(_9=-1), bad(_13=7), bad(_14=-1), bad(_4=out.at(1)), bad(_5=ws.at(4)), bad(_1=s.at(2)), bad(_13=1 << 62)
    bad(_5=null, _14=64)
    g = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="F16", b_rows=128, grouped=True)
    st = dev(np.array([0, 4], np.int32))
    good = [a, s, a, s, st, out, ws, 4, 8, 128, 1, 128, 1, 128, 1, 1024, 1, 8, 0]
    g.launch(*good)
    for i, v in ((10, 1025), (10, -1), (4, null), (4, st.at(2)), (15, -1)):
        invalid(g, *good[:i], v, *good[i + 1:])
    w = executor("lower_grouped_matmul", dtype="Bf16", out="F32", direction="weight")
    st = dev(np.array([0, 4, 4], np.int32))
    good = [a, a, st, out, ws, 4, 8, 16, 2, 8, 16, 128, 16, 0]
    w.launch(*good)
    for i, v in ((11, 127), (12, 15), (9, -8), (3, out.at(2)), (0, a.at(1)), (5, (1 << 28) + 1)):
        invalid(w, *good[:i], v, *good[i + 1:])
    u.synchronize()
    for e, scalars in ((ex, (1, 2)), (g, (1, 2, 3)), (w, (1, 2, 3)), (ex, (1, -2, 3))):
        with pytest.raises(u.UnpError):
            e.workspace_bytes(*scalars)
    assert w.workspace_bytes(rows=4, n=8, k=16, groups=2) == w.workspace_bytes(4, 8, groups=2, k=16)
    with pytest.raises(TypeError):
        w.workspace_bytes(4, 8, 16, batch=2)


# ---------------------------------------------------------------------------------------
# The rows of each group
# ---------------------------------------------------------------------------------------
def rows_case(count, per, groups, index="I32", way="any", workspace=None, seed=0):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, groups, count)
    if way == "any":
        ids[rng.random(count) < 0.1] = rng.choice([-1, groups, 2 ** 31 - 1, -2 ** 31])
    if way == "one":
        ids[:] = groups - 1
    if way == "none":
        ids[:] = -1
    if index == "I64" and count > 4 and way == "any":
        ids[3], ids[4] = 1 << 32, -1 << 40
    starts, rows, place = ref.group_rows(ids, per, groups)
    ex = executor("lower_group_rows", index_dtype=index)
    need = ex.workspace_bytes(count, per, groups)
    ws = need if workspace is None else workspace
    bufs = [dev(np.full(n + 4, 77, np.int32)) for n in (groups + 1, count, count)]
    run(ex, dev(ids.astype(ref.INDEX[index])), *bufs, u.DeviceBuffer(max(ws, 16)), count, per, groups, ws)
    for buf, want in zip(bufs, (starts, rows, place)):
        got = buf.download(np.int32, len(want) + 4)
        assert np.array_equal(got[:-4], want) and (got[-4:] == 77).all()
    return ex.last_launch()


@pytest.mark.parametrize("count, per, groups, index, way", [
    (1, 1, 1, "I32", "any"), (5, 1, 1024, "I64", "any"), (64, 4, 8, "I32", "any"), (511, 2, 100, "I32", "any"), (512, 8, 3, "I64", "one"),
    (513, 3, 7, "I32", "none"), (4096, 4, 64, "I32", "any"), (4097, 1, 64, "I32", "any"), (30000, 6, 129, "I64", "any"),
    (131072, 8, 128, "I32", "any"), (70001, 2, 1000, "I32", "one"),
])
def test_rows_of_groups(hip_device, count, per, groups, index, way):
    rows_case(count, per, groups, index, way)


def test_rows_of_groups_with_less_workspace(hip_device):
    assert rows_case(20000, 2, 64)["chunks"] > rows_case(20000, 2, 64, workspace=4 * 64 * 3)["chunks"] == 3
    assert rows_case(20000, 2, 64, workspace=0)["chunks"] == 1


def test_rows_of_groups_refuse(hip_device):
    ex = executor("lower_group_rows", index_dtype="I32")
    b, null = u.DeviceBuffer(1024), u.DeviceBuffer.held(0, 0, None)
    good = [dev(np.zeros(8, np.int32)), b, b.at(256), b.at(512), b.at(768), 8, 2, 4, 0]
    ex.launch(*good)
    for i, v in ((0, null), (1, null), (1, b.at(2)), (5, -1), (5, (1 << 28) + 1), (6, 0), (7, 0), (7, 1025), (8, -1)):
        invalid(ex, *good[:i], v, *good[i + 1:])
    ex.launch(null, b, null, null, null, 0, 1, 4, 0)
    u.synchronize()
    assert (b.download(np.int32, 5) == 0).all()


# ---------------------------------------------------------------------------------------
# Each kernel, at the edges of its tiles
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("m, n, k, kw, entry", [
    (1, 100, 2048, {}, "_one"), (16, 33, 1040, {}, "_one"), (17, 64, 1024, {}, "_slim"), (32, 2100, 272, {}, "_slim"),
    (33, 128, 1024, {}, "_slim"), (64, 130, 2176, dict(b_rows=1), "_one"), (65, 129, 1168, {}, "_one"), (200, 300, 128, dict(b_rows=1), "_slim"),
    (2049, 3849, 144, {}, "_wide"), (2817, 2820, 400, dict(b_rows=1), "_wide"), (2817, 2561, 16, dict(a_kind="Fp8E5M2"), "_tile"),
    (2817, 2700, 272, dict(out="F16", out_pad=1), "_tile"), (130, 140, 200, dict(pad=1), "_any"), (3, 5, 128, dict(pad=1), "_any"),
    # Lengths that end inside 16 bytes, in rows of whole vectors.
    (1, 100, 2001, dict(pad=15), "_one"), (20, 100, 1039, dict(pad=1), "_one"), (60, 130, 129, dict(pad=15), "_slim"), (70, 129, 1151, dict(pad=1), "_one"),
    (2817, 2561, 257, dict(pad=15), "_tile"), (2817, 2561, 7, dict(pad=9, first=16), "_tile"), (2817, 2561, 143, dict(pad=1, b_rows=1), "_tile"),
    (100, 2100, 16, {}, "_few"), (33, 8200, 143, dict(pad=1), "_few"), (65, 4100, 272, dict(b_rows=1), "_few"), (31, 8200, 1039, dict(pad=1), "_few"),
    (100, 8200, 143, dict(pad=1), "_some"), (600, 2100, 272, dict(b_rows=1), "_some"), (4000, 264, 144, dict(a_kind="Fp8E5M2"), "_some"),
    (1000, 2100, 16, {}, "_tile"), (2049, 2561, 257, dict(pad=15), "_tile"), (4000, 2561, 272, {}, "_wide"), (4000, 2100, 143, dict(pad=1, b_rows=1), "_wide"),
    (2817, 4100, 257, dict(pad=15, out="F16", out_pad=1), "_wide"), (4000, 8200, 7, dict(pad=9, first=16), "_wide"),
])
def test_product_of_codes_by_kernel(hip_device, m, n, k, kw, entry):
    assert matmul8_case(m, n, k, **kw)["entry"].endswith(entry)


@pytest.mark.parametrize("m, n, k, groups, way, entry", [
    (40, 48, 256, 8, "all", "_slim"), (500, 2100, 144, 40, "gaps", "_few"), (500, 260, 640, 10, "all", "_slim"), (900, 300, 272, 6, "gaps", "_few"),
    (4000, 2300, 144, 5, "gaps", "_wide"), (3500, 2561, 272, 2, "one", "_wide"),
    (40, 48, 1040, 8, "all", "_slim"), (40, 48, 2064, 8, "all", "_one"), (500, 1100, 640, 10, "all", "_few"), (900, 1300, 272, 6, "gaps", "_some"), (2000, 2100, 272, 6, "gaps", "_tile"),
])
def test_product_of_codes_by_group_and_kernel(hip_device, m, n, k, groups, way, entry):
    assert matmul8_case(m, n, k, groups=groups, way=way)["entry"].endswith(entry)


@pytest.mark.parametrize("direction, rows, n, k, groups, way, entry", [
    ("forward", 40, 48, 256, 8, "all", "_slim"), ("forward", 500, 2104, 136, 40, "gaps", "_few"), ("forward", 500, 264, 640, 10, "all", "_slim"),
    ("forward", 900, 304, 72, 6, "gaps", "_few"), ("forward", 4000, 2304, 72, 5, "gaps", "_wide"), ("forward", 3500, 2561, 200, 2, "one", "_wide"),
    ("input", 40, 256, 48, 8, "all", "_slim"), ("input", 500, 136, 2104, 40, "gaps", "_few"), ("input", 500, 640, 264, 10, "all", "_slim"),
    ("input", 900, 72, 304, 6, "gaps", "_few"), ("input", 4000, 72, 2304, 5, "gaps", "_wide"), ("input", 3500, 200, 2568, 2, "one", "_wide"),
    ("weight", 300, 264, 520, 3, "gaps", "_tile"), ("weight", 700, 1104, 1288, 6, "gaps", "_wide"), ("weight", 131, 2312, 2824, 2, "one", "_wide"),
    ("weight", 300, 2056, 2056, 2, "all", "_wide"),
    ("forward", 40, 48, 1040, 8, "all", "_one"), ("forward", 900, 1304, 136, 6, "gaps", "_some"), ("forward", 2000, 2104, 136, 6, "gaps", "_tile"),
    ("input", 40, 1040, 48, 8, "all", "_one"), ("input", 900, 136, 1304, 6, "gaps", "_some"), ("input", 2000, 136, 2104, 6, "gaps", "_tile"),
])
def test_grouped_product_by_kernel(hip_device, direction, rows, n, k, groups, way, entry):
    assert grouped_case(direction, rows, n, k, groups, way=way)["entry"].endswith(entry)


@pytest.mark.parametrize("direction, rows, n, k, groups, pad, entry", [
    ("forward", 40, 48, 257, 8, 7, "_slim"), ("forward", 900, 304, 71, 6, 1, "_few"), ("forward", 4000, 2304, 129, 5, 7, "_wide"),
    ("input", 40, 257, 48, 8, 7, "_slim"), ("input", 900, 71, 304, 6, 1, "_few"), ("input", 4000, 129, 2304, 5, 7, "_wide"),
    ("forward", 40, 48, 1041, 8, 7, "_one"), ("forward", 900, 1304, 135, 6, 1, "_some"), ("forward", 2000, 2104, 71, 6, 1, "_tile"),
    ("input", 40, 1041, 48, 8, 7, "_one"), ("input", 900, 135, 1304, 6, 1, "_some"), ("input", 2000, 71, 2104, 6, 1, "_tile"),
])
def test_grouped_product_of_lengths_inside_a_vector(hip_device, direction, rows, n, k, groups, pad, entry):
    """The depth alone; the columns of an operand that lie along out are whole vectors."""
    if direction == "forward":
        assert grouped_case(direction, rows, n, k, groups, way="gaps", pad=pad)["entry"].endswith(entry)
    else:
        assert grouped_case(direction, rows, n, k, groups, way="gaps", pad=8, x_pad=pad)["entry"].endswith(entry)


@pytest.mark.parametrize("workspace", [None, 0])
def test_a_split_depth_gives_the_same_whole_numbers(hip_device, workspace):
    parts = [matmul8_case(60, 200, 28000, top=1, workspace=workspace)["chunks"],
             grouped_case("forward", 60, 136, 16384, 2, way="gaps", workspace=workspace)["chunks"],
             grouped_case("input", 60, 16384, 136, 1, workspace=workspace)["chunks"],
             grouped_case("weight", 4096, 136, 200, 2, out="F32", workspace=workspace)["chunks"]]
    assert all(p > 1 for p in parts) if workspace is None else parts == [1] * 4


def test_a_split_depth_that_ends_inside_a_vector(hip_device):
    parts = [matmul8_case(60, 200, 28001, top=1, pad=15)["chunks"], matmul8_case(33, 70, 20007, top=1, pad=9, b_rows=1)["chunks"],
             grouped_case("forward", 60, 136, 16385, 2, way="gaps", pad=7)["chunks"],
             grouped_case("input", 60, 16391, 136, 1, pad=8, x_pad=1)["chunks"]]
    assert all(p > 1 for p in parts)


def test_more_tiles_than_a_launch_has(hip_device):
    ex, b, null = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="Bf16", b_rows=128, grouped=False), u.DeviceBuffer(64), \
        u.DeviceBuffer.held(0, 0, None)
    invalid(ex, null, null, null, null, b, b.at(16), 1 << 28, 1 << 28, 0, 0, 0, 0, 0, 1 << 28, 0)


@pytest.mark.parametrize("case", ["codes", "forward", "input", "weight", "weight16"])
def test_more_wide_tiles_than_compute_units(hip_device, case):
    """Tiles of 256 x 256, of whole and half heights, at the edges of each operand."""
    if case == "codes":
        starts = [0, 700, 700, 1000, 3111, 3240, 4200]
        got = matmul8_case(4300, 8200, 272, groups=6, starts=starts, out_pad=8)
    elif case == "forward":
        got = grouped_case("forward", 4300, 8200, 136, 6, way="gaps")
    elif case == "input":
        got = grouped_case("input", 4300, 136, 8200, 6, way="gaps")
    else:
        got = grouped_case("weight", 1000, 2104, 1544, 8, way="gaps", out="F32" if case == "weight" else "Bf16")
    assert got["entry"].endswith("_wide") and got["grid"][0] > 256, got


# ---------------------------------------------------------------------------------------
# As they are used: together, for gradients, on streams, in graphs and far apart
# ---------------------------------------------------------------------------------------
def gather(table, rows, out, n, cols, extent, dtype="Bf16"):
    key = ("gather", dtype)
    if key not in _execs:
        _execs[key] = u.Executor(B.lower_form(kind="gather", dtype=dtype, rank=2, index_dtype="I32", oob="ZeroFill"))
    _execs[key].launch(table, rows, out, n, cols, extent)


def test_experts_of_tokens_together(hip_device):
    """Choices to rows by expert, the tokens' rows gathered, their products in 16 bits and from codes, and the results gathered
    back to the choices, on the device from end to end."""
    rng = np.random.default_rng(5)
    tokens, per, groups, n, k = 37, 3, 6, 72, 136
    count = tokens * per
    ids = rng.integers(0, groups, count)
    ids[ids == 2] = 4  # an expert of no rows
    ids[::11] = -1     # choices of none
    x, w = rng.integers(-1, 2, (tokens, k)).astype(float), rng.integers(-1, 2, (groups, n, k)).astype(float)
    starts, rows, place = ref.group_rows(ids, per, groups)
    d_starts, d_rows, d_place = (u.DeviceBuffer(4 * s) for s in (groups + 1, count, count))
    sort = executor("lower_group_rows", index_dtype="I32")
    sort.launch(dev(ids.astype(np.int32)), d_starts, d_rows, d_place, u.DeviceBuffer(16), count, per, groups, 0)
    d_x, d_xs = dev(held(x, "Bf16")), u.DeviceBuffer(2 * count * k)
    gather(d_x, d_rows, d_xs, count, k, tokens)
    # In 16 bits: sums of at most k products of -1, 0 and 1 are whole numbers that bf16 holds.
    ex = executor("lower_grouped_matmul", dtype="Bf16", out="Bf16", direction="forward")
    d_y, d_out = dev(np.zeros(count * n, np.uint16)), u.DeviceBuffer(2 * count * n)
    need = ex.workspace_bytes(count, n, k, groups)
    ex.launch(d_xs, dev(held(w, "Bf16")), d_starts, d_y, u.DeviceBuffer(max(need, 16)), count, n, k, groups, k, n * k, k, n, need)
    gather(d_y, d_place, d_out, count, n, count)
    u.synchronize()
    assert np.array_equal(d_starts.download(np.int32, groups + 1), starts)
    want = np.zeros((count, n))
    for i, g in enumerate(ids):
        if g >= 0:
            want[i] = w[g] @ x[i // per]
    assert np.array_equal(read(d_out, count * n, "Bf16").reshape(count, n), want)
    # From codes: the rows' and the weights' scales are the device's own.
    blocks = -(-k // 128)
    quant = executor("lower_quant8", dtype="Bf16", kind="Fp8E4M3FN", block_rows=1, transpose=False)
    d_a, d_sa = u.DeviceBuffer(count * k), u.DeviceBuffer(4 * count * blocks)
    quant.launch(d_xs, d_a, d_sa, count, k, k, k, blocks)
    wide = executor("lower_quant8", dtype="F32", kind="Fp8E4M3FN", block_rows=128, transpose=False)
    d_b, d_sb = u.DeviceBuffer(groups * n * k), u.DeviceBuffer(4 * groups * blocks)
    for g in range(groups):
        wide.launch(dev(w[g].astype(np.float32)), d_b.at(g * n * k), d_sb.at(4 * g * blocks), n, k, k, k, blocks)
        u.synchronize()
    ex = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="Bf16", b_rows=128, grouped=True)
    need = ex.workspace_bytes(count, n, k, groups)
    ex.launch(d_a, d_sa, d_b, d_sb, d_starts, d_y, u.DeviceBuffer(max(need, 16)), count, n, k, groups, k, blocks, k, blocks, n * k, blocks,
              n, need)
    gather(d_y, d_place, d_out, count, n, count)
    u.synchronize()
    got = read(d_out, count * n, "Bf16").reshape(count, n)
    # 1 is the code 448 times f32(1 / 448), off by 2^-24: a product of two is off by 2^-23 and two blocks' sum of magnitudes is at
    # most k.  Two of the matrix unit's sums of 16 keep 2^-13 of the largest term, which is 1, in each of k / 16 + 1 runs for 15
    # products; then sums of 11 steps a block to 2^-23, and bf16's half step.
    tol = k * (2.0 ** -22 + (8 + 3 * blocks) * 2.0 ** -23) + (k / 16 + 1) * 15 * 2.0 ** -13
    assert (np.abs(got - want) <= tol + (np.abs(want) + tol) * 2.0 ** -8).all()
    assert (got[ids < 0] == 0).all()


def test_gradients_against_differences(hip_device):
    """A product is linear in its rows and in its weights: the change of sum(c * y) over any step is the gradient's sum."""
    rng = np.random.default_rng(8)
    rows, n, k, groups = 150, 88, 104, 5
    starts = starts_of(rng, rows, groups, "all")
    whole = lambda s: rng.integers(-2, 3, s).astype(float)  # noqa: E731
    x, w, c, dx, dw = whole((rows, k)), whole((groups, n, k)), whole((rows, n)), whole((rows, k)), whole((groups, n, k))

    def product(direction, a, b, shape, strides):
        out = "F32"
        ex = executor("lower_grouped_matmul", dtype="F16", out=out, direction=direction)
        size, buf = ex.workspace_bytes(rows, n, k, groups), dev(np.zeros(shape, np.float32))
        ex.launch(dev(held(a, "F16")), dev(held(b, "F16")), dev(starts.astype(np.int32)), buf, u.DeviceBuffer(max(size, 16)), rows, n, k,
                  groups, *strides, size)
        u.synchronize()
        return read(buf, int(np.prod(shape)), out).reshape(shape)

    forward = lambda x, w: (c * product("forward", x, w, (rows, n), (k, n * k, k, n))).sum()  # noqa: E731
    gx = product("input", c, w, (rows, k), (n, n * k, k, k))
    gw = product("weight", c, x, (groups, n, k), (n, k, n * k, k))
    at = forward(x, w)
    assert forward(x + dx, w) - at == (gx * dx).sum() != 0
    assert forward(x, w + dw) - at == (gw * dw).sum() != 0


def steps_for_streams():
    """Launches of each form with every buffer of their own: (launch(stream, how), output, bytes of it, workspace or None)."""
    rng = np.random.default_rng(2)
    found = []

    def codes(shape):
        return dev(ref.encoded(rng.normal(size=shape), "Fp8E4M3FN"))

    def add(ex, buffers, out, size, need, scalars):
        ws = u.DeviceBuffer(max(need, 16)) if need is not None else None
        args = [*buffers, *([ws] if ws else []), *scalars, *([need] if ws else [])]
        found.append((lambda stream, how="launch", ex=ex, args=args: getattr(ex, how)(*args, stream=stream), out, size, ws, ex))

    m, n, k = 60, 200, 28000
    blocks, sides = -(-k // 128), -(-n // 128)
    ex, out = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="F16", b_rows=128, grouped=False), u.DeviceBuffer(2 * m * n)
    add(ex, [codes((m, k)), dev(np.exp(rng.normal(size=(m, blocks))).astype(np.float32)), codes((n, k)),
             dev(np.exp(rng.normal(size=(sides, blocks))).astype(np.float32) / 100), out], out, 2 * m * n,
        ex.workspace_bytes(m, n, k), [m, n, k, k, blocks, k, blocks, n])
    rows, n, k, g = 5000, 136, 200, 2
    starts = dev(np.array([0, 2100, 5000], np.int32))
    ex, out = executor("lower_grouped_matmul", dtype="Bf16", out="F32", direction="weight"), u.DeviceBuffer(4 * g * n * k)
    add(ex, [dev(held(rng.normal(size=(rows, n)), "Bf16")), dev(held(rng.normal(size=(rows, k)), "Bf16")), starts, out], out, 4 * g * n * k,
        ex.workspace_bytes(rows, n, k, g), [rows, n, k, g, n, k, n * k, k])
    m, n, k, g = 4300, 2304, 264, 3
    ex, out = executor("lower_grouped_matmul", dtype="Bf16", out="Bf16", direction="forward"), u.DeviceBuffer(2 * m * n)
    add(ex, [dev(held(rng.normal(size=(m, k)), "Bf16")), dev(held(rng.normal(size=(g, n, k)), "Bf16")),
             dev(np.array([0, 1000, 4200, 4300], np.int32)), out], out, 2 * m * n, ex.workspace_bytes(m, n, k, g),
        [m, n, k, g, k, n * k, k, n])
    r, c = 700, 900
    ex, out = executor("lower_quant8", dtype="F32", kind="Fp8E5M2", block_rows=128, transpose=True), u.DeviceBuffer(r * c)
    add(ex, [dev(rng.normal(size=(r, c)).astype(np.float32)), out, u.DeviceBuffer(4 * 64)], out, r * c, None, [r, c, c, r, 6])
    count, g = 20000, 64
    ex, out = executor("lower_group_rows", index_dtype="I32"), u.DeviceBuffer(4 * count)
    add(ex, [dev(rng.integers(-1, g, count).astype(np.int32)), u.DeviceBuffer(4 * (g + 1)), out, u.DeviceBuffer(4 * count)], out, 4 * count,
        ex.workspace_bytes(count, 4, g), [count, 4, g])
    return found


def test_streams_graphs_and_workspaces(hip_device):
    """Each form captured into a graph and replayed between eager work, all of them at once on streams of their own, timed and
    without allocation: the same bits every time."""
    L = _lib.lib()
    steps, raw, streams, graphs = steps_for_streams(), [], [], []
    split = 0
    for launch, out, size, ws, ex in steps:
        launch(0)
        u.synchronize()
        split += ex.last_launch()["shared"]
        raw.append(out.download(np.uint8, size))
        out.fill(0x5A)
        launch(0, "launch_static")
        a, b = u.Event(), u.Event()
        ex.set_timing(a, b)
        launch(0)
        u.synchronize()
        assert 0 < a.elapsed_ms(b) < 1000
        ex.set_timing(None, None)
        assert np.array_equal(out.download(np.uint8, size), raw[-1])
    assert split >= 3  # the split products and the rows of groups have kernels that follow one another
    for launch, *_ in steps:
        st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
        assert L.hipStreamCreate(C.byref(st)) == 0
        assert L.hipStreamBeginCapture(st, 0) == 0
        launch(st.value)
        assert L.hipStreamEndCapture(st, C.byref(graph)) == 0
        assert L.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        streams.append(st)
        graphs.append((graph, exe))
    others = steps_for_streams()
    for turn in range(4):
        for _, out, _, ws, _ in steps:
            out.fill(0)
            if ws:
                ws.fill(0xFF)
        u.synchronize()
        for _ in range(3):
            for (_, exe), st in zip(graphs, streams):
                assert L.hipGraphLaunch(exe, st) == 0
        others[turn][0](0)  # eager work on buffers of its own beside them
        u.synchronize()
        for (_, out, size, _, _), r in zip(steps, raw):
            assert np.array_equal(out.download(np.uint8, size), r), turn
    for (launch, out, *_), st in zip(steps, streams):
        out.fill(0)
        u.synchronize()
        launch(st.value)
    u.synchronize()
    for (_, out, size, _, _), r in zip(steps, raw):
        assert np.array_equal(out.download(np.uint8, size), r)
    for graph, exe in graphs:
        assert L.hipGraphExecDestroy(exe) == 0 and L.hipGraphDestroy(graph) == 0
    for st in streams:
        assert L.hipStreamDestroy(st) == 0


@pytest.mark.parametrize("direct", [True, False])
def test_products_past_four_gigabytes(hip_device, direct):
    """Rows, groups and results at byte offsets that need more than 32 bits, in rows that load directly and in others."""
    rng = np.random.default_rng(4)
    m, n, k, groups = 1300, 17, 256, 2
    a_row, b_row, out_row, b_group = (1 << 22) if direct else (1 << 22) + 1, 256, 1 << 21, (5 << 30) + (0 if direct else 2)
    a, b = rng.integers(-4, 5, (m, k)).astype(float), rng.integers(-4, 5, (groups, n, k)).astype(float)
    da, db, do = u.DeviceBuffer(m * a_row + 16), u.DeviceBuffer(b_group + n * b_row), u.DeviceBuffer(m * out_row * 2)
    for i in range(m):
        da.at(i * a_row).upload(ref.encoded(a[i], "Fp8E4M3FN"))
    for g in range(groups):
        db.at(g * b_group).upload(ref.encoded(b[g], "Fp8E4M3FN"))
    ones = dev(np.ones(2 * m, np.float32))
    starts = dev(np.array([0, 70, m], np.int32))
    ex = executor("lower_matmul8", a_kind="Fp8E4M3FN", b_kind="Fp8E4M3FN", out="Bf16", b_rows=128, grouped=True)
    run(ex, da, ones, db, ones, starts, do, u.DeviceBuffer(16), m, n, k, groups, a_row, 2, b_row, 2, b_group, 2, out_row, 0)
    assert ex.last_launch()["entry"].endswith("_any") != direct
    for i in (0, 1, 69, 70, 500, 1024, 1025, m - 1):
        assert np.array_equal(read(do.at(2 * i * out_row), n, "Bf16"), once(b[int(i >= 70)] @ a[i], "Bf16")), i
