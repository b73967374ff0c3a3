"""Cache attention over values whose scales lie far apart: between groups, between keys, and at keys that a row does not
see or hardly weighs."""
import numpy as np
import pytest

import unpopped_amd as u
from tests import cache4_reference as ref
from tests.test_gpu_cache4 import dev, executor, filled, run

pytestmark = pytest.mark.gpu


def with_value_scales(cache, slots, scales, zeros):
    """The value words of the slots set to f16 scales and zero points, [slots, heads, groups]."""
    for i, slot in enumerate(slots):
        for h in range(cache.heads):
            for g in range(cache.dim // cache.group):
                at = cache.word_at(slot % cache.page, g, True)
                word = int(np.float16(scales[i, h, g]).view(np.uint16)) | int(zeros[i, h, g]) << 16
                cache.bytes[slot // cache.page, h, at:at + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)


def of_scales(cache, slots, scales):
    """The cache with every value 15 |scale|."""
    c = ref.Cache(cache.bytes.shape[0], cache.heads, cache.dim, cache.group, cache.page)
    c.bytes[:] = cache.bytes
    half = cache.page * cache.dim // 2
    c.bytes[..., half:2 * half] = 0xFF
    with_value_scales(c, slots, np.abs(scales), np.zeros(scales.shape, int))
    return c


def tolerance(out, mass, fifteen, reach, keys, dim, dtype):
    """What rounding may do to an output, per element.  `fifteen` is the sum of p 15 |scale| of the element's group.

    * The probability and its product with the scale are each rounded once to 11 bits, scores and the softmax's sum as
      attention_tolerance has it: of sum p |v|.
    * The sums of p s n and of p s zero are in f32, codes and zeros of at most 15: (keys + 8) roundings of 2^-23 of `fifteen` each.
    * Where no two scales are further apart than 2^15, a probability is held to 2^-36 of the row's largest and a product to
      2^-36 of that and four times the largest scale: 5 x 2^-36 x 2^15 of the smallest scale, which `fifteen` is 15 times of
      at least, in each of keys: less than keys 2^-18 of it.  Where they are, a product is held to 2^-35 of the step's largest.
    * The output is rounded once to its type, whose smallest step is 2^-24 for F16 (below Bf16's no output here comes).
    """
    score = reach[..., None] * (30.0 / 7.0) * (dim + 4) * 2.0 ** -23
    off = mass * (2 * 2.0 ** -11 + 2 * score + (keys + 8) * 2.0 ** -23) + fifteen * (keys * 2.0 ** -18 + 2 * (keys + 8) * 2.0 ** -23)
    return off + (np.abs(out) + off) * ref.HALF_STEP[dtype] + (2.0 ** -25 if dtype == "F16" else 0.0)


def ranges_case(kind, dtype, heads, kv, dim, group, rows, lengths, page=16, window=0, workspace=True, entry=None):
    rng = np.random.default_rng(dim + group + len(rows) + rows[0])
    need = [-(-n // page) for n in lengths]
    pages, width, batch = sum(need) + 1, max(need), len(rows)
    order = rng.permutation(pages)
    table = np.full((batch, width), -1, np.int32)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    tokens, groups = int(starts[-1]), dim // group
    slots, exponent, fading = [], [], []
    for b, n in enumerate(lengths):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
        j = np.arange(n)
        slots += [int(table[b, i // page]) * page + i % page for i in j]
        e = np.full((n, kv, groups), -7.0)
        if kind == "groups":  # neighbouring groups 2^22 apart
            e[..., 0::2] = 11.0
            e[..., 1::2] = -11.0
        elif kind == "later":  # the last keys' are 2^18 above the others': most rows do not see them
            e[n - n // 4:] = 11.0
        elif kind == "earlier":  # the first keys', which the window hides
            e[:n - n // 4] = 11.0
        elif kind == "faint":  # some keys that every row sees, by e^-15 to e^-40, 2^14 to 2^22 above the others
            e[n // 4::7] = 11.0 - rng.integers(0, 5)
        elif kind == "small":  # down to the smallest f16 numbers
            e[:] = rng.integers(-24, -8, e.shape)
        elif kind == "any":
            e[:] = rng.integers(-20, 12, e.shape)
        fading += list((kind == "faint") & (e[:, 0, 0] > -7.0))
        exponent.append(e)
    exponent, slots = np.concatenate(exponent), np.array(slots)
    cache = filled(rng, pages, kv, dim, group, page, dtype, slots)
    q = ref.rounded(rng.normal(size=(tokens, heads, dim)), dtype)
    if kind == "faint":
        q = ref.rounded(np.abs(q) * 0.4 + 0.5, dtype)
        for s in slots[np.array(fading)]:
            for h in range(kv):
                cache.put(int(s), h, ref.rounded(np.full(dim, -rng.uniform(20, 50) / np.sqrt(dim)), dtype), False)
    scales = np.ldexp(rng.uniform(1, 2, exponent.shape), exponent.astype(int)).astype(np.float16).astype(np.float64)
    if kind == "any":
        scales *= rng.choice([-1, 1], scales.shape)
    with_value_scales(cache, slots, scales, rng.integers(0, 16, scales.shape))
    args = (table, starts, np.array(lengths), True, window)
    want, _, mass, _, reach = ref.attend(q, cache, *args)
    fifteen = ref.attend(q, of_scales(cache, slots, scales), *args)[0]
    ex = executor("lower_cache4_attention", dtype=dtype, heads=heads, kv_heads=kv, head_dim=dim, group=group, page=page)
    size = ex.workspace_bytes(tokens, batch, width, pages) if workspace else 0
    out, strides = dev(np.zeros(q.size, np.uint16)), (heads * dim, dim) * 2
    run(ex, dev(ref.stored(q, dtype)), dev(cache.bytes), dev(table), dev(starts), dev(np.array(lengths, np.int32)), out,
        dev(np.zeros(size + 16, np.uint8)), tokens, batch, width, pages, *strides, window, size)
    if entry:
        assert ex.last_launch()["entry"].endswith(entry)
    got = ref.loaded(out.download(np.uint16, q.size), dtype).reshape(q.shape)
    off = np.abs(got - want) / tolerance(want, mass, fifteen, reach, max(lengths), dim, dtype)
    at = np.unravel_index(np.nanargmax(off), off.shape)
    print(kind, "largest error / tolerance %.3g" % off[at], at, got[at], want[at], flush=True)
    assert (off <= 1).all()


KINDS = ["groups", "later", "earlier", "faint", "small", "any"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype, heads, kv, dim, group, rows, lengths, entry", [
    ("Bf16", 4, 2, 64, 32, [1, 1, 1], [40, 9, 300], "_few"),
    ("F16", 8, 2, 128, 128, [1, 1], [140, 33], "_few"),
    ("Bf16", 6, 1, 96, 32, [1], [90], "_few"),
    ("Bf16", 12, 2, 192, 192, [1, 2], [70, 300], "_some"),
    ("F16", 4, 1, 64, 64, [3, 4], [40, 50], "_some"),
    ("Bf16", 8, 4, 128, 64, [45], [700], "_more"),
    ("F16", 6, 2, 256, 32, [44, 20], [60, 900], "_more"),
    ("Bf16", 4, 2, 128, 128, [70, 41], [70, 90], "_many"),
    ("F16", 2, 2, 96, 96, [150], [150], "_many"),
    ("Bf16", 3, 1, 256, 64, [40], [50], "_many"),
])
def test_attention_over_scales_far_apart(hip_device, kind, dtype, heads, kv, dim, group, rows, lengths, entry):
    ranges_case(kind, dtype, heads, kv, dim, group, rows, lengths, window=7 if kind == "earlier" else 0, workspace=False, entry=entry)


@pytest.mark.parametrize("kind", ["groups", "faint", "any"])
@pytest.mark.parametrize("dtype, rows, n", [("Bf16", [1], 2300), ("F16", [1], 2300), ("Bf16", [12], 4400)])
def test_attention_of_split_contexts_over_scales_far_apart(hip_device, kind, dtype, rows, n):
    ranges_case(kind, dtype, 4, 1, 64, 32, rows, [n], page=64, entry="_join")


@pytest.mark.parametrize("dtype, rows", [("Bf16", 1), ("F16", 1), ("Bf16", 50)])
@pytest.mark.parametrize("dim, group", [(64, 32), (128, 128)])
def test_values_of_zero_beside_others(hip_device, dtype, rows, dim, group):
    """Keys whose values are all 0 (a scale of 0) and keys whose are not, in the same steps."""
    rng = np.random.default_rng(rows)
    n, page = 75, 16
    cache = filled(rng, 5, 1, dim, group, page, dtype, range(n))
    for s in range(0, n, 3):
        cache.put(s, 0, np.zeros(dim), True)
    q = ref.rounded(rng.normal(size=(rows, 2, dim)), dtype)
    table, starts, lengths = np.arange(5, dtype=np.int32)[None], np.array([0, rows], np.int32), np.array([n], np.int32)
    want, _, mass, top, reach = ref.attend(q, cache, table, starts, lengths)
    ex = executor("lower_cache4_attention", dtype=dtype, heads=2, kv_heads=1, head_dim=dim, group=group, page=page)
    out = dev(np.zeros(q.size, np.uint16))
    run(ex, dev(ref.stored(q, dtype)), dev(cache.bytes), dev(table), dev(starts), dev(lengths), out, dev(np.zeros(16, np.uint8)),
        rows, 1, 5, 5, 2 * dim, dim, 2 * dim, dim, 0, 0)
    got = ref.loaded(out.download(np.uint16, q.size), dtype).reshape(q.shape)
    assert (np.abs(got - want) <= ref.attention_tolerance(want, mass, top, reach, n, dim, dtype)).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("spread", [0, 20])
def test_a_scale_that_is_no_number_stays_with_its_group(hip_device, bad, spread):
    """Beside scales of one size and scales far apart: rows that do not see the key, and the other group, keep their values."""
    rng = np.random.default_rng(spread)
    dim, group, page, n = 64, 32, 16, 40
    slots = np.arange(n)
    cache = filled(rng, 3, 1, dim, group, page, "Bf16", slots)
    scales = np.ldexp(rng.uniform(1, 2, (n, 1, 2)), rng.integers(-8 - spread // 2, -7 + spread // 2, (n, 1, 2))).astype(np.float16).astype(np.float64)
    zeros = rng.integers(0, 16, scales.shape)
    q = ref.rounded(rng.normal(size=(n, 2, dim)), "Bf16")
    args = (np.arange(3, dtype=np.int32)[None], np.array([0, n], np.int32), np.array([n], np.int32))
    with_value_scales(cache, slots, scales, zeros)
    want, _, mass, _, reach = ref.attend(q, cache, *args)
    fifteen = ref.attend(q, of_scales(cache, slots, scales), *args)[0]
    scales[25, 0, 0] = bad
    with_value_scales(cache, slots, scales, zeros)
    ex = executor("lower_cache4_attention", dtype="Bf16", heads=2, kv_heads=1, head_dim=dim, group=group, page=page)
    out = dev(np.zeros(q.size, np.uint16))
    run(ex, dev(ref.stored(q, "Bf16")), dev(cache.bytes), *(dev(a) for a in args), out, dev(np.zeros(16, np.uint8)), n, 1, 3, 3,
        2 * dim, dim, 2 * dim, dim, 0, 0)
    got = ref.loaded(out.download(np.uint16, q.size), "Bf16").reshape(q.shape)
    hit = np.zeros(q.shape, bool)
    hit[25:, :, :group] = True
    assert not np.isfinite(got[hit]).any()
    assert (np.abs(got - want) <= tolerance(want, mass, fifteen, reach, n, dim, "Bf16"))[~hit].all()


@pytest.mark.parametrize("code, zero", [(0, 15), (15, 0), (15, 7)])
@pytest.mark.parametrize("dtype, heads, dim, group, rows", [("F16", 16, 64, 64, 1), ("Bf16", 2, 64, 32, 20), ("F16", 2, 128, 32, 70),
                                                            ("Bf16", 4, 128, 128, 90)])
def test_faint_keys_beside_one_whose_value_is_zero(hip_device, dtype, heads, dim, group, rows, code, zero):
    """A key that takes all but 2^-13 of the weight and whose value is 0: the output is the others'.  Products of theirs, of a
    code or a zero point with 2^-18.2 of the largest weight, are among the smallest that a step's sums hold."""
    n, page, scale = 32, 16, 0.25
    cache = ref.Cache(2, 1, dim, group, page)
    slots = np.arange(n)
    for s in slots:
        cache.put(s, 0, np.where((np.arange(dim) == 3) & (s > 0), -1.0, 0.0), False)
        for d in range(dim):
            at, shift = cache.code_at(s % page, d, True)
            cache.bytes[s // page, 0, at] |= np.uint8((8 if s == 0 else code) << shift)
    zeros = np.full((n, 1, dim // group), zero)
    zeros[0] = 8
    with_value_scales(cache, slots, np.full(zeros.shape, scale), zeros)
    q = np.zeros((rows, heads, dim))
    q[..., 3] = ref.rounded(np.float32(18.2 * np.log(2) * np.sqrt(dim)), dtype)
    args = (np.arange(2, dtype=np.int32)[None], np.array([0, rows], np.int32), np.array([n], np.int32))
    want, _, mass, _, reach = ref.attend(q, cache, *args, causal=False)
    ex = executor("lower_cache4_attention", dtype=dtype, heads=heads, kv_heads=1, head_dim=dim, group=group, page=page, causal=False)
    out = dev(np.zeros(q.size, np.uint16))
    run(ex, dev(ref.stored(q, dtype)), dev(cache.bytes), *(dev(a) for a in args), out, dev(np.zeros(16, np.uint8)), rows, 1, 2, 2,
        heads * dim, dim, heads * dim, dim, 0, 0)
    got = ref.loaded(out.download(np.uint16, q.size), dtype).reshape(q.shape)
    # As tolerance() has them: the roundings of p and p s and the scores', and f32 sums of at most (8 + 31 x 15 x 2^-18) p s.
    # A product of a code is held to 2^-16 (odd elements 2^-20) of the step's largest p s, one of a zero point to 2^-21.
    score = reach[..., None] * (30.0 / 7.0) * (dim + 4) * 2.0 ** -23
    off = mass * (2 * 2.0 ** -11 + 2 * score + (n + 8) * 2.0 ** -23) + 2 * 8.1 * scale * (n + 8) * 2.0 ** -23
    off += (n - 1) * scale * (np.where(np.arange(dim) % 2 == 0, 2.0 ** -16, 2.0 ** -20) * (code > 0) + 2.0 ** -21 * (zero > 0))
    off += (np.abs(want) + off) * ref.HALF_STEP[dtype] + (2.0 ** -25 if dtype == "F16" else 0.0)
    print("largest error / tolerance %.3g" % (np.abs(got - want) / off).max(), np.abs(want).max(), flush=True)
    assert (np.abs(got - want) <= off).all()
