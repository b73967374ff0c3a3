"""The rotary and 4-bit cache forms on the GPU against their numpy reference: values, masks, borders, refusals."""
import ctypes as C

import numpy as np
import pytest

import unpopped_amd as u
from tests import cache4_reference as ref
from unpopped_amd import _lib

pytestmark = pytest.mark.gpu
B = u.HipBackend()
_execs: dict = {}


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


# ---------------------------------------------------------------------------------------
# Position tables
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("rot, first, count, how", [
    (128, 0, 1, {}), (2, 0, 513, {}), (6, -40, 100, dict(base=500.0)),
    (64, 0, 777, dict(scaling="linear", factor=4.0)), (128, (1 << 22) + 3, 300, dict(base=1e6)),
    (80, 130000, 257, dict(scaling="ramp", factor=8.0, original=8192, amplitude=1.25)),
    (96, 5, 64, dict(scaling="ramp", factor=32.0, low=1.0, high=32.0, original=4096)),
])
def test_position_table(hip_device, rot, first, count, how):
    ex = executor("lower_rope_table", rot=rot, **how)
    want = ref.table(rot, first, count, **how)
    out = dev(np.full(count * rot + 4, 7, np.float32))
    run(ex, out, first, count)
    got = out.download(np.float32, count * rot + 4)
    assert (got[-4:] == 7).all()
    # Rounded once; the frequency's logarithm (up to 14) and exponential, and the product, each 2^-52 of the angle.
    angle = np.abs((first + np.arange(count))[:, None] * ref.frequencies(rot, **{k: v for k, v in how.items() if k != "amplitude"}))
    tol = how.get("amplitude", 1.0) * (2.0 ** -24 + angle[..., None] * 64 * 2.0 ** -52 + 2.0 ** -50)
    assert (np.abs(got[:-4].reshape(count, rot // 2, 2) - want) <= tol).all()


def test_position_table_refuses(hip_device):
    ex = executor("lower_rope_table", rot=64)
    out = dev(np.zeros(64, np.float32))
    invalid(ex, out, 0)
    invalid(ex, 0, 0, 1)
    invalid(ex, out, 0, -1)
    invalid(ex, out, 1 << 53, 1)
    invalid(ex, out, 0, (1 << 52) + 1)
    invalid(ex, out.at(4), 0, 1)
    ex.launch(out, 0, 0)  # nothing to do


# ---------------------------------------------------------------------------------------
# Rotation
# ---------------------------------------------------------------------------------------
def rope_case(dtype, tokens, heads, dim, rot, layout, index, inverse, pad=(0, 0), in_place=False, seed=0, first=0):
    rng = np.random.default_rng(seed)
    x_head, out_head = dim + pad[0], dim + pad[1]
    x_token, out_token = heads * x_head + pad[0], heads * out_head + 3 * pad[1]
    if in_place:
        out_head, out_token = x_head, x_token
    x = ref.rounded(rng.normal(size=tokens * x_token + 16), dtype)
    rows = 50
    pos = rng.integers(first, first + rows, tokens).astype(ref.INDEX[index])
    tab = ref.table(rot, first, rows).astype(np.float32)
    off = pos.copy()
    if tokens > 3:
        off[1], off[2] = first - 1, first + rows  # outside the table: skipped
    ex = executor("lower_rope", dtype=dtype, head_dim=dim, rot=rot, layout=layout, index_dtype=index, inverse=inverse)
    xb, fill = dev(ref.stored(x, dtype)), 9.0
    ob = xb if in_place else dev(ref.stored(np.full(tokens * out_token + 16, fill), dtype))
    run(ex, xb, dev(off), dev(tab), ob, tokens, heads, x_token, x_head, out_token, out_head, first, rows)
    got = ref.loaded(ob.download(ref.stored(np.zeros(1), dtype).dtype, tokens * out_token + 16), dtype)
    want = x.copy() if in_place else np.full(tokens * out_token + 16, fill)
    tol = np.zeros(want.shape)
    at_x = np.arange(tokens)[:, None, None] * x_token + np.arange(heads)[None, :, None] * x_head + np.arange(dim)
    at_o = np.arange(tokens)[:, None, None] * out_token + np.arange(heads)[None, :, None] * out_head + np.arange(dim)
    cs = tab.astype(np.float64)[np.clip(off - first, 0, rows - 1)]
    y = ref.rotate(x[at_x], cs, rot, layout, inverse)
    # One product rounded to 32 bits (at most |x|), the sum to 32 bits, then to the type.
    i0, i1 = ref.pairs_of(rot, layout)
    size = np.zeros(y.shape)
    size[..., i0] = size[..., i1] = np.abs(x[at_x][..., i0]) + np.abs(x[at_x][..., i1])
    t = size * 2.0 ** -24 * 2
    t = t + (np.abs(y) + t) * ref.HALF_STEP[dtype]
    t[..., rot:] = 0
    keep = (off >= first) & (off < first + rows)
    want[at_o[keep]] = y[keep]
    tol[at_o[keep]] = t[keep]
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype, tokens, heads, dim, rot, layout, index, inverse, pad", [
    ("Bf16", 1, 1, 128, 128, "halves", "I32", False, (0, 0)),
    ("Bf16", 37, 5, 128, 64, "pairs", "I64", True, (0, 0)),
    ("F16", 300, 7, 64, 64, "halves", "I32", True, (8, 16)),
    ("F16", 13, 3, 256, 64, "pairs", "I32", False, (1, 0)),     # strides of no whole vectors
    ("F32", 33, 2, 80, 40, "halves", "I64", False, (4, 8)),
    ("F32", 6, 9, 96, 96, "pairs", "I32", True, (0, 0)),
    ("Bf16", 5, 4, 80, 20, "halves", "I32", False, (0, 0)),     # a part that is no whole vector
    ("F32", 4, 3, 7, 6, "pairs", "I32", False, (0, 2)),
    ("Bf16", 4097, 2, 32, 16, "halves", "I32", False, (0, 0)),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_rotation(hip_device, dtype, tokens, heads, dim, rot, layout, index, inverse, pad, in_place):
    rope_case(dtype, tokens, heads, dim, rot, layout, index, inverse, pad, in_place, seed=tokens, first=-7 if heads == 2 else 3)


def test_rotation_and_inverse_are_transposes(hip_device):
    """The inverse is the gradient: <R x, g> = <x, R' g>, and it agrees with differences of the sum."""
    rng = np.random.default_rng(5)
    t, h, d, rot = 9, 2, 64, 32
    x, g = (rng.normal(size=(t, h, d)).astype(np.float32) for _ in range(2))
    pos, tab = rng.integers(0, 99, t).astype(np.int32), ref.table(rot, 0, 99).astype(np.float32)

    def turn(a, inverse):
        out = dev(np.zeros(a.size, np.float32))
        run(executor("lower_rope", dtype="F32", head_dim=d, rot=rot, layout="pairs", inverse=inverse), dev(a), dev(pos),
            dev(tab), out, t, h, h * d, d, h * d, d, 0, 99)
        return out.download(np.float32, a.size).reshape(t, h, d).astype(np.float64)

    back = turn(g, True)
    # Each output is two products and a sum in 32 bits: 2^-23 of the absolute sums.
    bound = 2.0 ** -22 * (np.abs(x.astype(np.float64)).sum() * np.abs(g).max() * 2)
    assert abs((turn(x, False) * g).sum() - (x * back).sum()) <= bound
    for at in ((0, 0, 0), (3, 1, 31), (8, 0, 40)):
        step = np.zeros(x.shape, np.float32)
        step[at] = 0.5
        lo, hi = (turn(x + s * step, False) for s in (-1, 1))
        # The rotation is linear; each side is rounded to 32 bits, as is x + step.
        slack = 2.0 ** -22 * (np.abs(hi[at[:2]]) * np.abs(g[at[:2]])).sum() * 4 + 2.0 ** -22 * 4
        assert abs(((hi - lo) * g).sum() - back[at]) <= slack


def test_rotation_refuses(hip_device):
    ex = executor("lower_rope", dtype="Bf16", head_dim=64, rot=64, layout="halves", index_dtype="I32", inverse=False)
    x, o, p, t = dev(np.zeros(4096, np.uint16)), dev(np.zeros(4096, np.uint16)), dev(np.zeros(8, np.int32)), dev(np.zeros(640, np.float32))
    good = [x, p, t, o, 4, 2, 128, 64, 128, 64, 0, 10]
    run(ex, *good)
    for at, bad in ((0, 0), (3, 0), (4, -1), (5, -1), (5, 65537), (6, -128), (9, 32), (8, 64), (8, 0), (11, -1), (10, 1 << 53),
                    (6, 1 << 60), (8, 1 << 60)):
        args = list(good)
        args[at] = bad
        invalid(ex, *args)
    invalid(ex, x.at(1), *good[1:])
    invalid(ex, x, p, t.at(8), *good[3:])
    invalid(ex, x, p, t, x, 4, 2, 128, 64, 256, 64, 0, 10)  # in place with other strides
    invalid(ex, *good[:-1])
    for nothing in ((4, 0), (5, 0), (11, 0)):
        args = list(good)
        args[nothing[0]] = nothing[1]
        ex.launch(*args)
    with pytest.raises(u.UnpError) as e:
        ex.launch_views([(x, (4, 2, 64), None, 0)] * 4, [0] * 8)
    assert e.value.kind == "InvalidArgument"


# ---------------------------------------------------------------------------------------
# Append and read
# ---------------------------------------------------------------------------------------
def strided(rng, tokens, heads, dim, pad, dtype, scale=1.0):
    head = dim + pad
    token = heads * head + 2 * pad
    flat = ref.rounded(rng.normal(size=tokens * token + 8) * scale, dtype)
    at = np.arange(tokens)[:, None, None] * token + np.arange(heads)[None, :, None] * head + np.arange(dim)
    return flat, at, token, head


@pytest.mark.parametrize("dtype, tokens, heads, dim, group, page, rot, layout, index, pad", [
    ("Bf16", 1, 1, 128, 128, 16, 128, "halves", "I32", 0),
    ("Bf16", 40, 3, 128, 64, 16, 64, "pairs", "I64", 0),
    ("F16", 23, 2, 96, 32, 32, 32, "halves", "I32", 8),
    ("F16", 17, 5, 96, 96, 64, 96, "pairs", "I32", 0),
    ("Bf16", 9, 2, 160, 160, 256, 0, "halves", "I64", 3),        # strides of no whole vectors
    ("F16", 30, 1, 256, 128, 128, 112, "halves", "I32", 0),
    ("Bf16", 12, 4, 32, 32, 16, 16, "pairs", "I32", 1),
    ("Bf16", 5, 2, 192, 64, 32, 192, "halves", "I32", 0),
])
def test_append_and_read(hip_device, dtype, tokens, heads, dim, group, page, rot, layout, index, pad):
    rng = np.random.default_rng(tokens)
    k, at_k, k_token, k_head = strided(rng, tokens, heads, dim, pad, dtype)
    v, at_v, v_token, v_head = strided(rng, tokens, heads, dim, 0, dtype, 0.01)
    # Groups without a range, of one sign, at a tie, and at the edge of f16's smallest scales.
    v[at_v[0, 0, :32]] = 0.0
    k[at_k[-1, -1]] = np.abs(k[at_k[-1, -1]]) + 2.0
    if tokens > 4:
        v[at_v[2, 0]] = ref.rounded(np.arange(dim) % 31 * 0.5 - 7.5, dtype)
        v[at_v[3, 0]] = ref.rounded(v[at_v[3, 0]] * 2.0 ** -14, dtype)
    k, v = (ref.loaded(ref.stored(a, dtype), dtype) for a in (k, v))  # what the device is given
    pages = -(-2 * tokens // page) + 1
    slots = rng.permutation(pages * page)[:tokens].astype(ref.INDEX[index])
    pos = rng.integers(100, 164, tokens).astype(ref.INDEX[index])
    tab = ref.table(max(rot, 2), 100, 64).astype(np.float32)
    gone = np.zeros(tokens, bool)
    if tokens > 6:
        slots[4], slots[5] = -1, pages * page
        gone[4:6] = True
        if rot:
            pos[6], gone[6] = 99, True
    want = ref.Cache(pages, heads, dim, group, page, fill=0xA5)
    kk = k[at_k]
    if rot:
        kk = ref.rounded(ref.rotate(kk, tab.astype(np.float64)[np.clip(pos - 100, 0, 63)], rot, layout), dtype)
    for t in range(tokens):
        for h in range(heads if not gone[t] else 0):
            want.put(int(slots[t]), h, kk[t, h], False)
            want.put(int(slots[t]), h, v[at_v][t, h], True)
    form = dict(dtype=dtype, kv_heads=heads, head_dim=dim, group=group, page=page, index_dtype=index)
    cache = dev(np.full(want.bytes.size, 0xA5, np.uint8))
    kb, vb, sb = dev(ref.stored(k, dtype)), dev(ref.stored(v, dtype)), dev(slots)
    more, rows = ([dev(pos), dev(tab)], [100, 64]) if rot else ([], [])
    run(executor("lower_cache4_append", **form, rot=rot, layout=layout), kb, vb, sb, cache, *more, tokens, pages, k_token,
        k_head, v_token, v_head, *rows)
    got = cache.download(np.uint8, want.bytes.size).reshape(want.bytes.shape)
    wrong = np.argwhere(got != want.bytes)
    assert not len(wrong), [(w.tolist(), int(got[tuple(w)]), int(want.bytes[tuple(w)])) for w in wrong[:8]]
    # Read back: the values rounded once, zeros for a slot outside the cache, nothing between the heads.
    ko, vo = (dev(np.full(k.size, 0x3333, np.uint16)) for _ in range(2))
    run(executor("lower_cache4_read", **form), sb, cache, ko, vo, tokens, pages, k_token, k_head, v_token, v_head)
    for out, at, value in ((ko, at_k, False), (vo, at_v, True)):
        raw = out.download(np.uint16, k.size)
        expect = np.full(k.size, 0x3333, np.uint16)
        for t in range(tokens):
            inside = 0 <= slots[t] < pages * page
            expect[at[t]] = ref.stored(want.get(int(slots[t]), value), dtype) if inside else 0
        assert np.array_equal(raw, expect)


def test_append_of_values_that_are_no_numbers(hip_device):
    """A group with a NaN, an infinity or a range past f16 reads as NaN; its neighbours keep their values."""
    dim, group = 128, 32
    y = np.tile(np.linspace(-1, 1, dim), (4, 1))
    y[0, 5], y[1, 40], y[2, 127], y[3, 64] = np.nan, np.inf, -np.inf, 3e6
    y = ref.rounded(y, "Bf16")
    form = dict(dtype="Bf16", kv_heads=1, head_dim=dim, group=group, page=16)
    cache, slots = dev(np.zeros(16 * (dim + 32), np.uint8)), dev(np.arange(4, dtype=np.int32))
    yb, ko, vo = dev(ref.stored(y, "Bf16")), dev(np.zeros(4 * dim, np.uint16)), dev(np.zeros(4 * dim, np.uint16))
    run(executor("lower_cache4_append", **form, rot=0), yb, yb, slots, cache, 4, 1, dim, dim, dim, dim)
    run(executor("lower_cache4_read", **form), slots, cache, ko, vo, 4, 1, dim, dim, dim, dim)
    for out in (ko, vo):
        got = ref.loaded(out.download(np.uint16, 4 * dim), "Bf16").reshape(4, 4, group)
        bad = np.zeros((4, 4), bool)
        bad[0, 0] = bad[1, 1] = bad[2, 3] = bad[3, 2] = True
        assert np.array_equal(np.isnan(got).all(-1), bad) and np.isfinite(got[~bad]).all()


def test_append_and_read_refuse(hip_device):
    form = dict(dtype="Bf16", kv_heads=2, head_dim=64, group=64, page=16)
    k, cache, slots = dev(np.zeros(1024, np.uint16)), dev(np.zeros(2 * 2 * 16 * 72, np.uint8)), dev(np.full(4, -1, np.int32))
    pos, tab = dev(np.zeros(4, np.int32)), dev(np.zeros(640, np.float32))
    ex = executor("lower_cache4_append", **form, rot=64)
    good = [k, k, slots, cache, pos, tab, 4, 2, 128, 64, 128, 64, 0, 10]
    run(ex, *good)
    for at, bad in ((0, 0), (1, 0), (2, 0), (3, 0), (4, 0), (5, 0), (6, -1), (7, -1), (7, 1 << 31), (8, -1), (11, -64),
                    (12, 1 << 60), (13, -1), (8, 1 << 60)):
        args = list(good)
        args[at] = bad
        invalid(ex, *args)
    invalid(ex, *good[:3], cache.at(4), *good[4:])
    invalid(ex, *good[:5], tab.at(4), *good[6:])
    invalid(ex, *good[:2], slots.at(2), *good[3:])
    invalid(ex, *good[:-2])
    for at in (6, 7, 13):
        args = list(good)
        args[at] = 0
        ex.launch(*args)
    rd = executor("lower_cache4_read", **form)
    out = dev(np.zeros(1024, np.uint16))
    good = [slots, cache, k, out, 4, 2, 128, 64, 128, 64]
    run(rd, *good)
    for at, bad in ((0, 0), (1, 0), (2, 0), (3, 0), (4, -1), (5, -1), (6, 64), (7, 32), (8, 0), (9, -1)):
        args = list(good)
        args[at] = bad
        invalid(rd, *args)


# ---------------------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------------------
def filled(rng, pages, heads, dim, group, page, dtype, used, live=None):
    """A cache whose named slots hold values and whose other bytes are NaN scales and stray codes."""
    c = ref.Cache(pages, heads, dim, group, page, fill=0xFF)
    for s in used:
        for h in range(heads):
            for value in (False, True):
                c.put(int(s), h, ref.rounded(rng.normal(size=dim), dtype), value)
    return c


def attention_case(dtype, heads, kv, dim, group, page, rows, lengths, causal=True, window=0, scale=None, lse=True, pad=0,
                   width=None, workspace=True, seed=0, q_scale=1.0, before=0, behind=3, bad=()):
    """One launch against the reference; `rows` and `lengths` per sequence, `bad` (sequence, place) page entries."""
    rng = np.random.default_rng(seed)
    batch = len(rows)
    need = [-(-n // page) for n in lengths]
    width = max(need + [1]) + 1 if width is None else width
    pages = sum(need) + 2
    order = rng.permutation(pages)
    table = np.full((batch, width), -1, np.int32)
    used = []
    for b in range(batch):
        mine = order[sum(need[:b]):sum(need[:b + 1])][:width]
        table[b, :len(mine)] = mine
        used += [int(mine[j // page]) * page + j % page for j in range(min(lengths[b], len(mine) * page))]
    for b, place in bad:
        table[b, place] = pages + 5 if (b + place) % 2 else -3
    cache = filled(rng, pages, kv, dim, group, page, dtype, used)
    starts = before + np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    tokens = int(starts[-1]) + behind
    q, at_q, q_token, q_head = strided(rng, tokens, heads, dim, pad, dtype, q_scale)
    o, at_o, o_token, o_head = strided(rng, tokens, heads, dim, 2 * pad, dtype)
    want, want_lse, mass, top, reach = ref.attend(q[at_q], cache, table, starts, np.array(lengths), causal, window, scale)
    form = dict(dtype=dtype, heads=heads, kv_heads=kv, head_dim=dim, group=group, page=page, causal=causal, lse=lse,
                scale=scale or 0.0)
    ex = executor("lower_cache4_attention", **form)
    ob, lb = dev(ref.stored(o, dtype)), dev(np.full(tokens * heads, 77, np.float32))
    size = ex.workspace_bytes(tokens, batch, width, pages) if workspace is True else int(workspace)
    ws = dev(np.full(size + 256, 0xFF, np.uint8))
    args = [dev(ref.stored(q, dtype)), dev(cache.bytes), dev(table), dev(starts), dev(np.array(lengths, np.int32)), ob,
            *([lb] if lse else []), ws, tokens, batch, width, pages, q_token, q_head, o_token, o_head, window, size]
    run(ex, *args)
    raw = ob.download(np.uint16, o.size)
    got = ref.loaded(raw, dtype)
    expect, tol = o.copy(), np.zeros(o.shape)
    there = ~np.isnan(want).any((1, 2))
    tolerance = ref.attention_tolerance(want, mass, top, reach, max(lengths + [1]), dim, dtype)
    expect[at_o[there]], tol[at_o[there]] = want[there], tolerance[there]
    off = np.abs(got - expect)
    wrong = np.argwhere(~(off <= tol)).ravel()
    assert not len(wrong), [(int(i), got[i], expect[i], tol[i]) for i in wrong[:6]]
    if lse:
        got_lse = lb.download(np.float32, tokens * heads).reshape(tokens, heads).astype(np.float64)
        assert (got_lse[~there] == 77).all()
        empty = np.isneginf(want_lse[there])
        assert np.array_equal(np.isneginf(got_lse[there]), empty)
        # The sum's relative error and the scores' (attention_tolerance), and the logarithm rounded to 32 bits.
        keys = max(lengths + [1])
        slack = reach[there] * (30 / 7) * (dim + 4) * 2.0 ** -23 + (keys + 8) * 2.0 ** -23 + np.abs(want_lse[there]) * 2.0 ** -22
        assert (np.abs(got_lse[there] - want_lse[there])[~empty] <= slack[~empty]).all()
    assert (ws.download(np.uint8, size + 256)[size:] == 0xFF).all()
    # The same call again gives the same bits.
    ex.launch(*args)
    u.synchronize()
    assert np.array_equal(ob.download(np.uint16, o.size), raw)


@pytest.mark.parametrize("dim, group, page", [(128, 128, 16), (64, 64, 16), (96, 32, 32), (96, 96, 64), (160, 32, 16),
                                              (192, 64, 256), (256, 128, 32), (32, 32, 128), (256, 256, 16), (128, 32, 64)])
@pytest.mark.parametrize("dtype", ["Bf16", "F16"])
def test_attention_of_single_tokens(hip_device, dim, group, page, dtype):
    attention_case(dtype, 6, 2, dim, group, page, [1, 1, 1, 1], [1, 16, 33, 70], seed=dim + group)


@pytest.mark.parametrize("heads, kv", [(1, 1), (5, 5), (8, 1), (14, 2), (16, 1), (20, 4), (34, 2), (128, 1)])
def test_attention_of_head_groups(hip_device, heads, kv):
    attention_case("Bf16", heads, kv, 64, 64, 16, [1, 3, 1], [40, 21, 5], seed=heads)


@pytest.mark.parametrize("rows, lengths", [
    ([5], [5]), ([17], [17]), ([33], [50]), ([1, 20, 0, 7], [9, 20, 30, 90]), ([64], [64]), ([0, 0], [4, 0]),
    ([2] * 9, [3, 2, 7, 40, 16, 17, 31, 32, 33]), ([130], [131]), ([3], [0]), ([6, 1], [4, 1]),  # rows that see nothing
])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_ragged_rows(hip_device, rows, lengths, causal):
    attention_case("Bf16", 4, 2, 64, 32, 16, rows, lengths, causal=causal, seed=len(rows), before=2, pad=8)


@pytest.mark.parametrize("window", [1, 5, 16, 33, 1000])
def test_attention_in_a_window(hip_device, window):
    attention_case("F16", 4, 2, 96, 96, 16, [1, 40, 3], [70, 45, 2], window=window, seed=window)


@pytest.mark.parametrize("workspace", [True, 0, 5000, 70000])
def test_attention_over_a_long_context(hip_device, workspace):
    """One context that several blocks share, with as much workspace as it asks for, less, and none."""
    attention_case("Bf16", 4, 1, 64, 64, 64, [1], [2500], workspace=workspace, seed=3)


def test_attention_with_strides_of_no_whole_vectors(hip_device):
    attention_case("Bf16", 4, 2, 64, 64, 16, [1, 9], [30, 9], pad=1, seed=8)


def test_attention_without_lse_and_with_a_scale(hip_device):
    attention_case("F16", 4, 2, 128, 64, 16, [1, 9], [30, 9], lse=False, scale=0.3, seed=9)


def test_attention_over_bad_pages_and_short_tables(hip_device):
    """Pages outside the cache and keys past the table count for nothing."""
    attention_case("Bf16", 4, 2, 64, 64, 16, [1, 20, 2], [40, 50, 30], bad=[(0, 1), (1, 0), (1, 3), (2, 0), (2, 1)], seed=4)
    attention_case("Bf16", 4, 2, 64, 64, 16, [1, 20], [40, 50], width=2, seed=5)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-3, 30.0, 1e4])
def test_attention_of_small_and_large_queries(hip_device, q_scale):
    """Flat distributions and ones that a single key takes; the sizes of q pass far out of f16's range."""
    rng = np.random.default_rng(2)
    if q_scale >= 30.0:
        # One key dominates only if its score's error is below the gap: the keys' order is what is checked.
        kv, dim, page = 1, 64, 16
        cache = ref.Cache(3, kv, dim, dim, page, fill=0xFF)
        for s in range(40):
            for value in (False, True):
                cache.put(s, 0, ref.rounded(rng.normal(size=dim), "Bf16"), value)
        q = ref.rounded(rng.normal(size=(1, 2, dim)) * q_scale, "Bf16")
        table, starts = np.arange(3, dtype=np.int32)[None], np.array([0, 1], np.int32)
        want = ref.attend(q, cache, table, starts, np.array([40]))[0]
        k = np.array([cache.get(s, False)[0] for s in range(40)])
        score = np.sort(np.einsum("hd,kd->hk", q[0], k) / 8.0, -1)
        gap = score[:, -1] - score[:, -2]
        ex = executor("lower_cache4_attention", dtype="Bf16", heads=2, kv_heads=1, head_dim=dim, group=dim, page=page)
        ob = dev(np.zeros(2 * dim, np.uint16))
        run(ex, dev(ref.stored(q, "Bf16")), dev(cache.bytes), dev(table), dev(starts), dev(np.array([40], np.int32)), ob,
            dev(np.zeros(16, np.uint8)), 1, 1, 3, 3, 2 * dim, dim, 2 * dim, dim, 0, 0)
        got = ref.loaded(ob.download(np.uint16, 2 * dim), "Bf16").reshape(2, dim)
        err = np.abs(q[0]).sum(-1) * np.abs(k).max() / 8.0 * (30 / 7) * 68 * 2.0 ** -23
        for h in range(2):
            if gap[h] > 2 * err[h] + 20:  # the others weigh less than 40 e^-20
                assert (np.abs(got[h] - want[0, h]) <= np.abs(want[0, h]) * 2.0 ** -8 + 6 * (2.0 ** -10 + 40 * np.exp(-20.0))).all()
        assert np.isfinite(got).all()
    else:
        attention_case("Bf16", 4, 2, 64, 64, 16, [1, 9], [30, 29], q_scale=q_scale, seed=11)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("q_scale", [1e8, 1e20, 1e30, 1e36])
def test_attention_of_queries_beyond_every_exponent(hip_device, rows, q_scale):
    """Scores of which one unit of the last place is more than exp reaches: a row is the value of its highest score."""
    rng = np.random.default_rng(12)
    dim, page, n = 64, 16, 40
    cache = filled(rng, 3, 1, dim, dim, page, "Bf16", range(n))
    q = ref.rounded(rng.normal(size=(rows, 2, dim)) * q_scale, "Bf16")
    table, starts, lengths = np.arange(3, dtype=np.int32)[None], np.array([0, rows], np.int32), np.array([n], np.int32)
    k = np.array([cache.get(s, False)[0] for s in range(n)])
    v = np.array([cache.get(s, True)[0] for s in range(n)])
    score = q.reshape(-1, dim) @ k.T / 8.0
    first = score.argmax(-1)
    gap = np.sort(score, -1)[:, -1] - np.sort(score, -1)[:, -2]
    # attention_tolerance's error of a score; the others weigh nothing where they are e^-200 below.
    err = np.abs(q.reshape(-1, dim)).sum(-1) * np.abs(k).max() / 8.0 * (30 / 7) * (dim + 4) * 2.0 ** -23
    clear = gap > 2 * err + 200
    assert clear.any()
    ex = executor("lower_cache4_attention", dtype="Bf16", heads=2, kv_heads=1, head_dim=dim, group=dim, page=page, causal=False)
    ob = dev(np.zeros(rows * 2 * dim, np.uint16))
    run(ex, dev(ref.stored(q, "Bf16")), dev(cache.bytes), dev(table), dev(starts), dev(lengths), ob,
        dev(np.zeros(16, np.uint8)), rows, 1, 3, 3, 2 * dim, dim, 2 * dim, dim, 0, 0)
    got = ref.loaded(ob.download(np.uint16, rows * 2 * dim), "Bf16").reshape(-1, dim)
    want, top = v[first], np.abs(v).max()
    # A value rounded twice to 11 bits and once to its type, and sums of codes and zeros as in attention_tolerance.
    off = np.abs(want) * 2 * 2.0 ** -11 + top * (n * 2.0 ** -35 + 30 / 7 * (n + 8) * 2.0 ** -23)
    off += (np.abs(want) + off) * 2.0 ** -8
    assert (np.abs(got - want) <= off)[clear].all()
    assert (np.abs(got) <= top * 1.01).all()  # of the others: some mean of the values


def test_attention_keeps_what_no_row_sees_out(hip_device):
    """A value that is no number reaches the rows that see its key, and no other row of the same call."""
    rng = np.random.default_rng(6)
    dim, page, n = 64, 16, 40
    cache = filled(rng, 3, 1, dim, 32, page, "Bf16", range(n))
    nan = np.zeros(dim)
    nan[3] = np.nan
    cache.put(25, 0, nan, True)   # a value whose first group is no number
    cache.put(33, 0, nan, False)  # a key
    q = ref.rounded(rng.normal(size=(n, 2, dim)), "Bf16")
    table, starts, lengths = np.arange(3, dtype=np.int32)[None], np.array([0, n], np.int32), np.array([n], np.int32)
    ex = executor("lower_cache4_attention", dtype="Bf16", heads=2, kv_heads=1, head_dim=dim, group=32, page=page)
    ob = dev(np.zeros(n * 2 * dim, np.uint16))
    size = ex.workspace_bytes(n, 1, 3, 3)
    run(ex, dev(ref.stored(q, "Bf16")), dev(cache.bytes), dev(table), dev(starts), dev(lengths), ob,
        dev(np.zeros(size + 16, np.uint8)), n, 1, 3, 3, 2 * dim, dim, 2 * dim, dim, 0, size)
    got = ref.loaded(ob.download(np.uint16, n * 2 * dim), "Bf16").reshape(n, 2, dim)
    assert np.isfinite(got[:25]).all() and np.isfinite(got[25:33, :, 32:]).all()
    assert np.isnan(got[25:, :, :32]).all() and np.isnan(got[33:]).all()
    want, _, mass, top, reach = ref.attend(q[:25], cache, table, np.array([0, 25]), np.array([25]))
    assert (np.abs(got[:25] - want) <= ref.attention_tolerance(want, mass, top, reach, n, dim, "Bf16")).all()


def test_attention_refuses(hip_device):
    form = dict(dtype="Bf16", heads=4, kv_heads=2, head_dim=64, group=64, page=16)
    ex = executor("lower_cache4_attention", **form)
    q, o = dev(np.zeros(2048, np.uint16)), dev(np.zeros(2048, np.uint16))
    cache, table = dev(np.zeros(2 * 2 * 16 * 72, np.uint8)), dev(np.zeros(4, np.int32))
    starts, lengths, ws = dev(np.array([0, 1, 2], np.int32)), dev(np.array([3, 4], np.int32)), dev(np.zeros(64, np.uint8))
    good = [q, cache, table, starts, lengths, o, ws, 2, 2, 2, 2, 256, 64, 256, 64, 0, 64]
    run(ex, *good)
    for at, bad in ((0, 0), (1, 0), (2, 0), (3, 0), (4, 0), (5, 0), (6, 0), (7, -1), (8, -1), (9, -1), (10, -1), (7, 1 << 31),
                    (11, -1), (12, -64), (13, 64), (14, 32), (15, -1), (16, -1), (11, 1 << 60)):
        args = list(good)
        args[at] = bad
        invalid(ex, *args)
    invalid(ex, q, cache.at(8), *good[2:])
    invalid(ex, *good[:6], ws.at(4), *good[7:])
    invalid(ex, q.at(1), *good[1:])
    invalid(ex, *good[:-1])
    full = executor("lower_cache4_attention", **form, causal=False)
    invalid(full, *good[:15], 5, 64)  # a window needs the causal form
    for at in (7, 8):
        args = list(good)
        args[at] = 0
        ex.launch(*args)
    with pytest.raises(u.UnpError) as e:
        ex.workspace_bytes(-1, 1, 1, 1)
    assert e.value.kind == "InvalidArgument"
    with pytest.raises(u.UnpError):
        executor("lower_cache4_read", **{k: v for k, v in form.items() if k != "heads"}).workspace_bytes(1, 1, 1, 1)


def test_attention_over_an_empty_cache_gives_zeros(hip_device):
    form = dict(dtype="F16", heads=2, kv_heads=2, head_dim=32, group=32, page=16)
    ex = executor("lower_cache4_attention", **form)
    o = dev(np.full(3 * 64, 0x3C00, np.uint16))
    ex.launch(dev(np.zeros(192, np.uint16)), dev(np.zeros(16, np.uint8)), dev(np.zeros(4, np.int32)), dev(np.array([0, 2], np.int32)),
              dev(np.array([9], np.int32)), o, dev(np.zeros(16, np.uint8)), 3, 1, 0, 0, 64, 32, 64, 32, 0, 0)
    u.synchronize()
    got = o.download(np.uint16, 192)
    assert (got[:128] == 0).all() and (got[128:] == 0x3C00).all()


# ---------------------------------------------------------------------------------------
# A run of them together, as a serving program has them
# ---------------------------------------------------------------------------------------
def test_prompt_then_tokens(hip_device):
    """A table is made; a prompt's keys and values are appended and attended, then a token at a time: each step's
    outputs are those of the reference over the cache that the reference's own appends made."""
    rng = np.random.default_rng(12)
    dtype, heads, kv, dim, group, page = "Bf16", 4, 2, 64, 64, 16
    batch, steps = 2, [[19, 6], [1, 1], [1, 1]]
    width, pages = 3, 7
    tables = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.int32)
    form = dict(dtype=dtype, kv_heads=kv, head_dim=dim, group=group, page=page)
    make = executor("lower_rope_table", rot=dim, base=10000.0)
    rope = executor("lower_rope", dtype=dtype, head_dim=dim, rot=dim, layout="halves")
    app = executor("lower_cache4_append", **form, rot=dim, layout="halves")
    att = executor("lower_cache4_attention", **form, heads=heads)
    tab = dev(np.zeros(64 * dim, np.float32))
    run(make, tab, 0, 64)
    rows_of = tab.download(np.float32, 64 * dim).reshape(64, dim // 2, 2).astype(np.float64)
    want = ref.Cache(pages, kv, dim, group, page)
    cache = dev(np.zeros(want.bytes.size, np.uint8))
    lengths = np.zeros(batch, np.int32)
    for new in steps:
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        tokens = int(starts[-1])
        pos = np.concatenate([lengths[b] + np.arange(new[b]) for b in range(batch)]).astype(np.int32)
        slots = np.concatenate([tables[b, (lengths[b] + np.arange(new[b])) // page] * page + (lengths[b] + np.arange(new[b])) % page
                                for b in range(batch)]).astype(np.int32)
        lengths = lengths + np.array(new, np.int32)
        row = (heads + 2 * kv) * dim  # a fused projection's row
        x = ref.rounded(rng.normal(size=(tokens, heads + 2 * kv, dim)), dtype)
        xb, pb, sb, st = dev(ref.stored(x, dtype)), dev(pos), dev(slots), dev(starts)
        kb, vb = xb.at(2 * heads * dim), xb.at(2 * (heads + kv) * dim)
        qb, ob = dev(np.zeros(tokens * heads * dim, np.uint16)), dev(np.zeros(tokens * heads * dim, np.uint16))
        run(app, kb, vb, sb, cache, pb, tab, tokens, pages, row, dim, row, dim, 0, 64)
        run(rope, xb, pb, tab, qb, tokens, heads, row, dim, heads * dim, dim, 0, 64)
        size = att.workspace_bytes(tokens, batch, width, pages)
        run(att, qb, cache, dev(tables), st, dev(lengths), ob, dev(np.zeros(size + 16, np.uint8)), tokens, batch, width, pages,
            heads * dim, dim, heads * dim, dim, 0, size)
        kk = ref.rounded(ref.rotate(x[:, heads:heads + kv], rows_of[pos], dim, "halves"), dtype)
        for t in range(tokens):
            for h in range(kv):
                want.put(int(slots[t]), h, kk[t, h], False)
                want.put(int(slots[t]), h, x[t, heads + kv + h], True)
        assert np.array_equal(cache.download(np.uint8, want.bytes.size), want.bytes.ravel())
        q = ref.loaded(qb.download(np.uint16, tokens * heads * dim), dtype).reshape(tokens, heads, dim)
        out, _, mass, top, reach = ref.attend(q, want, tables, starts, lengths)
        got = ref.loaded(ob.download(np.uint16, q.size), dtype).reshape(q.shape)
        assert (np.abs(got - out) <= ref.attention_tolerance(out, mass, top, reach, int(lengths.max()), dim, dtype)).all()


# ---------------------------------------------------------------------------------------
# Splits, streams, graphs and far places
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("heads, rows", [(1, [1]), (6, [1]), (12, [1]), (4, [21]), (5, [2, 1])])
@pytest.mark.parametrize("window", [0, 1500])
def test_attention_splits_of_every_kind_of_block(hip_device, heads, rows, window):
    """Contexts that are split over blocks, for each number of rows a block takes; a window leaves parts without keys."""
    attention_case("F16", heads, 1, 64, 32, 32, rows, [2300, 90][:len(rows)], window=window, seed=heads, lse=heads != 6)


@pytest.mark.parametrize("dtype, heads, kv, dim, group, rows, lengths, entry", [
    ("Bf16", 8, 2, 64, 64, [9, 3, 12], [700, 520, 12], "_some"),     # several tiles of a sequence
    ("F16", 12, 1, 64, 32, [4, 1], [600, 601], "_few"),              # the same, of more heads than columns are shared by
    ("Bf16", 8, 2, 96, 32, [30, 41], [530, 900], "_more"),
    ("F16", 4, 4, 128, 128, [170, 190, 0, 1], [1300, 190, 7, 5], "_more"),
    ("Bf16", 6, 2, 32, 32, [60, 61, 90], [200, 150, 90], "_many"),   # a context that is no longer than its steps
])
@pytest.mark.parametrize("workspace", [True, 0])
def test_attention_of_some_tiles_a_sequence(hip_device, dtype, heads, kv, dim, group, rows, lengths, entry, workspace):
    ex = executor("lower_cache4_attention", dtype=dtype, heads=heads, kv_heads=kv, head_dim=dim, group=group, page=32,
                  causal=True, lse=True, scale=0.0)
    attention_case(dtype, heads, kv, dim, group, 32, rows, lengths, workspace=workspace, seed=21)
    last = ex.last_launch()["entry"]
    assert last.endswith(entry) or last.endswith("_join"), last


@pytest.mark.parametrize("parts", range(1, 12))
def test_attention_of_every_number_of_parts(hip_device, parts):
    """Joins of few parts (several rows a block) and of many, by the workspace that they get."""
    tokens, heads, dim = 2, 3, 96
    size = (parts * tokens * heads * 8 + 15) // 16 * 16 + parts * tokens * heads * dim * 4
    attention_case("F16", heads, 1, dim, 96, 16, [1], [1700], behind=1, workspace=size, seed=parts)


def test_attention_of_many_sequences(hip_device):
    """More sequences than one look of a wave finds, some without rows and some without keys."""
    rng = np.random.default_rng(3)
    rows = rng.integers(0, 3, 150).tolist()
    lengths = [int(n) if i % 9 else 0 for i, n in enumerate(rng.integers(1, 40, 150))]
    attention_case("Bf16", 2, 1, 32, 32, 16, rows, [max(n, r) for n, r in zip(lengths, rows)], seed=1)


def small_step(dtype="Bf16", heads=4, kv=2, dim=64, page=16, rows=(1, 1, 1), lengths=(700, 33, 1200), seed=0):
    """A decode step's buffers, its reference and a launch: (launch(stream, workspace), out, want, tolerance)."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lengths]
    width, pages, tokens = max(need), sum(need), sum(rows)
    order = rng.permutation(pages)
    table = np.full((len(rows), width), -1, np.int32)
    for b in range(len(rows)):
        table[b, :need[b]] = order[sum(need[:b]):sum(need[:b + 1])]
    cache = ref.Cache(pages, kv, dim, dim, page)
    # Random codes and finite scales of every size.
    cache.bytes[:] = rng.integers(0, 256, cache.bytes.shape, np.uint8)
    words = cache.bytes[..., page * dim:].copy().view(np.uint16).reshape(pages, kv, -1, 2)
    words[..., 0] = (rng.random(words.shape[:-1]) * 0.3 + 0.02).astype(np.float16).view(np.uint16)
    words[..., 1] = rng.integers(0, 16, words.shape[:-1])
    cache.bytes[..., page * dim:] = words.reshape(pages, kv, -1).view(np.uint8)
    q = ref.rounded(rng.normal(size=(tokens, heads, dim)), dtype)
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    want, _, mass, top, reach = ref.attend(q, cache, table, starts, np.array(lengths))
    # With any codes a step may be as large as the largest |v| and |k| themselves, not a seventh of them.
    tol = ref.attention_tolerance(want, mass, 7 * top, 7 * reach, max(lengths), dim, dtype)
    ex = executor("lower_cache4_attention", dtype=dtype, heads=heads, kv_heads=kv, head_dim=dim, group=dim, page=page)
    out = dev(np.zeros(q.size, np.uint16))
    held = [dev(ref.stored(q, dtype)), dev(cache.bytes), dev(table), dev(starts), dev(np.array(lengths, np.int32))]
    size = ex.workspace_bytes(tokens, len(rows), width, pages)
    strides = (heads * dim, dim, heads * dim, dim)

    def launch(stream, ws, how="launch"):
        getattr(ex, how)(*held, out, ws, tokens, len(rows), width, pages, *strides, 0, size, stream=stream)

    return launch, out, want, tol, size, q.shape, ex


def close(out, want, tol, dtype="Bf16"):
    got = ref.loaded(out.download(np.uint16, want.size), dtype).reshape(want.shape)
    return bool((np.abs(got - want) <= tol).all())


def test_streams_graphs_and_workspaces(hip_device):
    """A step captured into a graph and replayed between eager work, two graphs with workspaces of their own replayed
    at once on two streams, and the launches that take no allocation or are timed: each gives the eager bits."""
    L = _lib.lib()
    steps = [small_step(seed=s, lengths=n) for s, n in ((0, (700, 33, 1200)), (1, (2048, 1, 3000)))]
    raw = []
    assert steps[1][4] > 0  # one of the two is split over blocks and joined
    for launch, out, want, tol, size, shape, ex in steps:
        size = max(size, 16)
        launch(0, u.DeviceBuffer(size))
        u.synchronize()
        assert ex.last_launch()["shared"] == (size > 16) == ex.last_launch()["entry"].endswith("_join")
        assert close(out, want, tol)
        raw.append(out.download(np.uint16, want.size))
        launch(0, u.DeviceBuffer(size), "launch_static")
        a, b = u.Event(), u.Event()
        ex.set_timing(a, b)
        launch(0, u.DeviceBuffer(size))
        u.synchronize()
        assert 0 < a.elapsed_ms(b) < 1000
        ex.set_timing(None, None)
        assert np.array_equal(out.download(np.uint16, want.size), raw[-1])
    workspaces, streams, graphs = [u.DeviceBuffer(max(s[4], 16)) for s in steps], [], []
    for (launch, *_), ws in zip(steps, workspaces):
        st, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
        assert L.hipStreamCreate(C.byref(st)) == 0
        assert L.hipStreamBeginCapture(st, 0) == 0
        launch(st.value, ws)
        assert L.hipStreamEndCapture(st, C.byref(graph)) == 0
        assert L.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        streams.append(st)
        graphs.append((graph, exe))
    spare = u.DeviceBuffer(max(steps[0][4], 16))
    for turn in range(4):
        for (_, out, *_), ws in zip(steps, workspaces):
            out.fill(0)
            ws.fill(0xFF)
        u.synchronize()
        for _ in range(3):
            for (_, exe), st in zip(graphs, streams):
                assert L.hipGraphLaunch(exe, st) == 0
        u.synchronize()
        for (_, out, want, *_), r in zip(steps, raw):
            assert np.array_equal(out.download(np.uint16, want.size), r), turn
        steps[0][0](0, spare)  # eager work between the replays
        u.synchronize()
    # The same two eagerly, on their streams at once.
    for (launch, out, *_), ws, st in zip(steps, workspaces, streams):
        out.fill(0)
        u.synchronize()
        launch(st.value, ws)
    u.synchronize()
    for (_, out, want, *_), r in zip(steps, raw):
        assert np.array_equal(out.download(np.uint16, want.size), r)
    for graph, exe in graphs:
        assert L.hipGraphExecDestroy(exe) == 0 and L.hipGraphDestroy(graph) == 0
    for st in streams:
        assert L.hipStreamDestroy(st) == 0


def test_pages_past_four_gigabytes(hip_device):
    """Slots and pages whose byte offsets need more than 32 bits: appended, read back and attended."""
    form = dict(dtype="Bf16", kv_heads=2, head_dim=64, group=64, page=16)
    each = u.cache4_page_bytes(**form)
    pages = (5 << 30) // each
    cache = u.DeviceBuffer(pages * each)
    rng = np.random.default_rng(0)
    y = ref.rounded(rng.normal(size=(20, 2, 64)), "Bf16")
    far = [pages - 1, pages // 2]
    slots = np.array([far[t // 16] * 16 + t % 16 for t in range(20)], np.int64)
    sb, yb, ko, vo = dev(slots), dev(ref.stored(y, "Bf16")), dev(np.zeros(y.size, np.uint16)), dev(np.zeros(y.size, np.uint16))
    run(executor("lower_cache4_append", **form, rot=0, index_dtype="I64"), yb, yb, sb, cache, 20, pages, 128, 64, 128, 64)
    run(executor("lower_cache4_read", **form, index_dtype="I64"), sb, cache, ko, vo, 20, pages, 128, 64, 128, 64)
    want = ref.Cache(2, 2, 64, 64, 16)
    for t in range(20):
        for h in range(2):
            want.put(t, h, y[t, h], False)
            want.put(t, h, y[t, h], True)
    expect = np.array([want.get(t, True) for t in range(20)])
    for out in (ko, vo):
        assert np.array_equal(out.download(np.uint16, y.size), ref.stored(expect, "Bf16").ravel())
    q = ref.rounded(rng.normal(size=(1, 4, 64)), "Bf16")
    out = dev(np.zeros(256, np.uint16))
    ex = executor("lower_cache4_attention", **form, heads=4)
    run(ex, dev(ref.stored(q, "Bf16")), cache, dev(np.array([far], np.int32)), dev(np.array([0, 1], np.int32)),
        dev(np.array([20], np.int32)), out, dev(np.zeros(16, np.uint8)), 1, 1, 2, pages, 256, 64, 256, 64, 0, 0)
    o, _, mass, top, reach = ref.attend(q, want, np.array([[0, 1]]), [0, 1], [20])
    assert close(out, o, ref.attention_tolerance(o, mass, top, reach, 20, 64, "Bf16"))


def test_indexes_of_any_value(hip_device):
    """Positions, slots, lengths and starts at the ends of their types leave what they do not name as it was."""
    ends = np.array([np.iinfo(np.int64).min, np.iinfo(np.int64).max, -1, 0, 1 << 40, -(1 << 40)], np.int64)
    x = ref.rounded(np.random.default_rng(0).normal(size=(6, 1, 64)), "Bf16")
    xb, out, tab = dev(ref.stored(x, "Bf16")), dev(np.full(6 * 64, 0x3333, np.uint16)), dev(ref.table(64, 0, 8).astype(np.float32))
    for first, row in ((0, 3), (np.iinfo(np.int64).max >> 11, -1)):  # position 0 only, or none
        out.upload(np.full(6 * 64, 0x3333, np.uint16))
        run(executor("lower_rope", dtype="Bf16", head_dim=64, index_dtype="I64"), xb, dev(ends), tab, out, 6, 1, 64, 64, 64, 64,
            int(first), 8)
        got = out.download(np.uint16, 6 * 64).reshape(6, 64)
        for t in range(6):
            assert np.array_equal(got[t], ref.stored(x[t, 0], "Bf16") if t == row else np.full(64, 0x3333, np.uint16))
    form = dict(dtype="Bf16", kv_heads=1, head_dim=64, group=64, page=16)
    size = u.cache4_page_bytes(**form)
    cache = dev(np.full(2 * size, 0x77, np.uint8))
    slots = np.array([ends[0], ends[1], -1, 3, 32, 31], np.int64)
    run(executor("lower_cache4_append", **form, rot=64, index_dtype="I64"), xb, xb, dev(slots), cache, dev(ends), tab, 6, 2, 64,
        64, 64, 64, 0, 8)
    got = cache.download(np.uint8, 2 * size)
    want = ref.Cache(2, 1, 64, 64, 16, fill=0x77)
    for value in (False, True):
        want.put(3, 0, x[3, 0], value)
    assert np.array_equal(got, want.bytes.ravel())
    # Lengths below zero and past the table, starts past the rows: the first sequence's row is the reference's, the
    # others see all of the table's keys or none, and rows behind the last are left.
    q = ref.rounded(np.random.default_rng(1).normal(size=(5, 2, 64)), "Bf16")
    rng = np.random.default_rng(2)
    full = filled(rng, 2, 1, 64, 64, 16, "Bf16", range(32))
    table = np.array([[0, 1]] * 4, np.int32)
    starts, lengths = np.array([0, 1, 2, 3, 4], np.int32), np.array([20, -7, np.iinfo(np.int32).max, np.iinfo(np.int32).min], np.int32)
    ob = dev(np.full(5 * 128, 0x3333, np.uint16))
    ex = executor("lower_cache4_attention", **form, heads=2)
    args = [dev(ref.stored(q, "Bf16")), dev(full.bytes), dev(table), None, None, ob, dev(np.zeros(16, np.uint8)), 5, 4, 2, 2, 128, 64,
            128, 64, 0, 0]
    args[3], args[4] = dev(starts), dev(lengths)
    run(ex, *args)
    got = ob.download(np.uint16, 5 * 128).reshape(5, 2, 64)
    o, _, mass, top, reach = ref.attend(q, full, table, starts, [20, 0, 33, 0])
    tol = ref.attention_tolerance(o, mass, top, reach, 32, 64, "Bf16")
    for t in (0, 2):
        assert (np.abs(ref.loaded(got[t], "Bf16") - o[t]) <= tol[t]).all()
    assert (got[[1, 3]] == 0).all() and (got[4] == 0x3333).all()
    for wrong in ([0, 9, 9, 9, 9], [5, 3, 1, 0, 0], [-4, -2, 7, 2, 1 << 30], [np.iinfo(np.int32).min] * 2 + [np.iinfo(np.int32).max] * 3):
        args[3] = dev(np.array(wrong, np.int32))
        run(ex, *args)  # every access stays inside: the rows are those of 0 .. 4 only


def test_attention_limits_refuse(hip_device):
    ex = executor("lower_cache4_attention", dtype="Bf16", heads=4, kv_heads=2, head_dim=64, group=64, page=16)
    for shape in ((1, 1, (1 << 26) + 1, 1), ((1 << 29) + 1, 1, 1, 1), (1, 1 << 31, 1, 1)):
        with pytest.raises(u.UnpError) as e:
            ex.workspace_bytes(*shape)
        assert e.value.kind == "InvalidArgument"
    assert ex.workspace_bytes(0, 5, 5, 5) == 0 and ex.workspace_bytes(5, 0, 5, 5) == 0


def test_attention_of_more_blocks_than_a_launch_has_refuses(hip_device):
    """Shapes whose blocks would pass 2^32 lanes: refused from the scalars, before anything is read."""
    ex = executor("lower_cache4_attention", dtype="Bf16", heads=4, kv_heads=2, head_dim=64, group=64, page=16)
    some = dev(np.zeros(64, np.uint8))
    for tokens, batch in ((1 << 23, 1 << 23), (1 << 29, 1)):
        invalid(ex, some, some, some, some, some, some, some, tokens, batch, 1, 1, 256, 64, 256, 64, 0, 0)


@pytest.mark.parametrize("dtype, bits", [("Bf16", 8), ("F16", 11)])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_append_rounds_a_rotated_key_to_32_bits_and_then_to_its_type(hip_device, dtype, bits, layout):
    """Sums within 2^-30 and 2^-20 of a tie of the type, each the largest of its group: the scale shows how it was rounded."""
    dim, rests = 32, [2.0 ** -30, -2.0 ** -30, 2.0 ** -20, -2.0 ** -20]
    x = np.zeros((len(rests), 1, dim))
    x[..., 0] = x[..., dim // 2 if layout == "halves" else 1] = 1.0
    tab = np.zeros((len(rests), dim // 2, 2), np.float32)
    tab[:, 0, 0], tab[:, 0, 1] = 1.0 + 2.0 ** -bits, np.negative(rests)
    # Beside the tie by less than half of a 32-bit step: the tie, and so the even one of its neighbours, 1.
    top = np.array([1.0, 1.0, 1.0 + 2.0 ** (1 - bits), 1.0])
    form = dict(dtype=dtype, kv_heads=1, head_dim=dim, page=16)
    cache, some = dev(np.zeros(u.cache4_page_bytes(**form), np.uint8)), dev(np.arange(len(rests), dtype=np.int32))
    run(executor("lower_cache4_append", **form, rot=dim, layout=layout), dev(ref.stored(x, dtype)), dev(ref.stored(x, dtype)), some,
        cache, some, dev(tab), len(rests), 1, dim, dim, dim, dim, 0, len(rests))
    words = cache.download(np.uint8, u.cache4_page_bytes(**form))[16 * dim:16 * dim + 4 * len(rests)].view(np.uint16)[::2]
    # The other element of the pair is c less s, of a smaller rest: the same largest but for the two sums' signs of it.
    other = ref.rounded(1.0 + 2.0 ** -bits - np.array(rests), dtype)
    want = (np.maximum(top, other).astype(np.float32) / np.float32(15)).astype(np.float16)
    assert np.array_equal(words.view(np.float16), want)


@pytest.mark.parametrize("dtype, heads, kv, dim, group, rows, lengths, entry", [
    ("Bf16", 16, 1, 128, 128, [1, 1], [600, 33], "_lse_few"),
    ("Bf16", 16, 1, 128, 128, [3, 2], [600, 530], "_cached_few"),    # more heads than columns are shared by
    ("F16", 8, 2, 192, 64, [5, 11], [540, 20], "_more"),             # more words than a wave holds twice
    ("Bf16", 12, 4, 64, 64, [2, 3], [900, 600], "_some"),
])
@pytest.mark.parametrize("workspace", [True, 0])
def test_attention_reads_what_several_blocks_read_through_the_caches(hip_device, dtype, heads, kv, dim, group, rows, lengths, entry,
                                                                     workspace):
    ex = executor("lower_cache4_attention", dtype=dtype, heads=heads, kv_heads=kv, head_dim=dim, group=group, page=32,
                  causal=True, lse=True, scale=0.0)
    attention_case(dtype, heads, kv, dim, group, 32, rows, lengths, workspace=workspace, seed=22, behind=0)
    last = ex.last_launch()["entry"]
    assert last.endswith(entry) or (workspace and last.endswith("_join")), last


def entry_case(entry, dtype, heads, kv, dim, group, rows, lengths, page=16, lse=False, joined=None, **how):
    """A launch without a workspace, whose entry it is, and then with one (`joined`: whether that splits the contexts)."""
    for workspace in (0, True):
        attention_case(dtype, heads, kv, dim, group, page, rows, lengths, lse=lse, workspace=workspace, behind=0, seed=dim + group + heads,
                       **how)
        last = executor("lower_cache4_attention", dtype=dtype, heads=heads, kv_heads=kv, head_dim=dim, group=group, page=page,
                        causal=True, lse=lse, scale=0.0).last_launch()["entry"]
        assert last.endswith(entry) or (workspace and last.endswith("_join")), last
        assert joined is None or not workspace or last.endswith("_join") == joined


DECODE = [(128, 128, 16), (128, 64, 64), (64, 64, 32)]


@pytest.mark.parametrize("group_heads", [1, 2, 4, 5, 7, 8, 9, 16])
@pytest.mark.parametrize("dim, group, page", DECODE)
def test_attention_of_a_decode_step(hip_device, group_heads, dim, group, page):
    """One token a sequence: the columns shared by four, two and one sets of keys, some of them past the last."""
    entry_case("_few", ["Bf16", "F16"][group_heads % 2], 2 * group_heads, 2, dim, group, [1, 1, 1], [1, 131, 70], page=page, joined=False)


@pytest.mark.parametrize("group_heads", [1, 4, 8, 16])
@pytest.mark.parametrize("dim, group, page", DECODE)
def test_attention_of_a_decode_step_over_a_split_context(hip_device, group_heads, dim, group, page):
    entry_case("_few", ["Bf16", "F16"][group_heads % 2], 2 * group_heads, 2, dim, group, [1, 1], [1400, 33], page=page, width=2400 // page,
               joined=True)


SHAPES = [("Bf16", d, g) for d, g in ((64, 32), (96, 96), (96, 32), (128, 128), (128, 64), (128, 32), (160, 160), (192, 192), (192, 64),
                                      (224, 224), (224, 32), (256, 256), (256, 128), (256, 32))]
SHAPES += [("F16", d, g) for d, g in ((64, 32), (128, 128), (128, 64), (160, 32), (192, 192), (256, 64))]


@pytest.mark.parametrize("dtype, dim, group", SHAPES)
def test_attention_of_prompts(hip_device, dtype, dim, group):
    """Waves of rows of their own: several blocks of a sequence, the last of them in part, and a sequence of one."""
    entry_case("_many", dtype, 6, 2, dim, group, [101, 1, 37], [101, 20, 60], page=32)


@pytest.mark.parametrize("dtype, dim, group", SHAPES)
def test_attention_of_a_few_dozen_rows(hip_device, dtype, dim, group):
    """Waves that share the keys of a tile or two, of the last row tile in part."""
    entry_case("_more", dtype, 6, 2, dim, group, [31, 26], [530, 61], page=32)
