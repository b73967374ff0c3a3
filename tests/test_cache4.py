"""The rotary and 4-bit cache forms without a GPU: what they refuse to lower, the sources' compilation, the record's
size, and the reference that the GPU tests compare with."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

import unpopped_amd as u
from tests import cache4_reference as ref
from unpopped_amd import _lib

B = u.HipBackend()


@pytest.mark.parametrize("kw, kind", [
    (dict(rot=7), "UnsupportedKernel"), (dict(rot=0), "UnsupportedKernel"), (dict(rot=4098), "UnsupportedKernel"),
    (dict(rot=64, base=0.0), "UnsupportedKernel"), (dict(rot=64, base=float("nan")), "UnsupportedKernel"),
    (dict(rot=64, scaling="linear", factor=0.0), "UnsupportedKernel"),
    (dict(rot=64, scaling="ramp", factor=2.0, low=4.0, high=4.0), "UnsupportedKernel"),
    (dict(rot=64, scaling="ramp", factor=2.0, original=0), "UnsupportedKernel"),
    (dict(rot=64, amplitude=float("inf")), "UnsupportedKernel"),
])
def test_a_position_table_refuses(kw, kind):
    with pytest.raises(u.UnpError) as e:
        B.lower_rope_table(**kw)
    assert e.value.kind == kind and e.value.detail


@pytest.mark.parametrize("kw, kind", [
    (dict(dtype="F64", head_dim=64), "UnsupportedDtype"), (dict(dtype="I32", head_dim=64), "UnsupportedDtype"),
    (dict(dtype="F32", head_dim=64, index_dtype="U32"), "UnsupportedDtype"),
    (dict(dtype="F32", head_dim=64, rot=66), "UnsupportedKernel"), (dict(dtype="F32", head_dim=64, rot=3), "UnsupportedKernel"),
    (dict(dtype="F32", head_dim=8192), "UnsupportedKernel"),
])
def test_a_rotation_refuses(kw, kind):
    with pytest.raises(u.UnpError) as e:
        B.lower_rope(**kw)
    assert e.value.kind == kind and e.value.detail


CACHE = dict(dtype="Bf16", kv_heads=4, head_dim=128, group=64, page=16)


@pytest.mark.parametrize("change, kind", [
    (dict(dtype="F32"), "UnsupportedDtype"), (dict(kv_heads=0), "UnsupportedKernel"), (dict(kv_heads=1025), "UnsupportedKernel"),
    (dict(head_dim=80, group=80), "UnsupportedKernel"), (dict(head_dim=288, group=32), "UnsupportedKernel"),
    (dict(group=16), "UnsupportedKernel"), (dict(group=0), "UnsupportedKernel"), (dict(head_dim=96, group=64), "UnsupportedKernel"),
    (dict(page=8), "UnsupportedKernel"), (dict(page=48), "UnsupportedKernel"), (dict(page=512), "UnsupportedKernel"),
])
def test_a_cache_refuses(change, kind):
    form = {**CACHE, **change}
    for call in (lambda: B.lower_cache4_append(**form), lambda: B.lower_cache4_read(**form),
                 lambda: B.lower_cache4_attention(heads=max(1, 2 * form["kv_heads"]), **form),
                 lambda: u.cache4_page_bytes(**form)):
        with pytest.raises(u.UnpError) as e:
            call()
        assert e.value.kind == kind and e.value.detail


@pytest.mark.parametrize("call, kind", [
    (lambda: B.lower_cache4_append(**CACHE, rot=8), "UnsupportedKernel"),
    (lambda: B.lower_cache4_append(**CACHE, rot=144), "UnsupportedKernel"),
    (lambda: B.lower_cache4_append(**CACHE, index_dtype="U32"), "UnsupportedDtype"),
    (lambda: B.lower_cache4_attention(heads=6, **CACHE), "UnsupportedKernel"),
    (lambda: B.lower_cache4_attention(heads=0, **CACHE), "UnsupportedKernel"),
    (lambda: B.lower_cache4_attention(heads=4 * 129, **CACHE), "UnsupportedKernel"),
    (lambda: B.lower_cache4_attention(heads=8, **CACHE, scale=-1.0), "UnsupportedKernel"),
    (lambda: B.lower_cache4_attention(heads=8, **CACHE, scale=float("nan")), "UnsupportedKernel"),
])
def test_a_cache_form_refuses(call, kind):
    with pytest.raises(u.UnpError) as e:
        call()
    assert e.value.kind == kind and e.value.detail


def test_descriptors_out_of_range_and_null():
    """Values that the Python names cannot spell, and null pointers, through the C ABI."""
    L, out, err = _lib.lib(), C.c_void_p(), _lib.Error()
    assert L.unp_hip_lower_rope_table(None, C.byref(out), C.byref(err)) == _lib.INVALID_ARGUMENT
    t = _lib.RopeTable(64, 3, 1e4, 1, 1, 4, 8192, 1)
    assert L.unp_hip_lower_rope_table(C.byref(t), C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_OP
    r = _lib.Rope(2, 64, 64, 2, 9, 0)
    assert L.unp_hip_lower_rope(C.byref(r), C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_OP
    r = _lib.Rope(2, 64, 64, 0, 9, 2)
    assert L.unp_hip_lower_rope(C.byref(r), C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_KERNEL
    c = _lib.Cache4(1, 4, 128, 64, 16, 9)
    assert L.unp_hip_lower_cache4_append(C.byref(c), 0, 5, C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_OP
    assert L.unp_hip_lower_cache4_attention(C.byref(c), None, C.byref(out), C.byref(err)) == _lib.INVALID_ARGUMENT
    a = _lib.Attention(8, 2, 0, 0, 0.0)
    assert L.unp_hip_lower_cache4_attention(C.byref(c), C.byref(a), C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_KERNEL
    assert L.unp_cache4_record_bytes(C.byref(c), None, C.byref(err)) == _lib.INVALID_ARGUMENT
    assert not out.value
    for kind in range(8, 13):  # the forms that come only from a descriptor
        f = B.form("reduction")
        f.kind = kind
        assert L.unp_hip_lower_form(C.byref(f), C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_KERNEL


def test_every_form_compiles_and_states_its_parameters():
    cc = u.HipCompiler()
    forms = [B.lower_rope_table(96, scaling="ramp", factor=8.0),
             B.lower_rope("F32", 80, 40, "pairs", inverse=True), B.lower_rope("Bf16", 70, 6),
             B.lower_cache4_append("F16", 5, 96, 32, rot=32, layout="pairs", index_dtype="I64"),
             B.lower_cache4_append("Bf16", 8, 160, page=256), B.lower_cache4_read("Bf16", 2, 256, 128, page=64),
             B.lower_cache4_attention("Bf16", 32, 8, 128), B.lower_cache4_attention("F16", 15, 3, 96, 32, causal=False, lse=True)]
    for g in forms:
        assert len(cc.compile(g.source, g.name)) > 0
        names = [p["name"] for p in g.interface["params"]]
        kinds = [p["kind"] for p in g.interface["params"]]
        assert len(set(names)) == len(names) and kinds == sorted(kinds)  # buffers, then scalars
        assert g.interface["entries"] and all(e["symbol"] in g.source for e in g.interface["entries"])


@pytest.mark.parametrize("heads, dim, group, page", [(8, 128, 128, 16), (3, 96, 32, 64), (1, 256, 64, 256), (2, 32, 32, 32)])
def test_the_record_has_the_references_size(heads, dim, group, page):
    assert u.cache4_page_bytes("F16", heads, dim, group, page) == heads * ref.Cache(1, heads, dim, group, page).record


@pytest.mark.parametrize("dim, group, page", [(128, 128, 16), (96, 32, 32), (64, 64, 64)])
def test_the_reference_holds_what_it_is_given(dim, group, page):
    """put and get agree, every code of a record has a place of its own, and a step is at most a scale wide."""
    rng = np.random.default_rng(dim)
    c = ref.Cache(2, 2, dim, group, page)
    seen = {c.code_at(t, d, v) for t in range(page) for d in range(dim) for v in (False, True)}
    assert len(seen) == 2 * page * dim and max(at for at, _ in seen) < page * dim
    words = {c.word_at(t, g, v) for t in range(page) for g in range(dim // group) for v in (False, True)}
    assert len(words) == 2 * page * (dim // group) and min(words) == page * dim and max(words) == c.record - 4
    for value in (False, True):
        for slot in (0, page - 1, page + 3):
            y = ref.rounded(rng.normal(size=(2, dim)), "Bf16")
            for h in range(2):
                c.put(slot, h, y[h], value)
            got = c.get(slot, value)
            step = ref.quantise(y, group)[1].astype(np.float64).repeat(group, -1).reshape(2, dim)
            # Half a step for the code, half for the zero point.
            assert (np.abs(got - y) <= 1.0001 * step).all()


def test_a_planted_mistake_in_the_reference_shows():
    """The attention reference's tolerance is far below what a wrong mask or a wrong page does."""
    rng = np.random.default_rng(1)
    c = ref.Cache(4, 1, 64, 64, 16)
    for s in range(64):
        for v in (False, True):
            c.put(s, 0, ref.rounded(rng.normal(size=64), "Bf16"), v)
    q = ref.rounded(rng.normal(size=(3, 2, 64)), "Bf16")
    args = (np.array([[2, 0, 1]]), np.array([0, 3]), np.array([40]))
    out, _, mass, top, reach = ref.attend(q, c, *args)
    tol = ref.attention_tolerance(out, mass, top, reach, 40, 64, "Bf16")
    for wrong in ((args[0], args[1], np.array([41])), (np.array([[2, 1, 0]]), args[1], args[2])):
        other = ref.attend(q, c, *wrong)[0]
        assert (np.abs(other - out) > tol).mean() > 0.5


@pytest.mark.parametrize("owner", [None, 0, object()])
def test_held_memory_is_not_freed(monkeypatch, owner):
    freed = []

    class Lib:
        @staticmethod
        def unp_hip_free(p):
            freed.append(p)

    monkeypatch.setattr(u._lib, "lib", lambda: Lib)
    b = u.DeviceBuffer.held(4096, 64, owner)
    part = b.at(16)
    assert (b.ptr, b.nbytes, part.ptr, part.nbytes) == (4096, 64, 4112, 48)
    b.free()
    del part, b
    assert freed == []


def nearest(x: Fraction, bits: int) -> Fraction:
    """x rounded to `bits` significant bits, ties to even (no range)."""
    step = Fraction(1)
    while abs(x) >= step * 2 ** bits:
        step *= 2
    while abs(x) < step * 2 ** (bits - 1):
        step /= 2
    return Fraction(round(x / step)) * step  # Python rounds a tie to the even number


@pytest.mark.parametrize("dtype, bits", [("Bf16", 8), ("F16", 11)])
@pytest.mark.parametrize("rest, sign", [(2.0 ** -30, 1), (-2.0 ** -30, 1), (2.0 ** -30, -1), (2.0 ** -20, 1)])
def test_a_rotated_key_is_rounded_to_32_bits_and_then_to_its_type(dtype, bits, rest, sign):
    """A sum beside a tie of the type: 2^-30 beside it the 32-bit number is the tie itself, 2^-20 beside it is not."""
    x = np.zeros((1, 1, 32))
    x[0, 0, 0], x[0, 0, 16] = sign, 1.0
    tab = np.zeros((1, 16, 2), np.float32)
    tab[0, 0] = 1.0 + 2.0 ** -bits, -rest * sign
    sum_ = Fraction(float(tab[0, 0, 0])) * sign + Fraction(rest) * sign
    want = nearest(nearest(nearest(sum_, 53), 24), bits)
    assert (want == nearest(sum_, bits)) == (rest != 2.0 ** -30)
    got = ref.rounded(ref.rotate(x, tab.astype(np.float64), 32, "halves"), dtype)
    assert Fraction(float(got[0, 0, 0])) == want
