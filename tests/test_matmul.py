"""The floating point products without a GPU: what they refuse to lower, the sources' compilation, and the reference that the
GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest
import torch

import unpopped_amd as u
from tests import matmul_reference as ref
from unpopped_amd import _lib

B = u.HipBackend()
TORCH = {"Fp8E4M3FN": torch.float8_e4m3fn, "Fp8E5M2": torch.float8_e5m2}


@pytest.mark.parametrize("call, kind", [
    (lambda: B.lower_quant8("F64"), "UnsupportedDtype"), (lambda: B.lower_quant8("I32"), "UnsupportedDtype"),
    (lambda: B.lower_quant8("Bf16", "Fp8E4M3FNUZ"), "UnsupportedDtype"), (lambda: B.lower_quant8("Bf16", "I8"), "UnsupportedDtype"),
    (lambda: B.lower_quant8("Bf16", block_rows=64), "UnsupportedKernel"), (lambda: B.lower_quant8("Bf16", block_rows=0), "UnsupportedKernel"),
    (lambda: B.lower_matmul8(a_kind="Bf16"), "UnsupportedDtype"), (lambda: B.lower_matmul8(b_kind="I8"), "UnsupportedDtype"),
    (lambda: B.lower_matmul8(out="F32"), "UnsupportedDtype"), (lambda: B.lower_matmul8(b_rows=16), "UnsupportedKernel"),
    (lambda: B.lower_grouped_matmul("F32"), "UnsupportedDtype"), (lambda: B.lower_grouped_matmul("Bf16", "F16"), "UnsupportedDtype"),
    (lambda: B.lower_group_rows("U32"), "UnsupportedDtype"),
])
def test_a_form_refuses(call, kind):
    with pytest.raises(u.UnpError) as e:
        call()
    assert e.value.kind == kind and e.value.detail


def test_descriptors_out_of_range_and_null():
    L, out, err = _lib.lib(), C.c_void_p(), _lib.Error()
    calls = [(L.unp_hip_lower_quant8, _lib.Quant8(1, 12, 1, 2), _lib.UNSUPPORTED_KERNEL),
             (L.unp_hip_lower_matmul8, _lib.Matmul8(12, 12, 1, 128, 2), _lib.UNSUPPORTED_KERNEL),
             (L.unp_hip_lower_grouped_matmul, _lib.GroupedMatmul(1, 1, 3), _lib.UNSUPPORTED_OP),
             (L.unp_hip_lower_group_rows, _lib.GroupRows(2), _lib.UNSUPPORTED_DTYPE)]
    for call, descriptor, rc in calls:
        assert call(None, C.byref(out), C.byref(err)) == _lib.INVALID_ARGUMENT
        assert call(C.byref(descriptor), None, C.byref(err)) == _lib.INVALID_ARGUMENT
        assert call(C.byref(descriptor), C.byref(out), C.byref(err)) == rc and err.detail
    assert not out.value
    for kind in range(13, 17):  # the forms that come only from a descriptor
        f = B.form("reduction")
        f.kind = kind
        assert L.unp_hip_lower_form(C.byref(f), C.byref(out), C.byref(err)) == _lib.UNSUPPORTED_KERNEL


@pytest.mark.parametrize("lower", [
    lambda: B.lower_quant8("Bf16"), lambda: B.lower_quant8("F32", "Fp8E5M2", 128, True), lambda: B.lower_quant8("F16", block_rows=128),
    lambda: B.lower_quant8("Bf16", transpose=True), lambda: B.lower_matmul8(), lambda: B.lower_matmul8("Fp8E5M2", "Fp8E4M3FN", "F16", 1, True),
    lambda: B.lower_grouped_matmul("Bf16"), lambda: B.lower_grouped_matmul("F16", "F32", "input"),
    lambda: B.lower_grouped_matmul("Bf16", "F32", "weight"), lambda: B.lower_group_rows(), lambda: B.lower_group_rows("I64"),
])
def test_a_form_compiles_and_states_its_parameters(lower):
    g = lower()
    assert len(u.HipCompiler().compile(g.source, g.name)) > 0
    names = [p["name"] for p in g.interface["params"]]
    kinds = [p["kind"] for p in g.interface["params"]]
    assert len(set(names)) == len(names) and kinds == sorted(kinds)  # buffers, then scalars
    assert g.interface["entries"] and all(e["symbol"] in g.source for e in g.interface["entries"])


# ---------------------------------------------------------------------------------------
# The reference
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["Fp8E4M3FN", "Fp8E5M2"])
def test_the_references_numbers_are_those_of_the_type(kind):
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes.copy()).view(TORCH[kind]).float().numpy()
    assert np.array_equal(ref.decoded(codes, kind), want, equal_nan=True)
    v = np.random.default_rng(0).normal(size=4096) * np.exp2(np.random.default_rng(1).integers(-20, 9, 4096))
    v = np.clip(np.concatenate([v, want[np.isfinite(want)], [0.0, -0.0]]), -ref.LARGEST[kind], ref.LARGEST[kind]).astype(np.float32)
    got = ref.encoded(v, kind)
    assert np.array_equal(got, torch.from_numpy(v).to(TORCH[kind]).view(torch.uint8).numpy())


def test_the_references_quantisation_by_hand():
    x = np.zeros((3, 130))
    x[0, 0], x[0, 1], x[0, 129] = 896.0, 3.0, -1.0
    x[2, 5] = np.nan
    codes, scales = ref.quantised(x, "Fp8E4M3FN", 1, False)
    assert scales.tolist()[0] == [2.0, np.float32(1.0 / 448.0)] and scales.tolist()[1] == [0.0, 0.0]
    assert np.isnan(scales[2, 0]) and scales[2, 1] == 0.0 and (codes[1:] == 0).all()
    assert ref.decoded(codes[0, [0, 1, 129]], "Fp8E4M3FN").tolist() == [448.0, 1.5, -448.0]
    turned, same = ref.quantised(x, "Fp8E4M3FN", 128, True)
    assert turned.shape == (130, 3) and same.shape == (2, 1) and np.isnan(same[0, 0])


def test_the_references_rows_by_hand():
    starts, rows, place = ref.group_rows([1, 0, -1, 1, 5, 0], 2, 3)
    assert starts.tolist() == [0, 2, 4, 4] and rows.tolist() == [0, 2, 0, 1, -1, -1] and place.tolist() == [2, 0, -1, 3, -1, 1]
