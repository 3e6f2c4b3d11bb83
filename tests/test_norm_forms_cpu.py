"""The norms' verification hooks: which kernel a launch takes, by sizes and
alignments alone (no pointer is read, no kernel launched)."""

import ctypes

import pytest

from test_abi_cpu import test_struct_layout_matches_header as struct_layout_matches_header
from test_norm_forms_gpu import DIRECT, FORMS, GATED, RING, SHIFTED, form


@pytest.fixture(scope="module")
def abi():
    from sgl_glm53_ascend_ops import abi as _abi
    return _abi


def test_struct_layout(abi, tmp_path):
    struct_layout_matches_header(abi, tmp_path, "KdaNormForm")


def rmsnorm_args(abi, T, N, offset=0, extra=0, res_offset=0, res_extra=0, residual=True, fp8=False):
    res = 512 + 2 * res_offset if residual else None
    return abi.KdaNormArgs(x=512 + 2 * offset, x_row_stride=N + extra, residual=res, residual_row_stride=N + res_extra,
                           residual_out=res, residual_out_row_stride=N + res_extra, weight=512, out=512, out_row_stride=N,
                           scale=512 if fp8 else None, num_tokens=T, hidden=N)


def test_lists_of_the_gpu_tests_take_the_forms_they_name(abi):
    seen = set()
    for T, N, offset, extra, res_offset, res_extra, kind in FORMS:
        for fp8 in (False, True):
            a = rmsnorm_args(abi, T, N, offset, extra, res_offset, res_extra, True, fp8)
            assert form(abi, abi.lib().kda_rmsnorm_form, a) == kind, (T, N)
        seen.add(kind)
    assert {(DIRECT, r, u) for r in range(3) for u in (1, 2, 4)} | {(RING, 0, u) for u in (1, 2, 4)} < seen
    seen = set()
    for T, H, D, gap, offset, kind in GATED:
        a = abi.KdaGatedNormArgs(o=512, gate=512 + 2 * offset, gate_row_stride=H * D, weight=512, out=512,
                                 out_row_stride=H * D, num_tokens=T, num_heads=H, head_dim=D, activation=abi.KDA_ACT_SILU)
        a.o_stride[0], a.o_stride[1] = H * (D + gap), D + gap
        assert form(abi, abi.lib().kda_gated_rmsnorm_form, a) == kind, (T, H, D)
        seen.add(kind)
    assert {(DIRECT, r, u) for r in (0, 2) for u in (1, 2, 4)} | {(RING, 0, u) for u in (1, 2, 4)} < seen


def test_rule(abi):
    """The sizes whose both sides the rules' comments measure."""
    kind = lambda T, N: form(abi, abi.lib().kda_rmsnorm_form, rmsnorm_args(abi, T, N))  # noqa: E731
    assert kind(256, 4096) == (DIRECT, 0, 1) and kind(1000, 4096) == (DIRECT, 0, 4)
    assert kind(8256, 4096) == (RING, 0, 4) and kind(33494, 4096) == (RING, 0, 4)
    assert kind(33494, 1001)[:2] == (DIRECT, SHIFTED)


def test_form_hooks_refuse(abi):
    lib = abi.lib()
    f = abi.KdaNormForm()
    a = rmsnorm_args(abi, 4, 64)
    assert lib.kda_rmsnorm_form(None, 148, ctypes.byref(f)) == abi.KDA_ERR_INVALID_ARGUMENT
    assert lib.kda_rmsnorm_form(ctypes.byref(a), 148, None) == abi.KDA_ERR_INVALID_ARGUMENT
    assert lib.kda_rmsnorm_form(ctypes.byref(a), -1, ctypes.byref(f)) == abi.KDA_ERR_INVALID_ARGUMENT
    a.num_tokens = 0
    assert lib.kda_rmsnorm_form(ctypes.byref(a), 148, ctypes.byref(f)) == abi.KDA_ERR_INVALID_ARGUMENT
    g = abi.KdaGatedNormArgs(num_tokens=2, num_heads=2, head_dim=96)
    assert lib.kda_gated_rmsnorm_form(ctypes.byref(g), 148, ctypes.byref(f)) == abi.KDA_ERR_UNSUPPORTED
