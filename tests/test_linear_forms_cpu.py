"""The rule that picks a projection's kernel, and the refusals of its
verification hooks. No kernel is launched."""

import ctypes
import random

import pytest

from linear_abi import form_of
from test_abi_cpu import test_struct_layout_matches_header as struct_layout_matches_header


@pytest.fixture(scope="module")
def abi():
    from sgl_glm53_ascend_ops import abi as _abi
    return _abi


def test_struct_layout(abi, tmp_path):
    struct_layout_matches_header(abi, tmp_path, "KdaLinearForm")


@pytest.mark.parametrize("T,K,N,dtype,form", [
    (1, 4096, 4096, 2, (0, 16, 8)), (1, 4096, 12576, 0, (0, 16, 2)), (64, 4096, 4096, 0, (0, 16, 2)),
    (64, 4096, 12576, 0, (0, 64, 2)), (128, 4096, 4096, 0, (0, 32, 2)), (256, 4096, 4096, 0, (0, 64, 2)),
    (256, 4096, 12576, 2, (1, 192, 1)), (512, 4096, 4096, 0, (1, 128, 1)), (8256, 4096, 12576, 0, (1, 256, 1)),
    (77, 1001, 515, 1, (0, 16, 4)), (1, 64, 160000, 0, (0, 16, 1)), (5, 7, 3, 0, (0, 16, 1)),
])
def test_the_rule_at_sizes_that_its_comment_measures(T, K, N, dtype, form):
    assert form_of(T, K, N, dtype) == form


def test_every_choice_is_a_form(abi):
    """Over the whole range of sizes and SM counts: a known tile, K split into no empty part, clusters of at most 8."""
    rng = random.Random(0)
    seen = set()
    for _ in range(20000):
        T, K, N = (round(2 ** rng.uniform(0, top)) for top in (17, 14, 18))
        dtype = rng.randrange(3)
        kernel, tile, splits = form_of(T, K, N, dtype, rng.choice((148, 132, 74, 1)))
        blocks = -(-K * (1 if dtype == 2 else 2) // 128)
        if kernel == abi.KDA_LINEAR_PAIR:
            assert splits == 1 and tile in (64, 128, 192, 256) and T > 64
        else:
            # More tokens a tile never come with 4 splits or more: only 16 have a form that sends its sums.
            assert splits < 4 or tile == 16
            assert tile in (16, 32, 64) and 1 <= splits <= min(8, blocks) and -(-T // tile) <= 65535
        seen.add((kernel, tile))
    assert seen == {(0, 16), (0, 32), (0, 64), (1, 64), (1, 128), (1, 192), (1, 256)}


def test_form_hooks_refuse(abi):
    lib = abi.lib()
    buf = (ctypes.c_uint8 * 64)()
    at = ctypes.addressof(buf)
    a = abi.KdaLinearArgs(x=at, x_row_stride=128, weight=at, weight_row_stride=128, out=at, out_row_stride=16, num_tokens=4,
                          in_features=128, out_features=16)
    f = abi.KdaLinearForm()
    assert lib.kda_linear_form(None, 148, ctypes.byref(f)) == abi.KDA_ERR_INVALID_ARGUMENT
    assert lib.kda_linear_form(ctypes.byref(a), 148, None) == abi.KDA_ERR_INVALID_ARGUMENT
    assert lib.kda_linear_form(ctypes.byref(a), -1, ctypes.byref(f)) == abi.KDA_ERR_INVALID_ARGUMENT
    launch = lambda *form: lib.kda_linear_launch_form(ctypes.byref(a), None, 0, ctypes.byref(abi.KdaLinearForm(*form)),  # noqa: E731
                                                      None)
    assert lib.kda_linear_launch_form(ctypes.byref(a), None, 0, None, None) == abi.KDA_ERR_INVALID_ARGUMENT
    for form in ((2, 64, 1), (1, 64, 2), (1, 32, 1), (1, 320, 1), (1, 96, 1), (0, 128, 1), (0, 16, 0), (0, 16, 3), (0, 8, 1)):
        assert launch(*form) == abi.KDA_ERR_INVALID_ARGUMENT, form       # (0, 16, 3): K has two blocks
    a.num_tokens = 0
    assert lib.kda_linear_form(ctypes.byref(a), 148, ctypes.byref(f)) == abi.KDA_ERR_INVALID_ARGUMENT
    a.num_tokens = 1 << 24
    assert launch(0, 64, 1) == abi.KDA_ERR_INVALID_ARGUMENT             # more token tiles than a grid's second dimension
