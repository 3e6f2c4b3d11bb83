"""Every form of the projection kernels, given through the verification hook, so
that a change of the rule that picks them takes no test away. Small products:
each form accepts any size."""

import pytest
import torch

from layer_checks import check_linear
from linear_abi import FP8, form_of, launch_form, linear_args
from oracle import layer_ref

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
ACTS = ["none", "silu", "sigmoid", "relu", "gelu_tanh"]
WIDTHS = [64, 128, 192, 256]
TYPES = [(BF16, BF16), (FP16, FP16), (FP8, BF16), (FP8, FP16)]   # operands, output
NARROW, PAIR = 0, 1


def strided(T, N, dtype, offset=0, extra=0):
    """[T, N] zeros whose rows are `extra` elements apart, the first `offset` elements in."""
    buf = torch.zeros(T * (N + extra) + offset, dtype=dtype, device="cuda")
    return buf[offset:].view(T, N + extra)[:, :N]


def operands(T, K, N, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, w = torch.randn(T, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda") * K ** -0.5
    if dtype != FP8:
        return x.to(dtype), w.to(dtype), {}
    sx, sw = x.abs().amax(dim=1) / 448, w.abs().amax(dim=1) / 448
    return (x / sx[:, None]).to(FP8), (w / sw[:, None]).to(FP8), {"x_scale": sx, "weight_scale": sw}


def check(form, x, w, scales, out, act="none", bias=None, residual=None, in_place=False):
    """One launch into `out` (over `residual` with in_place) against the definition; out's gaps stay as they were."""
    want = layer_ref.linear(x, w, bias, residual, act=act, **scales)
    into = residual if in_place else out
    assert launch_form(linear_args(x, w, into, bias, residual, act=ACTS.index(act), **scales), form) == 0
    check_linear(into, want, into.dtype, x.shape[1])
    return into


def epilogue(T, N, dtype, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(N, generator=g, device="cuda"), torch.randn(T, N, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("N", [520, 515])          # rows that TMA stores, and rows off 16 bytes
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("types", TYPES)
def test_pair_epilogues(types, width, N):
    """Each activation with every choice of bias and residual."""
    T, K = 300, 144
    x, w, s = operands(T, K, N, types[0], width)
    bias, residual = epilogue(T, N, types[1])
    for act in ACTS:
        for b in (None, bias):
            for r in (None, residual):
                check((PAIR, width, 1), x, w, s, strided(T, N, types[1]), act, b, r)


# Output and residual: by TMA, or off 16 bytes by their offset, by their stride.
LAYOUTS = [((0, 0), (0, 0)), ((0, 0), (1, 7)), ((3, 5), (0, 8)), ((1, 7), (1, 7)), ((0, 3), (5, 0)), ((8, 8), (0, 0))]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("form", [(PAIR, 64, 1), (PAIR, 128, 1), (PAIR, 192, 1), (PAIR, 256, 1), (NARROW, 16, 2),
                                  (NARROW, 16, 1), (NARROW, 32, 2), (NARROW, 64, 1)])
@pytest.mark.parametrize("types", [(BF16, BF16), (FP8, FP16)])
def test_rows_on_and_off_boundaries(types, form, layout):
    """Output and residual rows that each start on 16 bytes or do not, with gaps that no store touches; and
    the output written over a residual of either kind."""
    T, K, N = 290, 160, 264
    x, w, s = operands(T, K, N, types[0], 3)
    bias, values = epilogue(T, N, types[1])
    (out_offset, out_extra), (res_offset, res_extra) = layout
    out, residual = strided(T, N, types[1], out_offset, out_extra), strided(T, N, types[1], res_offset, res_extra)
    residual.copy_(values)
    check(form, x, w, s, out, "silu", bias, residual)
    gaps = torch.ones(out._base.numel(), dtype=torch.bool, device="cuda")
    gaps.as_strided(out.shape, out.stride(), out.storage_offset()).fill_(False)
    assert (out._base[gaps] == 0).all()
    over = check(form, x, w, s, None, "silu", bias, residual, in_place=True)
    assert torch.equal(over, out)


@pytest.mark.parametrize("T", [1, 130, 300])
@pytest.mark.parametrize("N", [1, 3, 14, 65, 177, 260, 515])
@pytest.mark.parametrize("form", [(PAIR, 64, 1), (PAIR, 128, 1), (PAIR, 192, 1), (PAIR, 256, 1), (NARROW, 16, 2), (NARROW, 64, 1)])
def test_odd_widths_in_aligned_rows(form, N, T):
    """Rows that start on 16 bytes and end off them: a column slice of a wider output, whose other columns stay."""
    K, extra = 128, -N % 8 + 16
    x, w, s = operands(T, K, N, BF16, N)
    bias, values = epilogue(T, N, BF16)
    wide = torch.full((T, 8 + N + extra), 7.0, dtype=BF16, device="cuda")
    out, residual = wide[:, 8:8 + N], strided(T, N, BF16, 8, extra + 8)
    residual.copy_(values)
    for r in (None, residual):
        wide.fill_(7.0)
        check(form, x, w, s, out, "silu", bias, r)
        assert (wide[:, :8] == 7).all() and (wide[:, 8 + N:] == 7).all()


@pytest.mark.parametrize("N", [1, 7, 32, 33, 63, 64, 65, 96, 128, 160, 191, 255, 257, 300])
@pytest.mark.parametrize("width", WIDTHS)
def test_pair_widths_and_tails(width, N):
    """Every output width around the tiles' and boxes' edges, one token upwards."""
    for T in (1, 31, 128, 129, 257):
        x, w, s = operands(T, 96, N, BF16, N)
        bias, residual = epilogue(T, N, BF16)
        check((PAIR, width, 1), x, w, s, strided(T, N, BF16), "gelu_tanh", bias, residual)


@pytest.mark.parametrize("K", [1, 8, 63, 64, 65, 128, 320, 321, 1001, 4096])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("form", [(PAIR, 64, 1), (PAIR, 192, 1), (PAIR, 256, 1), (NARROW, 64, 1)])
def test_input_widths(form, types, K):
    """One block of K to many more than the stages, in place and copied to aligned rows."""
    T, N = 200, 136
    x, w, s = operands(T, K, N, types[0], K)
    check(form, x, w, s, strided(T, N, types[1]))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("types", TYPES)
def test_pair_many_tiles(types, width):
    """Several tiles a pair: both accumulators, all stages and boxes used again, strips that do not fill."""
    T, N = 6000, 1032
    for K in (64, 544):
        x, w, s = operands(T, K, N, types[0], width)
        bias, residual = epilogue(T, N, types[1])
        for r, out in ((residual, strided(T, N, types[1])), (residual, strided(T, N, types[1], 1)), (None, strided(T, N, types[1]))):
            check((PAIR, width, 1), x, w, s, out, "sigmoid", bias, r)


@pytest.mark.parametrize("tile,splits", [(16, 1), (16, 2), (16, 3), (16, 5), (16, 8), (32, 1), (32, 2), (32, 3), (32, 6), (64, 1), (64, 2),
                                         (64, 3), (64, 8)])
@pytest.mark.parametrize("types", TYPES)
def test_narrow(types, tile, splits):
    """Token counts around each tile, split K, every activation."""
    K, N = 1120, 203
    for i, T in enumerate((1, tile - 1, tile, tile + 1, 2 * tile + 5)):
        x, w, s = operands(T, K, N, types[0], T)
        bias, residual = epilogue(T, N, types[1])
        check((NARROW, tile, splits), x, w, s, strided(T, N, types[1]), ACTS[i], bias, residual)
        check((NARROW, tile, splits), x, w, s, strided(T, N, types[1], 0, 5), ACTS[i])


@pytest.mark.parametrize("form", [(PAIR, 64, 1), (PAIR, 256, 1), (NARROW, 16, 2), (NARROW, 64, 2)])
@pytest.mark.parametrize("stride", [(1 << 30) + 8, (1 << 30) + 7])
def test_output_rows_beyond_32_bits(form, stride):
    """Row strides of output and residual whose offsets pass 2^31 elements, on and off 16-byte boundaries."""
    T, K, N = 3, 128, 72
    x, w, s = operands(T, K, N, BF16, 9)
    _, values = epilogue(T, N, BF16)
    out, residual = (torch.empty(2 * stride + N, dtype=BF16, device="cuda").as_strided((T, N), (stride, 1)) for _ in range(2))
    residual.copy_(values)
    check(form, x, w, s, out, residual=residual)


@pytest.mark.parametrize("form", [(PAIR, 64, 1), (PAIR, 128, 1), (PAIR, 256, 1), (NARROW, 32, 2), (NARROW, 64, 2)])
@pytest.mark.parametrize("N", [160, 157])
def test_non_finite_values_stay_in_their_rows(form, N):
    """NaN and infinities in one token or one output touch no other."""
    x, w, _ = operands(300, 192, N, BF16, 6)
    clean, got = (strided(300, N, BF16) for _ in range(2))
    assert launch_form(linear_args(x, w, clean), form) == 0
    x[3, 7], x[5, 0], w[11, 3] = float("nan"), float("inf"), float("inf")
    assert launch_form(linear_args(x, w, got), form) == 0
    touched = torch.zeros(300, N, dtype=torch.bool, device="cuda")
    touched[[3, 5], :], touched[:, 11] = True, True
    assert torch.equal(got[~touched], clean[~touched])
    assert got[3].isnan().all() and not got[5, :11].isfinite().any() and not got[:, 11].isfinite().any()


def test_rule_reaches_each_form_through_the_op():
    """Products whose own form is each kernel and width, through the public op."""
    from sgl_glm53_ascend_ops import ops

    sms = torch.cuda.get_device_properties(0).multi_processor_count
    seen = set()
    for T, K, N, dtype in ((1, 2048, 256, BF16), (200, 512, 2048, FP16), (64, 256, 12576, BF16), (1300, 4096, 1024, FP16),
                           (300, 4096, 4096, FP8), (256, 4096, 12576, FP8), (8256, 128, 1032, BF16), (2100, 64, 64 * 75, FP8),
                           (20000, 512, 64, BF16)):
        x, w, s = operands(T, K, N, dtype, 11)
        bias, residual = epilogue(T, N, BF16 if dtype == FP8 else dtype)
        seen.add(form_of(T, K, N, {BF16: 0, FP16: 1, FP8: 2}[dtype], sms)[:2])
        got = ops.linear(x, w, bias=bias, residual=residual, activation="silu", **s)
        check_linear(got, layer_ref.linear(x, w, bias, residual, act="silu", **s), got.dtype, K)
    if sms == 148:
        assert seen == {(NARROW, t) for t in (16, 32, 64)} | {(PAIR, w) for w in WIDTHS}
