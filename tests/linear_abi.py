"""Projections through the C entries with their form given
(``kda_linear_launch_form``) or asked for (``kda_linear_form``)."""

import ctypes

import torch

FP8 = torch.float8_e4m3fn


def dtype_code(dtype):
    return {torch.bfloat16: 0, torch.float16: 1, FP8: 2}[dtype]


def linear_args(x, w, out, bias=None, residual=None, x_scale=None, weight_scale=None, act=0):
    """KdaLinearArgs of [T, K] x, [N, K] w and [T, N] out, any row strides."""
    from sgl_glm53_ascend_ops import abi

    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return abi.KdaLinearArgs(
        x=ptr(x), x_row_stride=x.stride(0), weight=ptr(w), weight_row_stride=w.stride(0), x_scale=ptr(x_scale),
        weight_scale=ptr(weight_scale), bias=ptr(bias), residual=ptr(residual),
        residual_row_stride=0 if residual is None else residual.stride(0), out=ptr(out), out_row_stride=out.stride(0),
        num_tokens=x.shape[0], in_features=x.shape[1], out_features=w.shape[0], in_dtype=dtype_code(x.dtype),
        out_dtype=dtype_code(out.dtype), activation=act)


def launch_form(args, form):
    """One launch in `form` = (kernel, tile, splits); returns its code."""
    from sgl_glm53_ascend_ops import abi

    n = abi.lib().kda_linear_workspace_bytes(ctypes.byref(args))
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    rc = abi.lib().kda_linear_launch_form(ctypes.byref(args), ws.data_ptr(), n, ctypes.byref(abi.KdaLinearForm(*form)),
                                          abi.stream_handle())
    torch.cuda.synchronize()
    return rc


def form_of(T, K, N, dtype=0, sms=148):
    """(kernel, tile, splits) that a launch of these sizes takes; no pointer is read."""
    from sgl_glm53_ascend_ops import abi

    scale = 16 if dtype == 2 else None
    a = abi.KdaLinearArgs(x=16, x_row_stride=K, weight=16, weight_row_stride=K, x_scale=scale, weight_scale=scale, out=16,
                          out_row_stride=N, num_tokens=T, in_features=K, out_features=N, in_dtype=dtype,
                          out_dtype=0 if dtype == 2 else dtype)
    f = abi.KdaLinearForm()
    assert abi.lib().kda_linear_form(ctypes.byref(a), sms, ctypes.byref(f)) == abi.KDA_OK
    return f.kernel, f.tile, f.splits
