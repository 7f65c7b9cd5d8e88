"""Linear layers of several networks over one batch sorted by network, with gradients: training's counterpart of `PackedNetworks` /
`PolicyPlan`, which evaluate every (row range, network) tile of a rollout step.  Thin torch front-end of the C ABI
(include/overcooked_ops.h)."""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import native
from .engine import _raw_stream
from .update_ops import _refuse_tangents

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _args(x, weight, offsets, bias):
    if not x.is_cuda or x.dtype not in _TYPES or x.dim() != 2:
        raise ValueError("x must be a float32, bfloat16 or float16 CUDA tensor [rows, in_features]")
    rows, k = x.shape
    if weight.dim() != 3 or weight.dtype != x.dtype or weight.device != x.device or not weight.is_contiguous() or weight.shape[2] != k or 0 in weight.shape or max(weight.shape) >= 2 ** 31:
        raise ValueError(f"weight must be a contiguous {x.dtype} tensor [groups, out_features, {k}] on {x.device}")
    groups, n = weight.shape[:2]
    if bias is not None and (tuple(bias.shape) != (groups, n) or bias.dtype != x.dtype or bias.device != x.device or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous {x.dtype} tensor [{groups}, {n}] on {x.device}")
    if offsets.dtype not in (torch.int32, torch.int64) or offsets.device != x.device or tuple(offsets.shape) != (groups + 1,) or not offsets.is_contiguous():
        raise ValueError(f"offsets must be a contiguous int32 or int64 tensor [{groups + 1}] on {x.device}")
    stride = x.stride(0) if rows > 1 else k
    if rows and ((k > 1 and x.stride(1) != 1) or stride < k):
        raise ValueError("x needs a last dimension of stride 1 and rows that do not overlap (call .contiguous())")
    a = native.OcGroupedLinearArgs()
    a.d_x, a.d_weight, a.d_offsets = x.data_ptr(), weight.data_ptr(), offsets.data_ptr()
    a.d_bias = None if bias is None else bias.data_ptr()
    a.rows, a.x_stride, a.groups, a.in_features, a.out_features = rows, stride, groups, k, n
    a.type, a.offsets64 = _TYPES[x.dtype], int(offsets.dtype == torch.int64)
    return a


def _workspace(a, backward, device):
    """What the C ABI asks for, a fresh one for every call; None if nothing."""
    size = native.lib().oc_grouped_linear_workspace_bytes(ctypes.byref(a), backward)
    return torch.empty(size, dtype=torch.uint8, device=device) if size > 0 else None


def _forward(x, weight, offsets, bias):
    a = _args(x, weight, offsets, bias)
    y = torch.empty((x.shape[0], weight.shape[1]), dtype=x.dtype, device=x.device)
    a.d_y = y.data_ptr()
    workspace = _workspace(a, 0, x.device)
    native.check(native.lib().oc_grouped_linear(ctypes.byref(a), workspace if workspace is None else workspace.data_ptr(), _raw_stream(x.device.index)))
    return y


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, bias):
        y = _forward(x, weight, offsets, bias)
        ctx.save_for_backward(x, weight, offsets)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        # looked at again: hooks on saved tensors (checkpointing, keeping them on the host) may hand back others
        x, weight, offsets = ctx.saved_tensors
        want_x, want_w, _, want_b = ctx.needs_input_grad
        a = _args(x, weight, offsets, None)
        dy = dy.contiguous()
        new = lambda *shape: torch.empty(shape, dtype=x.dtype, device=x.device)
        dx, dw, db = new(*x.shape) if want_x else None, new(*weight.shape) if want_w else None, new(*weight.shape[:2]) if want_b else None
        a.d_dy = dy.data_ptr()
        a.d_dx, a.d_dweight, a.d_dbias = (None if t is None else t.data_ptr() for t in (dx, dw, db))
        workspace = _workspace(a, 1, x.device)
        native.check(native.lib().oc_grouped_linear_backward(ctypes.byref(a), workspace if workspace is None else workspace.data_ptr(),
                                                             _raw_stream(x.device.index)))
        return dx, dw, None, db


def grouped_linear(x, weight, offsets, bias=None):
    """y[r] = x[r] @ weight[g].T + bias[g] for the rows offsets[g] <= r < offsets[g + 1] of network g, in one launch for all networks;
    differentiable in x, weight and bias.  Rows in front of offsets[0] and behind offsets[-1] belong to no network: their result and their
    gradient are 0.

    x f32 / bf16 / f16 [rows, in_features] (rows may be a slice of wider ones); weight [groups, out_features, in_features] and bias
    [groups, out_features] of the same type; offsets int32 / int64 [groups + 1] on the device, not decreasing and within [0, rows] --
    they are read there, nothing is synchronised; a network may have no rows.  Sums are kept in f32 and rounded once; results do not
    depend on timing.  -> y [rows, out_features]

    The segments of `pairing_segments` are such groups: the critics of all pairings (`segment_critics`) learn in one pass."""
    _refuse_tangents("grouped_linear", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GroupedLinear.apply(x, weight, offsets, bias)
    return _forward(x, weight, offsets, bias)
