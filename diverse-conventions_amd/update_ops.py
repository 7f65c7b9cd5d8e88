"""The update behind a rollout: clipped policy and value losses with their gradients, the global gradient norm with clipping.
Thin torch front-ends of the C ABI (include/overcooked_ops.h), next to `gae_returns` / `normalize_advantages` / `MinibatchSource`.

Every call works on its arguments' GPU and on that device's current stream, allocates its results and workspace from torch's caching
allocator and keeps nothing between calls.  Nothing synchronises with the host but a value normaliser given as an object, which is read back.
"""
import ctypes
import math
from array import array

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import native
from .engine import _raw_stream

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_FORWARD, _FORWARD_GRAD, _BACKWARD = 0, 1, 2

POLICY_STATS = ("policy_loss", "entropy", "kl", "clip_fraction", "ratio")


def _stream(device):
    return _raw_stream(device.index)


_workspace_bytes = {}


def _workspace(size_of, device):
    """A workspace of the size that the C ABI asks for: a fresh one for every call, so that calls on several streams never share it."""
    size = _workspace_bytes.get(size_of)
    if size is None:
        size = _workspace_bytes[size_of] = getattr(native.lib(), size_of)()
    return torch.empty(size, dtype=torch.uint8, device=device)


def _refuse_tangents(what, *tensors):
    """These operators have no forward-mode derivative; read by address, a dual tensor would lose its tangent without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} does not support forward mode automatic differentiation")


def _rows_f32(name, t, n, device):
    if t.dtype != torch.float32 or t.device != device or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{name} must be a contiguous float32 tensor of {n} elements on {device}")
    return t.data_ptr()


class _PolicyCall:
    """The checked arguments of one policy-loss call, as the C ABI takes them."""

    def __init__(self, logits, actions, old_log_probs, advantages, clip_param, entropy_coef, kl_coef, ref_log_probs, active_masks, available_actions):
        if not logits.is_cuda or logits.dtype not in _TYPES or logits.dim() < 1:
            raise ValueError("logits must be a float32, bfloat16 or float16 CUDA tensor [..., actions]")
        n_actions = logits.shape[-1]
        if not 1 <= n_actions <= 2 ** 28:
            raise ValueError("logits need 1 to 2^28 actions")
        rows = logits.numel() // n_actions
        dev = logits.device
        flat = logits if logits.dim() == 2 else logits.reshape(1, -1) if logits.dim() == 1 else logits.flatten(0, -2)
        stride = flat.stride(0) if rows > 1 else n_actions
        if rows and (flat.data_ptr() != logits.data_ptr() or (n_actions > 1 and flat.stride(1) != 1) or stride < n_actions):
            raise ValueError("logits need a last dimension of stride 1 and rows at one distance that do not overlap (call .contiguous())")
        if actions.dtype not in _ACTION_TYPES or actions.device != dev or not actions.is_contiguous() or actions.numel() != rows:
            raise ValueError(f"actions must be a contiguous int32, int64 or float32 tensor of {rows} elements on {dev}")
        if not clip_param >= 0:
            raise ValueError("clip_param must not be negative")
        self.shape, self.dtype, self.device = logits.shape, logits.dtype, dev
        a = self.args = native.OcPolicyLossArgs()
        a.d_logits, a.d_actions = logits.data_ptr(), actions.data_ptr()
        a.d_old_log_probs = _rows_f32("old_log_probs", old_log_probs, rows, dev)
        a.d_advantages = _rows_f32("advantages", advantages, rows, dev)
        if ref_log_probs is not None:
            a.d_ref_log_probs = _rows_f32("ref_log_probs", ref_log_probs, rows, dev)
        if active_masks is not None:
            a.d_active_masks = _rows_f32("active_masks", active_masks, rows, dev)
        if available_actions is not None:
            av = available_actions
            if av.dtype not in (torch.float32, torch.bool, torch.uint8) or av.device != dev or av.shape[-1] != n_actions or av.numel() != rows * n_actions:
                raise ValueError(f"available_actions must be float32, bool or uint8 of the logits' shape on {dev}")
            if rows:
                av2 = av if av.dim() == 2 else av.reshape(1, -1) if av.dim() == 1 else av.flatten(0, -2)
                if av2.data_ptr() != av.data_ptr() or (n_actions > 1 and av2.stride(1) != 1):
                    raise ValueError("available_actions need a last dimension of stride 1 and rows at one distance")
                a.d_available, a.available_u8 = av.data_ptr(), int(av.dtype != torch.float32)
                a.available_stride = av2.stride(0) if rows > 1 else n_actions
        a.rows, a.row_stride, a.n_actions = rows, stride, n_actions
        a.logits_type, a.action_type = _TYPES[logits.dtype], _ACTION_TYPES[actions.dtype]
        a.clip_param, a.entropy_coef, a.kl_coef, a.grad_scale = float(clip_param), float(entropy_coef), float(kl_coef), 1.0

    def forward(self, want_grad, grad_scale=1.0, weight=None):
        a, dev = self.args, self.device
        workspace = _workspace("oc_policy_loss_workspace_bytes", dev)
        loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(5, dtype=torch.float32, device=dev)
        grad = torch.empty(self.shape, dtype=self.dtype, device=dev) if want_grad else None
        a.d_loss, a.d_stats, a.d_weight = loss.data_ptr(), stats.data_ptr(), None if weight is None else weight.data_ptr()
        a.d_grad, a.grad_scale = grad.data_ptr() if want_grad else None, float(grad_scale)
        native.check(native.lib().oc_policy_loss(ctypes.byref(a), _FORWARD_GRAD if want_grad else _FORWARD, workspace.data_ptr(), _stream(dev)))
        return loss, stats, grad


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old, adv, ref, masks, avail, clip_param, entropy_coef, kl_coef):
        call = _PolicyCall(logits, actions, old, adv, clip_param, entropy_coef, kl_coef, ref, masks, avail)
        ctx.weight = torch.empty(1, dtype=torch.float64, device=logits.device)
        loss, stats, _ = call.forward(False, weight=ctx.weight)
        ctx.save_for_backward(logits, actions, old, adv, ref, masks, avail)
        ctx.coefs = (clip_param, entropy_coef, kl_coef)
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        # looked at again: hooks on saved tensors (checkpointing, keeping them on the host) may hand back others
        logits, actions, old, adv, ref, masks, avail = ctx.saved_tensors
        a = _PolicyCall(logits, actions, old, adv, *ctx.coefs, ref, masks, avail).args
        grad_loss = grad_loss.to(torch.float32).contiguous()
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a.d_weight, a.d_grad, a.d_grad_out = ctx.weight.data_ptr(), grad.data_ptr(), grad_loss.data_ptr()
        native.check(native.lib().oc_policy_loss(ctypes.byref(a), _BACKWARD, None, _stream(grad.device)))
        return (grad,) + (None,) * 9


def policy_loss(logits, actions, old_log_probs, advantages, clip_param=0.2, entropy_coef=0.01, kl_coef=0.0, ref_log_probs=None, active_masks=None,
                available_actions=None):
    """Clipped policy loss over action logits with an entropy bonus and a KL term to a reference policy -- the policy half of the
    reference's `R_MAPPO.ppo_update` (train/MAPPO/r_mappo.py) from the actor's logits on, differentiable in `logits`:

        lp = log softmax(logits)[action] over the possible actions;  ratio = exp(lp - old_log_probs)
        loss = mean_w( -min(ratio A, clamp(ratio, 1 - c, 1 + c) A) - entropy_coef H + kl_coef (exp(ref - lp) - (ref - lp) - 1) )

    logits f32 / bf16 / f16 [..., actions] (rows may be a slice of a padded buffer); actions int32 / int64 / float32, one per row, e.g.
    `[n, 1]` as MinibatchSource yields them -- an action outside [0, actions) marks a padded row; old_log_probs, advantages, ref_log_probs
    (None: no KL term), active_masks (the weights of the mean, None: 1) contiguous f32, one per row; available_actions of the logits'
    shape, f32 / bool / uint8, non-zero = available (a broadcast view is taken as it is).  A logit of -inf is an action that is not
    possible, too.  A row whose mask leaves nothing, or whose taken action is not possible, adds nothing to the sums; its weight stays in
    the mean's denominator, as in `active_masks.sum()`.  Rows of weight 0 may hold anything.
    -> (loss f32 scalar, stats f32 [5]: the means named in POLICY_STATS, not differentiable)

    `loss.backward()` recomputes the softmax from the logits: no [rows, actions] tensor is kept.  `policy_loss_grad` gives the gradient at once.
    """
    _refuse_tangents("policy_loss", logits, old_log_probs, advantages, ref_log_probs, active_masks)
    if logits.requires_grad and torch.is_grad_enabled():
        return _PolicyLoss.apply(logits, actions, old_log_probs, advantages, ref_log_probs, active_masks, available_actions, clip_param, entropy_coef, kl_coef)
    return _PolicyCall(logits, actions, old_log_probs, advantages, clip_param, entropy_coef, kl_coef, ref_log_probs, active_masks,
                       available_actions).forward(False)[:2]


def policy_loss_grad(logits, actions, old_log_probs, advantages, clip_param=0.2, entropy_coef=0.01, kl_coef=0.0, ref_log_probs=None, active_masks=None,
                     available_actions=None, grad_scale=1.0):
    """`policy_loss` and its gradient in one pass over the logits, outside autograd: -> (loss, stats, grad), grad = grad_scale * d loss /
    d logits, contiguous, of the logits' shape and type, for `logits.backward(grad)`.  grad_scale: loss scaling for float16, whose range a
    mean over many rows leaves."""
    _refuse_tangents("policy_loss_grad", logits, old_log_probs, advantages, ref_log_probs, active_masks)
    return _PolicyCall(logits, actions, old_log_probs, advantages, clip_param, entropy_coef, kl_coef, ref_log_probs, active_masks,
                       available_actions).forward(True, grad_scale)


class _ValueCall:
    def __init__(self, values, value_preds, returns, clip_param, huber_delta, active_masks, value_normalizer):
        if not values.is_cuda or values.dtype not in _TYPES or not values.is_contiguous():
            raise ValueError("values must be a contiguous float32, bfloat16 or float16 CUDA tensor")
        n, dev = values.numel(), values.device
        if clip_param is not None and not clip_param >= 0 or huber_delta is not None and not huber_delta >= 0:
            raise ValueError("clip_param and huber_delta must not be negative (None: without)")
        mean, std = (0.0, 1.0) if value_normalizer is None else (float(x) for x in value_normalizer)
        self.values = values
        a = self.args = native.OcValueLossArgs()
        a.d_values = values.data_ptr()
        a.d_value_preds, a.d_returns = _rows_f32("value_preds", value_preds, n, dev), _rows_f32("returns", returns, n, dev)
        if active_masks is not None:
            a.d_active_masks = _rows_f32("active_masks", active_masks, n, dev)
        a.n, a.values_type = n, _TYPES[values.dtype]
        a.clip_param = -1.0 if clip_param is None else float(clip_param)
        a.huber_delta = -1.0 if huber_delta is None else float(huber_delta)
        a.mean, a.std, a.grad_scale = mean, std, 1.0

    def forward(self, want_grad, grad_scale=1.0, weight=None):
        a, dev = self.args, self.values.device
        workspace = _workspace("oc_value_loss_workspace_bytes", dev)
        grad = torch.empty(self.values.shape, dtype=self.values.dtype, device=dev) if want_grad else None
        loss = torch.empty((), dtype=torch.float32, device=dev)
        a.d_loss, a.d_weight = loss.data_ptr(), None if weight is None else weight.data_ptr()
        a.d_grad, a.grad_scale = grad.data_ptr() if want_grad else None, float(grad_scale)
        native.check(native.lib().oc_value_loss(ctypes.byref(a), _FORWARD_GRAD if want_grad else _FORWARD, workspace.data_ptr(), _stream(dev)))
        return loss, grad


class _ValueLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, values, preds, returns, masks, clip_param, huber_delta, norm):
        ctx.weight = torch.empty(1, dtype=torch.float64, device=values.device)
        call = _ValueCall(values, preds, returns, clip_param, huber_delta, masks, norm)
        loss, _ = call.forward(False, weight=ctx.weight)
        ctx.save_for_backward(values, preds, returns, masks)
        ctx.rest = (clip_param, huber_delta, norm)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        values, preds, returns, masks = ctx.saved_tensors
        clip_param, huber_delta, norm = ctx.rest
        a = _ValueCall(values, preds, returns, clip_param, huber_delta, masks, norm).args
        grad_loss = grad_loss.to(torch.float32).contiguous()
        grad = torch.empty(values.shape, dtype=values.dtype, device=values.device)
        a.d_weight, a.d_grad, a.d_grad_out = ctx.weight.data_ptr(), grad.data_ptr(), grad_loss.data_ptr()
        native.check(native.lib().oc_value_loss(ctypes.byref(a), _BACKWARD, None, _stream(grad.device)))
        return (grad,) + (None,) * 6


def _normalizer(value_normalizer):
    """None, a (mean, std) pair, or the reference's ValueNorm / PopArt (`running_mean_var()`: read back, synchronises) -- as `gae_returns` takes it."""
    if value_normalizer is None:
        return None
    if hasattr(value_normalizer, "running_mean_var"):
        m, v = value_normalizer.running_mean_var()
        pair = float(m.reshape(-1)[0]), math.sqrt(float(v.reshape(-1)[0]))
    else:
        pair = tuple(float(x) for x in value_normalizer)
    if len(pair) != 2 or not pair[1] > 0:
        raise ValueError("value_normalizer must give a mean and a positive standard deviation")
    return pair


def value_loss(values, value_preds, returns, clip_param=0.2, huber_delta=10.0, active_masks=None, value_normalizer=None):
    """Clipped value loss of the reference's `R_MAPPO.cal_value_loss` (train/MAPPO/r_mappo.py), differentiable in `values`:

        y = (returns - mean) / std;   loss = mean_w max( h(y - v), h(y - (v0 + clamp(v - v0, -c, c))) )

    values f32 / bf16 / f16, value_preds (v0: the values of the rollout), returns and active_masks (None: 1) f32, all contiguous with as
    many elements; h: Huber's loss of `huber_delta`, None: e^2 / 2; clip_param None: without the clipped branch; value_normalizer: None, a
    (mean, std) pair or an object with `running_mean_var()`, as in `gae_returns` -- the object is read back to the host at the call: it waits
    for the GPU, and a captured graph wants the pair, which stays what it was at the capture.  Samples of weight 0 may hold anything.
    -> f32 scalar."""
    _refuse_tangents("value_loss", values, value_preds, returns, active_masks)
    norm = _normalizer(value_normalizer)
    if values.requires_grad and torch.is_grad_enabled():
        return _ValueLoss.apply(values, value_preds, returns, active_masks, clip_param, huber_delta, norm)
    return _ValueCall(values, value_preds, returns, clip_param, huber_delta, active_masks, norm).forward(False)[0]


def value_loss_grad(values, value_preds, returns, clip_param=0.2, huber_delta=10.0, active_masks=None, value_normalizer=None, grad_scale=1.0):
    """`value_loss` and its gradient in one pass, outside autograd: -> (loss, grad_scale * d loss / d values of the values' shape and type)."""
    _refuse_tangents("value_loss_grad", values, value_preds, returns, active_masks)
    return _ValueCall(values, value_preds, returns, clip_param, huber_delta, active_masks, _normalizer(value_normalizer)).forward(True, grad_scale)


def _one_piece(t):
    """Whether a tensor's elements fill one piece of memory without gaps or overlaps, in whatever order."""
    if t.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _look_at(tensors, name, device):
    """-> types, element counts, addresses of a list of tensors on one GPU"""
    dtypes = {t.dtype for t in tensors}
    if not tensors[0].is_cuda or set(map(torch.Tensor.get_device, tensors)) != {device.index} or not dtypes <= _TYPES.keys():
        raise ValueError(f"{name} must be float32, bfloat16 or float16 CUDA tensors of one device")
    types = [_TYPES[dtypes.pop()]] * len(tensors) if len(dtypes) == 1 else [_TYPES[t.dtype] for t in tensors]
    return types, list(map(torch.Tensor.numel, tensors)), list(map(torch.Tensor.data_ptr, tensors))


def clip_grad_norm(grads, max_norm=None, norm_type=2.0, out=None):
    """Norm of all elements of a list of gradient tensors, and clipping to it -- `torch.nn.utils.clip_grad_norm_` for the framework's
    updates (the reference: train/MAPPO/r_mappo.py before every optimiser step, `get_gard_norm` where it only logs):

        g <- g * min(1, max_norm / (norm + 1e-6))

    grads: f32 / bf16 / f16 CUDA tensors of one device, mixed as they come, each one dense piece of memory (any order of dimensions); or
    modules' parameters -- where an entry is an nn.Parameter its `.grad` is taken, and skipped if None.  max_norm None: the norm alone.
    norm_type 2 or inf.  out: tensors of the same shapes (contiguous ones: sizes), strides and types for the clipped gradients (default: in place; gradients that
    need no clipping are then not written; this goes past autograd's version counters).  The same
    tensor must not be listed twice, and none may overlap another.  -> norm, f32 scalar on the device; squares are
    added in f64, so no gradient is too small or too large for it."""
    if isinstance(grads, torch.Tensor):
        grads = [grads]
    plain = torch.Tensor                                 # hundreds of tensors: one cheap look at each property, all at once
    tensors = [g if type(g) is plain else g.grad if isinstance(g, torch.nn.Parameter) else g for g in grads]
    tensors = [t for t in tensors if t is not None]
    _refuse_tangents("clip_grad_norm", *tensors)
    if norm_type not in (2, 2.0, math.inf, "inf"):
        raise ValueError("norm_type must be 2 or inf")
    if max_norm is not None and not max_norm >= 0:
        raise ValueError("max_norm must not be negative")
    if out is not None and (max_norm is None or len(out) != len(tensors)):
        raise ValueError("out wants max_norm and one tensor per gradient")
    if not tensors:
        return torch.zeros((), dtype=torch.float32)
    n, device = len(tensors), tensors[0].device
    types, counts, src = _look_at(tensors, "gradients", device)
    dense = all(map(plain.is_contiguous, tensors))
    if not dense:
        for i, t in enumerate(tensors):
            if not _one_piece(t):
                raise ValueError(f"gradient {i} is not one dense piece of memory")
    if max_norm is not None and len({p for p, c in zip(src, counts) if c}) != n - counts.count(0):
        raise ValueError("a gradient is listed twice")
    dst = None
    if out is not None:
        out_types, out_counts, dst = _look_at(out, "out", device)
        if out_types != types or out_counts != counts:
            raise ValueError("out must have the types and sizes of the gradients")
        if not (dense and all(map(plain.is_contiguous, out))) and any(o.shape != t.shape or o.stride() != t.stride() for o, t in zip(out, tensors)):
            raise ValueError("out must have the shapes and strides of the gradients")
        dst = array("Q", dst)
    L = native.lib()
    workspace = torch.empty(L.oc_grad_norm_workspace_bytes(n), dtype=torch.uint8, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    src, counts, types = array("Q", src), array("q", counts), array("i", types)
    at = lambda a: None if a is None else a.buffer_info()[0]
    native.check(L.oc_grad_norm_clip(n, at(src), at(dst), at(counts), at(types), -1.0 if max_norm is None else float(max_norm),
                                     0 if norm_type in (2, 2.0) else 1, norm.data_ptr(), workspace.data_ptr(), _stream(device)))
    return norm
