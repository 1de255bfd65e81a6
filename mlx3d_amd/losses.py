"""Image losses of the training step (``src/mlx3d/losses/image_metrics.py``).

``photometric`` returns mean |pred - target| and mean SSIM of one image from
one fused kernel pass (``gsx_photometric_fwd``), and the gradient of any
combination of the two from a second (``gsx_photometric_bwd``).
``photometric_loss`` is the trainer's ``(1 - lambda) L1 + lambda (1 - SSIM)``
(trainer.py:303-305) as one op: the same kernels form the scalar and take
its cotangent (``gsx_photometric_loss_fwd`` / ``_bwd``), the values that
expression's autograd graph gives.  ``ssim`` is the reference's function on
top of ``photometric``, and ``l1_loss`` the L1 term alone
(``gsx_l1_fwd_signs`` / ``gsx_l1_bwd_signs``).

``distillation_loss`` compares a student's logits (a decoded feature render)
with the largest ones that a teacher kept for each row, and
``distillation_value_and_grad`` gives loss and gradient in one pass over the
logits (``gsx_distil_*``; no counterpart in the reference).
"""

from __future__ import annotations

import torch

from . import _lib
from .profiling import stage

__all__ = ["distillation_loss", "distillation_value_and_grad", "l1_loss", "photometric", "photometric_loss", "psnr", "ssim"]


class _PhotometricFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target, window_size, sigma, max_val):
        H, W, C = pred.shape
        L = _lib.load()
        nbytes = int(L.gsx_photometric_workspace_bytes(H, W, C))
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=pred.device)
        out = torch.empty((2,), dtype=torch.float32, device=pred.device)
        with stage("photometric_fwd"):
            _lib.check(L.gsx_photometric_fwd(H, W, C, _lib.ptr(pred), _lib.ptr(target),
                                             int(window_size), float(sigma), float(max_val),
                                             _lib.ptr(ws), nbytes, _lib.ptr(out),
                                             _lib.stream_handle(pred.device)),
                       "gsx_photometric_fwd")
        ctx.save_for_backward(pred, target, ws)
        ctx.window = (int(window_size), float(sigma))
        return out

    @staticmethod
    def backward(ctx, g_out):
        pred, target, ws = ctx.saved_tensors
        H, W, C = pred.shape
        g = _lib.f32c(g_out)
        grad = torch.empty_like(pred)
        with stage("photometric_bwd"):
            _lib.check(_lib.load().gsx_photometric_bwd(
                H, W, C, _lib.ptr(pred), _lib.ptr(target), ctx.window[0], ctx.window[1],
                _lib.ptr(ws), ws.numel(), _lib.ptr(g), _lib.ptr(grad),
                _lib.stream_handle(pred.device)), "gsx_photometric_bwd")
        return grad, None, None, None, None


class _PhotometricLossFn(torch.autograd.Function):
    """(1 - lam) L1 + lam (1 - SSIM) as one op: the scalar comes out of the
    loss kernels' reduction and its gradient goes straight into the SSIM
    backward, the same float32 values the expression's autograd graph
    produces, without its dozen elementwise launches."""

    @staticmethod
    def forward(ctx, pred, target, lam, window_size, sigma, max_val):
        H, W, C = pred.shape
        L = _lib.load()
        nbytes = int(L.gsx_photometric_workspace_bytes(H, W, C))
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=pred.device)
        out = torch.empty((3,), dtype=torch.float32, device=pred.device)
        with stage("photometric_fwd"):
            _lib.check(L.gsx_photometric_loss_fwd(
                H, W, C, _lib.ptr(pred), _lib.ptr(target), int(window_size), float(sigma),
                float(max_val), float(lam), _lib.ptr(ws), nbytes, _lib.ptr(out),
                _lib.stream_handle(pred.device)), "gsx_photometric_loss_fwd")
        ctx.save_for_backward(pred, target, ws)
        ctx.args = (float(lam), int(window_size), float(sigma))
        return out[2]

    @staticmethod
    def backward(ctx, g_out):
        pred, target, ws = ctx.saved_tensors
        lam, window_size, sigma = ctx.args
        H, W, C = pred.shape
        g = _lib.f32c(g_out.reshape(1))
        grad = torch.empty_like(pred)
        with stage("photometric_bwd"):
            _lib.check(_lib.load().gsx_photometric_loss_bwd(
                H, W, C, _lib.ptr(pred), _lib.ptr(target), window_size, sigma, lam,
                _lib.ptr(ws), ws.numel(), _lib.ptr(g), _lib.ptr(grad),
                _lib.stream_handle(pred.device)), "gsx_photometric_loss_bwd")
        return grad, None, None, None, None, None


def _check_window(window_size: int, sigma: float):
    if window_size < 1 or window_size % 2 == 0 or window_size > 15:
        raise ValueError("window_size must be odd and at most 15.")
    if not sigma > 0:
        raise ValueError("sigma must be positive.")


def photometric(pred: torch.Tensor, target: torch.Tensor, window_size: int = 11,
                sigma: float = 1.5, max_val: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(mean |pred - target|, mean SSIM) of (H, W, C) images, differentiable
    with respect to ``pred`` (image_metrics.py:13-14, 29-55)."""
    if pred.shape != target.shape or pred.ndim != 3:
        raise ValueError("pred and target must both have shape (H, W, C).")
    _check_window(window_size, sigma)
    _lib.require_device(pred, target)
    out = _PhotometricFn.apply(_lib.f32c(pred), _lib.f32c(target).detach(), window_size, sigma,
                               max_val)
    return out[0], out[1]


def photometric_loss(pred: torch.Tensor, target: torch.Tensor, lam: float,
                     window_size: int = 11, sigma: float = 1.5,
                     max_val: float = 1.0) -> torch.Tensor:
    """The trainer's objective (1 - lam) mean|pred - target| + lam (1 - mean
    SSIM) (trainer.py:303-305) as a scalar tensor, differentiable with
    respect to ``pred``; the same value and gradient, bit for bit, as that
    expression over :func:`photometric`'s two outputs, in two kernel calls."""
    if pred.shape != target.shape or pred.ndim != 3:
        raise ValueError("pred and target must both have shape (H, W, C).")
    _check_window(window_size, sigma)
    if not 0.0 <= float(lam) <= 1.0:
        raise ValueError("lam must lie in [0, 1].")
    _lib.require_device(pred, target)
    return _PhotometricLossFn.apply(_lib.f32c(pred), _lib.f32c(target).detach(), float(lam),
                                    window_size, sigma, max_val)


def ssim(pred: torch.Tensor, target: torch.Tensor, max_val: float = 1.0, window_size: int = 11,
         sigma: float = 1.5) -> torch.Tensor:
    """Mean SSIM with a Gaussian window (image_metrics.py:66-85).  ``pred``
    (H, W, C) or (N, H, W, C); the mean runs over every pixel and channel."""
    if pred.shape != target.shape:
        raise ValueError("pred and target must have the same shape.")
    if pred.ndim == 3:
        return photometric(pred, target, window_size, sigma, max_val)[1]
    if pred.ndim != 4:
        raise ValueError("pred must have shape (H, W, C) or (N, H, W, C).")
    vals = [photometric(pred[i], target[i], window_size, sigma, max_val)[1]
            for i in range(pred.shape[0])]
    return torch.stack(vals).mean()


class _L1Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, pred, target):
        n = pred.numel()
        L = _lib.load()
        nbytes = int(L.gsx_l1_workspace_bytes(n))
        ws = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device=pred.device)
        out = torch.empty((1,), dtype=torch.float32, device=pred.device)
        # the signs of pred - target, kept for the backward (1 byte each)
        signs = torch.empty((n,), dtype=torch.uint8, device=pred.device)
        with stage("l1_fwd"):
            _lib.check(L.gsx_l1_fwd_signs(n, _lib.ptr(pred), _lib.ptr(target), _lib.ptr(ws),
                                          nbytes, _lib.ptr(signs), _lib.ptr(out),
                                          _lib.stream_handle(pred.device)), "gsx_l1_fwd_signs")
        ctx.save_for_backward(pred, target, signs)
        return out[0]

    @staticmethod
    def backward(ctx, g_out):
        pred, target, signs = ctx.saved_tensors
        g = _lib.f32c(g_out.reshape(1))
        grad = torch.empty_like(pred)
        with stage("l1_bwd"):
            _lib.check(_lib.load().gsx_l1_bwd_signs(
                pred.numel(), _lib.ptr(signs), _lib.ptr(pred), _lib.ptr(target), _lib.ptr(g),
                _lib.ptr(grad), _lib.stream_handle(pred.device)), "gsx_l1_bwd_signs")
        return grad, None


def l1_loss(pred: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """Mean absolute error (image_metrics.py:13-14), differentiable with
    respect to ``pred``: one reduction kernel forward that also keeps the
    sign of each difference, one elementwise gradient kernel backward from
    those signs (gsx_l1_fwd_signs / gsx_l1_bwd_signs)."""
    if pred.shape != target.shape:
        raise ValueError("pred and target must have the same shape.")
    if pred.numel() == 0:
        raise ValueError("l1_loss of empty tensors.")
    _lib.require_device(pred, target)
    return _L1Fn.apply(_lib.f32c(pred), _lib.f32c(target).detach())


def psnr(pred: torch.Tensor, target: torch.Tensor, max_val: float = 1.0) -> torch.Tensor:
    """Peak signal-to-noise ratio in dB (image_metrics.py:17-20)."""
    mse = ((pred - target) ** 2).mean()
    return 10.0 * torch.log10((max_val * max_val) / torch.clamp(mse, min=1e-12))


_TEACHERS = {"logits": 0, "log_probs": 1}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
DISTILLATION_MAX_TOP = 256  # GSX_DISTIL_MAX_TOP


class _Distillation:
    """The checked arguments of one distillation call, as the C entry points
    take them."""

    def __init__(self, logits, values, indices, temperature, teacher, reduction):
        if logits.ndim < 1 or logits.dtype not in _lib.DTYPES:
            raise ValueError("logits must be (..., V) in float32, bfloat16 or float16.")
        if values.shape != indices.shape or values.ndim != logits.ndim or \
                values.shape[:-1] != logits.shape[:-1]:
            raise ValueError("teacher_values and teacher_indices must both have shape (..., K), "
                             "with the logits' leading dimensions.")
        if not values.is_floating_point():
            raise ValueError("teacher_values must be floating point.")
        if indices.dtype not in (torch.int32, torch.int64):
            raise ValueError("teacher_indices must be int32 or int64.")
        vocab, top = int(logits.shape[-1]), int(values.shape[-1])
        if not 1 <= top <= min(vocab, DISTILLATION_MAX_TOP):
            raise ValueError("a row must have between 1 and "
                             f"min(V, {DISTILLATION_MAX_TOP}) teacher entries.")
        if not 1e-38 <= float(temperature) < 3.0e38:
            raise ValueError("temperature must be positive and finite, with a reciprocal that "
                             "float32 holds (from 1e-38 on).")
        if teacher not in _TEACHERS:
            raise ValueError("teacher must be 'logits' or 'log_probs'.")
        if reduction not in _REDUCTIONS:
            raise ValueError("reduction must be 'none', 'sum' or 'mean'.")
        self.device = _lib.require_device(logits, values, indices)
        self.shape = logits.shape
        self.reduction = reduction
        self.values = _lib.f32c(values.detach())
        self.indices = indices.contiguous()
        rows = logits.numel() // vocab
        self.head = (_lib.DTYPES[logits.dtype], rows, vocab, top)
        self.tail = (_lib.ptr(self.values), _lib.ptr(self.indices),
                     int(indices.dtype == torch.int64), float(temperature), _TEACHERS[teacher],
                     _REDUCTIONS[reduction])

    def workspace(self) -> torch.Tensor:
        n = _lib.check(int(_lib.load().gsx_distil_workspace_bytes(*self.head)),
                       "gsx_distil_workspace_bytes")
        return torch.empty((n,), dtype=torch.uint8, device=self.device)

    def loss(self) -> torch.Tensor:
        shape = self.shape[:-1] if self.reduction == "none" else ()
        return torch.empty(shape, dtype=torch.float32, device=self.device)


class _DistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call):
        rows, stride = _lib.rows_of(logits)
        ws, loss = call.workspace(), call.loss()
        with stage("distil_fwd"):
            _lib.check(_lib.load().gsx_distil_fwd(
                *call.head, _lib.ptr(rows), stride, *call.tail, _lib.ptr(loss), _lib.ptr(ws),
                ws.numel(), _lib.stream_handle(call.device)), "gsx_distil_fwd")
        ctx.save_for_backward(logits, ws, call.values, call.indices)
        ctx.call = call
        return loss

    @staticmethod
    @_lib.once_differentiable("distillation_loss")
    def backward(ctx, saved, g_loss):
        # saved with the rest so that an entry changed in place since is noticed
        logits, ws, _, _ = saved
        call = ctx.call
        rows, stride = _lib.rows_of(logits)
        g = _lib.f32c(g_loss)
        grad = torch.empty(call.shape, dtype=logits.dtype, device=call.device)
        with stage("distil_bwd"):
            _lib.check(_lib.load().gsx_distil_bwd(
                *call.head, _lib.ptr(rows), stride, *call.tail, _lib.ptr(g), _lib.ptr(grad),
                _lib.ptr(ws), ws.numel(), _lib.stream_handle(call.device)), "gsx_distil_bwd")
        return grad, None


def distillation_loss(logits: torch.Tensor, teacher_values: torch.Tensor,
                      teacher_indices: torch.Tensor, temperature: float = 1.0,
                      teacher: str = "logits", reduction: str = "mean") -> torch.Tensor:
    """Kullback-Leibler divergence of a student's (..., V) ``logits`` from the
    (..., K) largest entries that a teacher kept for each row, times
    temperature^2; differentiable with respect to ``logits``.

    ``teacher="logits"``: the values are logits, p = softmax(values / T) over
    the row's entries, and the row's loss is T^2 sum p (log p - log q) with
    q = softmax(logits / T) over all V.  ``teacher="log_probs"``: the values
    are log-probabilities over the whole vocabulary (taken at the same
    temperature); the mass that the entries leave, r = 1 - sum p (0 if they
    exceed 1), is compared as one bucket with the student's mass outside them,
    or left out where the student has none there.

    An entry whose index lies outside [0, V) or whose value is -inf is absent.
    A row without entries has loss 0 and gradient 0 whatever its logits hold.
    ``reduction``: "mean" over the rows that have entries (0 if none has),
    "sum", or "none" (a loss for each row; weight rows by what multiplies it).
    At most 256 entries a row; values and indices carry no gradient, and the
    gradient none of its own (differentiating it raises an error)."""
    call = _Distillation(logits, teacher_values, teacher_indices, temperature, teacher, reduction)
    return _DistillationFn.apply(logits, call)


def distillation_value_and_grad(logits: torch.Tensor, teacher_values: torch.Tensor,
                                teacher_indices: torch.Tensor, temperature: float = 1.0,
                                teacher: str = "logits", reduction: str = "mean",
                                scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, gradient with respect to ``logits``) of
    :func:`distillation_loss`, both times ``scale``, in one pass over the
    logits: each is read once and its gradient written once, where autograd
    reads them a second time.  Feed the gradient on with
    ``logits.backward(grad)``.  ``reduction``: "mean" or "sum"."""
    if reduction == "none":
        raise ValueError("value_and_grad needs a scalar: reduction must be 'sum' or 'mean'.")
    call = _Distillation(logits, teacher_values, teacher_indices, temperature, teacher, reduction)
    rows, stride = _lib.rows_of(logits.detach())
    ws, loss = call.workspace(), call.loss()
    grad = torch.empty(call.shape, dtype=logits.dtype, device=call.device)
    with stage("distil_fwd_bwd"):
        _lib.check(_lib.load().gsx_distil_fwd_bwd(
            *call.head, _lib.ptr(rows), stride, *call.tail, float(scale), _lib.ptr(loss),
            _lib.ptr(grad), _lib.ptr(ws), ws.numel(), _lib.stream_handle(call.device)),
            "gsx_distil_fwd_bwd")
    return loss, grad
