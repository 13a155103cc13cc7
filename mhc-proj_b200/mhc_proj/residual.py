"""Autograd functions and modules of the residual path around a sublayer F of
an mHC layer with n = 4 streams X (no reference counterparts):

  MHCStreamNormN4   F's input: layer norm of sum_i h_pre[i] X[i]
  MHCStreamMixN4    X' = T X + h_post (x) dropout(F(...)), T a projected matrix
  MHCLayerNorm      layer norm of plain rows
  MHCDropout        dropout whose mask is never stored

    T = mhc_proj.MHCProjectionN4HRes()(H[..., 8:24], rms, alpha_res, b_res)
    X = mix(X, T, sublayer(norm(X, h_pre)), h_post)

Shapes are checked as in module.py (ValueError); a ``None`` incoming gradient
yields ``None``.  The backward functions are kernels, not differentiable once
more.
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _internal

_f = _internal.torch


class MHCLayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps=1e-5):
        x2 = x.reshape(-1, x.shape[-1])
        out = _f.layer_norm(x2, weight, bias, eps)
        ctx.save_for_backward(x2, out["mean"], out["rstd"], weight, bias)
        ctx.set_materialize_grads(False)
        return out["y"].view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        if grad_output is None or not any(ctx.needs_input_grad[:3]):
            return None, None, None, None
        x2, mean, rstd, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = _f.layer_norm_backward(grad_output.reshape(x2.shape), x2, mean, rstd, weight, bias if need[2] else None)
        return (g["d_x"].view(grad_output.shape) if need[0] else None, g["d_weight"] if need[1] else None,
                g["d_bias"] if need[2] else None, None)


class _Affine(nn.Module):
    def __init__(self, width, eps, affine, bias, device, dtype):
        super().__init__()
        if width < 1:
            raise ValueError("width must be at least 1")
        self.width, self.eps = width, eps
        kw = {"device": device, "dtype": dtype}
        self.weight = nn.Parameter(torch.ones(width, **kw)) if affine else None
        self.bias = nn.Parameter(torch.zeros(width, **kw)) if affine and bias else None

    def extra_repr(self):
        return f"{self.width}, eps={self.eps}, affine={self.weight is not None}, bias={self.bias is not None}"


class MHCLayerNorm(_Affine):
    """Layer norm over the last dimension (`width` elements); the weight and
    bias may be of x's type or fp32 (their gradients are summed in fp32 and
    returned in their own type).  affine=False: neither."""

    def __init__(self, width, eps=1e-5, affine=True, bias=True, device=None, dtype=None):
        super().__init__(width, eps, affine, bias, device, dtype)

    def forward(self, x):
        if x.ndim < 1 or x.shape[-1] != self.width:
            raise ValueError(f"x must be a tensor of size ... x {self.width}")
        return MHCLayerNormFunction.apply(x, self.weight, self.bias, self.eps)


class MHCStreamNormN4Function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, h_pre, weight, bias, eps=1e-5):
        X3 = X.reshape(-1, 4, X.shape[-1])
        h2 = h_pre.reshape(-1, 4)
        out = _f.stream_norm_n4(X3, h2, weight, bias, eps)
        ctx.save_for_backward(X3, h2, out["mean"], out["rstd"], weight, bias)
        ctx.shapes = X.shape, h_pre.shape
        ctx.set_materialize_grads(False)
        return out["y"].view(*X.shape[:-2], X.shape[-1])

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        if grad_output is None or not any(ctx.needs_input_grad[:4]):
            return None, None, None, None, None
        X3, h2, mean, rstd, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        g = _f.stream_norm_n4_backward(grad_output.reshape(-1, X3.shape[-1]), X3, h2, mean, rstd, weight,
                                       bias if need[3] else None)
        return (g["d_X"].view(ctx.shapes[0]) if need[0] else None, g["d_h_pre"].view(ctx.shapes[1]) if need[1] else None,
                g["d_weight"] if need[2] else None, g["d_bias"] if need[3] else None, None)


def _check_streams(X, width=None):
    if X.ndim < 2 or X.shape[-2] != 4 or (width is not None and X.shape[-1] != width):
        raise ValueError(f"X must be a tensor of size ... x 4 x {'C' if width is None else width}")


def _check_lead(t, shape, name):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be a tensor of size {' x '.join(str(s) for s in shape)}")


class MHCStreamNormN4(_Affine):
    """Layer norm of sum_i h_pre[..., i] * X[..., i, :], the sublayer's input
    from the four residual streams, without the sum in memory.

    forward(X, h_pre) with X (..., 4, width) and h_pre (..., 4); returns
    (..., width).  Gradients for both and for the weight and bias."""

    def __init__(self, width, eps=1e-5, affine=True, bias=True, device=None, dtype=None):
        super().__init__(width, eps, affine, bias, device, dtype)

    def forward(self, X, h_pre):
        _check_streams(X, self.width)
        _check_lead(h_pre, X.shape[:-1], "h_pre")
        return MHCStreamNormN4Function.apply(X, h_pre, self.weight, self.bias, self.eps)


def _fresh_seed(x):
    """A dropout seed from torch's generator of x's device, where it stays: no
    host read, `torch.manual_seed` decides it, and a captured graph draws
    another one at each replay."""
    device = x.device if x.is_cuda else "cuda"
    return torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), dtype=torch.int64, device=device)


class MHCDropoutFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, offset=0):
        ctx.p, ctx.offset = p, offset
        ctx.seed = None if torch.is_tensor(seed) else seed
        ctx.save_for_backward(*((seed,) if ctx.seed is None else ()))
        ctx.set_materialize_grads(False)
        return _f.dropout(x, p, seed, offset)["y"]

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        if grad_output is None or not ctx.needs_input_grad[0]:
            return None, None, None, None
        seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
        return _f.dropout_backward(grad_output, ctx.p, seed, ctx.offset)["d_x"], None, None, None


def _check_p(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be between 0 and 1")
    return p


class MHCDropout(nn.Module):
    """Dropout in training mode (the identity otherwise): each element is zero
    with probability p (to the nearest multiple of 2^-16), the others are
    scaled to keep the expectation.  The mask is formed again in the backward
    pass from the forward's seed.  forward(x, seed=None, offset=0): a number
    or a one-element int64 tensor fixes the mask; by default the seed comes from
    torch's generator of x's device."""

    def __init__(self, p=0.5):
        super().__init__()
        self.p = _check_p(p)

    def forward(self, x, seed=None, offset=0):
        if not self.training or self.p == 0.0:
            return x
        return MHCDropoutFunction.apply(x, self.p, _fresh_seed(x) if seed is None else seed, offset)

    def extra_repr(self):
        return f"p={self.p}"


class MHCStreamMixN4Function(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, T, y, h_post, p=0.0, seed=0, offset=0):
        width = X.shape[-1]
        X3, T3, y2, h2 = X.reshape(-1, 4, width), T.reshape(-1, 4, 4), y.reshape(-1, width), h_post.reshape(-1, 4)
        ctx.p, ctx.offset = p, offset
        ctx.seed = None if torch.is_tensor(seed) else seed
        ctx.save_for_backward(X3, T3, y2, h2, *((seed,) if ctx.seed is None else ()))
        ctx.shapes = X.shape, T.shape, y.shape, h_post.shape
        ctx.set_materialize_grads(False)
        return _f.stream_mix_n4(X3, T3, y2, h2, p, seed, offset)["X"].view(X.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        if grad_output is None or not any(ctx.needs_input_grad[:4]):
            return (None,) * 7
        X3, T3, y2, h2, *seed = ctx.saved_tensors
        g = _f.stream_mix_n4_backward(grad_output.reshape(X3.shape), X3, T3, y2, h2, ctx.p,
                                      seed[0] if seed else ctx.seed, ctx.offset)
        grads = (g["d_X"], g["d_T"], g["d_y"], g["d_h_post"])
        return (*(d.view(s) if n else None for d, s, n in zip(grads, ctx.shapes, ctx.needs_input_grad)),
                None, None, None)


class MHCStreamMixN4(nn.Module):
    """The residual update of an mHC layer, X' = T X + h_post (x) dropout(y):
    the projected matrices T applied to the four streams, and the sublayer's
    output y spread over them.  In training mode p drops elements of y as
    MHCDropout does (the same mask for the same seed), without y's dropped
    form or a mask in memory.

    forward(X, T, y, h_post, seed=None, offset=0) with X (..., 4, C), T
    (..., 4, 4), y (..., C) and h_post (..., 4); returns (..., 4, C).
    Gradients for all four."""

    def __init__(self, p=0.0):
        super().__init__()
        self.p = _check_p(p)

    def forward(self, X, T, y, h_post, seed=None, offset=0):
        _check_streams(X)
        lead, width = X.shape[:-2], X.shape[-1]
        _check_lead(T, (*lead, 4, 4), "T")
        _check_lead(y, (*lead, width), "y")
        _check_lead(h_post, (*lead, 4), "h_post")
        p = self.p if self.training else 0.0
        if seed is None:
            seed = _fresh_seed(X) if p else 0
        return MHCStreamMixN4Function.apply(X, T, y, h_post, p, seed, offset)

    def extra_repr(self):
        return f"p={self.p}"
