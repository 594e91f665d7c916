"""Token operators on MI355X: the channel-mixing half of a transformer stage, for networks that mix a U-Net level's pixels / voxels as tokens.

    a = layer_norm(x, w, b)
    h = gated_ffn(a, w_gate, w_up)                  # act(a w_gate^T) * (a w_up^T), one kernel
    y = linear(h, w_down, residual=x)               # h w_down^T + x, one kernel

x is (..., width) with any number of leading dimensions, float32 or bfloat16; weights are (out, width) as in nn.Linear, in x's type; biases and norm parameters are float32.  Each
function is differentiable once (forward and backward are HIP kernels of libmisamd; torch is the allocator and the tape) and keeps what its backward pass needs only when a gradient is
wanted.  Work is enqueued on torch's current stream of x's device.  Under stream capture take gradients with torch.autograd.grad, or call the ops.*_bwd functions.
There is no CPU path: a tensor that is not on the GPU raises."""
import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import MisError


def _rows(t, width, name):
    """(..., width) -> (rows, width) with unit stride inside a row: a view where the strides allow one, else a copy"""
    if not isinstance(t, torch.Tensor) or t.dim() < 1 or t.shape[-1] != width or width < 1:
        raise MisError(f"{name} must be a (..., {width}) tensor, got {tuple(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    if t.dim() != 2:
        t = t.reshape(t.numel() // width, width)
    return _unit(t)


def _unit(t):
    s0, s1 = t.stride()
    return t if (s1 == 1 or t.shape[1] == 1) and (s0 >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def _weight(w, name):
    if not isinstance(w, torch.Tensor) or w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        raise MisError(f"{name} must be an (out, in) matrix, got {tuple(w.shape) if isinstance(w, torch.Tensor) else type(w)}")
    return _unit(w)


def _pair(a, b):
    """two matrices with one row stride"""
    return (a, b) if a.shape[0] <= 1 or a.stride(0) == b.stride(0) else (a.contiguous(), b.contiguous())


def _grads(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _empty(like, *shape, dtype=None):
    return torch.empty(shape, dtype=like.dtype if dtype is None else dtype, device=like.device)


# ---- layer norm ----------------------------------------------------------------------------------------------------------------------------
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _rows(x, x.shape[-1], "layer_norm: x")
        M, D = x2.shape
        y, mean, rstd = _empty(x2, M, D), _empty(x2, M, dtype=torch.float32), _empty(x2, M, dtype=torch.float32)
        ops.layernorm_fwd(x2, y, weight, bias, mean, rstd, eps)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        M, D = x.shape
        need = ctx.needs_input_grad
        dx = _empty(x, M, D) if need[0] else None
        dw = _empty(x, D, dtype=torch.float32) if need[1] else None
        db = _empty(x, D, dtype=torch.float32) if need[2] else None
        ops.layernorm_bwd(_rows(dy, D, "dy"), x, mean, rstd, weight, dx, dw, db)
        return None if dx is None else dx.view(ctx.shape), dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension; weight, bias (width,) float32 or None"""
    if _grads(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    x2 = _rows(x, x.shape[-1], "layer_norm: x")
    y = _empty(x2, *x2.shape)
    ops.layernorm_fwd(x2, y, weight, bias, None, None, eps)
    return y.view(x.shape)


# ---- matrix product with bias, activation and residual ------------------------------------------------------------------------------------------
def _linear_fwd(x, weight, bias, activation, residual, keep):
    w = _weight(weight, "linear: weight")
    x2 = _rows(x, w.shape[1], "linear: x")
    M, N = x2.shape[0], w.shape[0]
    shape = x.shape[:-1] + (N,)
    if residual is not None and residual.shape != shape:
        raise MisError(f"linear: residual must have the result's shape {tuple(shape)}, got {tuple(residual.shape)}")
    y = _empty(x2, M, N)
    z = _empty(x2, M, N, dtype=torch.float32) if keep and ops.token_act(activation) else None
    ops.linear_fwd(x2, w, y, bias, activation, None if residual is None else _rows(residual, N, "linear: residual"), z)
    return x2, w, y.view(shape), z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual):
        x2, w, y, z = _linear_fwd(x, weight, bias, activation, residual, True)
        ctx.save_for_backward(x2, w, z)
        ctx.activation, ctx.shape = activation, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = _empty(x, *x.shape) if need[0] else None
        dw = _empty(w, *w.shape) if need[1] else None
        db = _empty(x, w.shape[0], dtype=torch.float32) if need[2] else None
        if need[0] or need[1] or need[2]:
            ops.linear_bwd(_rows(dy, w.shape[0], "dy"), x, w, ctx.activation, z, dx, dw, db)
        return None if dx is None else dx.view(ctx.shape), dw, db, None, dy if need[4] else None


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual; activation None | 'relu' | 'gelu' | 'gelu_tanh' | 'silu' | 'sigmoid', residual with the result's shape"""
    if _grads(x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, activation, residual)
    return _linear_fwd(x, weight, bias, activation, residual, False)[2]


# ---- gated feed-forward block ---------------------------------------------------------------------------------------------------------------
def _gated_fwd(x, w_gate, w_up, b_gate, b_up, activation, keep):
    wg, wu = _pair(_weight(w_gate, "gated_ffn: w_gate"), _weight(w_up, "gated_ffn: w_up"))
    x2 = _rows(x, wg.shape[1], "gated_ffn: x")
    M, F = x2.shape[0], wg.shape[0]
    h = _empty(x2, M, F)
    g, u = (_empty(x2, M, F, dtype=torch.float32), _empty(x2, M, F, dtype=torch.float32)) if keep else (None, None)
    ops.gated_ffn_fwd(x2, wg, wu, h, b_gate, b_up, activation, g, u)
    return x2, wg, wu, h.view(x.shape[:-1] + (F,)), g, u


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation):
        x2, wg, wu, h, g, u = _gated_fwd(x, w_gate, w_up, b_gate, b_up, activation, True)
        ctx.save_for_backward(x2, wg, wu, g, u)
        ctx.activation, ctx.shape = activation, x.shape
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, wg, wu, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        F, K = wg.shape
        dx = _empty(x, *x.shape) if need[0] else None
        dwg, dwu = (_empty(x, F, K), _empty(x, F, K)) if need[1] or need[2] else (None, None)
        dbg = _empty(x, F, dtype=torch.float32) if need[3] else None
        dbu = _empty(x, F, dtype=torch.float32) if need[4] else None
        ops.gated_ffn_bwd(_rows(dh, F, "dh"), x, wg, wu, g, u, ctx.activation, dx, dwg, dwu, dbg, dbu)
        return None if dx is None else dx.view(ctx.shape), dwg if need[1] else None, dwu if need[2] else None, dbg, dbu, None


def gated_ffn(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """activation(x w_gate^T + b_gate) * (x w_up^T + b_up); w_gate, w_up (features, width), activation 'silu' | 'gelu' | 'gelu_tanh' | 'relu' | 'sigmoid' | None"""
    if _grads(x, w_gate, w_up, b_gate, b_up):
        return _GatedFFN.apply(x, w_gate, w_up, b_gate, b_up, activation)
    return _gated_fwd(x, w_gate, w_up, b_gate, b_up, activation, False)[3]
