"""Token operators on MI355X: the channel-mixing half of a transformer stage, for networks that mix a U-Net level's pixels / voxels as tokens.

    a = layer_norm(x, w, b)
    h = gated_ffn(a, w_gate, w_up)                  # act(a w_gate^T) * (a w_up^T), one kernel
    y = linear(h, w_down, residual=x)               # h w_down^T + x, one kernel

x is (..., width) with any number of leading dimensions, float32 or bfloat16; weights are (out, width) as in nn.Linear, in x's type; biases and norm parameters are float32.  Each
function is differentiable once, in reverse mode (forward and backward are HIP kernels of libmisamd; torch is the allocator and the tape) and keeps what its backward pass needs only when a gradient is
wanted.  Work is enqueued on torch's current stream of x's device; workspaces come from the caching allocator call by call, so streams and captured graphs share none.  Under stream
capture take gradients with torch.autograd.grad, or call the ops.*_bwd functions.  There is no CPU path: a tensor that is not on the GPU raises.

The same kernels without the tape, on caller-owned buffers with any row strides: ops.layernorm_fwd / _bwd, ops.linear_fwd / _bwd, ops.gated_ffn_fwd / _bwd.  (A small call is bound by the
host: the functions here fill the C descriptors directly, with the checks inline.)"""
import ctypes as C

import torch
from torch.autograd import forward_ad as _fw
from torch.autograd.function import once_differentiable

from ._lib import MIS_BF16, MIS_F32, GatedDesc, LinearDesc, MisError, check, load
from .ops import token_act

_F32, _BF16 = torch.float32, torch.bfloat16
_WIDEST = (1 << 31) - 1          # widths are C ints (ctypes would cut a longer one to its low bits)
_FEW = 32          # rows up to which a forward product needs no workspace (misamd.h): single tokens save the question


def _refuse(who, what):
    raise MisError(f"{who}: {what}")


def _say(t):
    return f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)


def _no_width(who, t, name, n):
    if type(n) is not int:          # (torch.jit.trace makes tensors of sizes; it would record the outputs' allocation and lose the kernels)
        _refuse(who, f"cannot be traced: the sizes of {name} are no integers")
    _refuse(who, f"{name} has a width of 2^31 or more: {_say(t)}")


def _unit(t):
    """a matrix with unit stride inside its rows, rows that do not overlap and no negation pending: itself, or a copy"""
    if t.is_neg():
        return t.resolve_neg().contiguous()
    s0, s1 = t.stride()
    return t if (s1 == 1 or t.shape[1] == 1) and (s0 >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def _rows(who, t, width, name="x"):
    """(..., width) -> (rows, width): a view where the strides allow one, else a copy"""
    if not isinstance(t, torch.Tensor) or t.dim() < 1 or t.shape[-1] != width or width < 1:
        _refuse(who, f"{name} must be a (..., {width}) tensor, got {_say(t)}")
    if t.dim() != 2:
        t = t.reshape(t.numel() // width, width)
    return t if width > 1 and t.is_contiguous() else _unit(t)          # (a pending negation, from the imaginary part of a conjugate, leaves only one column contiguous)


def _tokens(who, x, width):
    """x as rows, and the library's code of its type"""
    x2 = _rows(who, x, width)
    if not x2.is_cuda:
        _refuse(who, f"runs on MI355X only: got {_say(x)} (no CPU fallback)")
    dt = x2.dtype
    if dt is not _BF16 and dt is not _F32:
        _refuse(who, f"x must be float32 or bfloat16, got {_say(x)}")
    return x2, MIS_BF16 if dt is _BF16 else MIS_F32


def _weight(who, w, name):
    if not isinstance(w, torch.Tensor) or w.dim() != 2 or w.shape[0] < 1 or w.shape[1] < 1:
        _refuse(who, f"{name} must be an (out, in) matrix, got {_say(w)}")
    return w if w.is_contiguous() and w.shape[1] > 1 else _unit(w)


def _like(who, t, name, x):
    if t.dtype is not x.dtype or t.device != x.device:
        _refuse(who, f"{name} must be {x.dtype} on {x.device} like x, got {_say(t)}")


def _vec(who, v, name, n, x):
    """pointer of a float32 vector of n, None for None"""
    if v is None:
        return None
    if not isinstance(v, torch.Tensor) or v.dtype is not _F32 or v.dim() != 1 or v.shape[0] != n or v.device != x.device or not v.is_contiguous() or (n == 1 and v.is_neg()):
        _refuse(who, f"{name} must be a contiguous ({n},) float32 tensor on {x.device}, got {_say(v)}")
    return v.data_ptr()


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(who, fn, x, *args):
    dev = x.get_device()
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        check(rc, who)


def _scratch(nbytes, x):
    return torch.empty((nbytes,), dtype=torch.uint8, device=x.device) if nbytes else None


def _no_tangents(who, *ts):
    """a forward-mode tangent, which the kernels would drop, is refused"""
    for t in ts:
        if isinstance(t, torch.Tensor) and _fw.unpack_dual(t).tangent is not None:
            _refuse(who, f"differentiable in reverse mode only, got a tensor with a forward-mode tangent: {_say(t)}")


def _wanted(who, *ts):
    """whether a gradient is (what is not a tensor is refused by the forward pass's checks)"""
    if _fw._current_level >= 0:
        _no_tangents(who, *ts)
    if torch.is_grad_enabled():
        for t in ts:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return True
    return False


def _new(t):
    """a contiguous matrix of t's shape and type (empty_like is the cheapest of torch's allocations)"""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _saved(t):
    """a saved matrix as the kernels read it: saved-tensor hooks may hand it back in another layout"""
    return t if t.is_contiguous() else _unit(t)


def _whole(t):
    """... and what is no matrix of rows"""
    return t if t is None or t.is_contiguous() else t.contiguous()


def _once(backward):
    """differentiable once: the plain function, unless a graph of the backward pass itself is asked for (then torch's wrapper, whose outputs refuse a second differentiation)"""
    wrapped = once_differentiable(backward)

    def run(ctx, dy):
        if _fw._current_level >= 0:
            _no_tangents("token operator (backward)", dy)
        return wrapped(ctx, dy) if torch.is_grad_enabled() else backward(ctx, dy)

    return staticmethod(run)


# ---- layer norm ----------------------------------------------------------------------------------------------------------------------------
def _norm_fwd(x, weight, bias, eps, keep):
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        _refuse("layer_norm", f"x must be a (..., width) tensor, got {_say(x)}")
    D = x.shape[-1]
    if type(D) is not int or D > _WIDEST:
        _no_width("layer_norm", x, "x", D)
    x2, code = _tokens("layer_norm", x, D)
    M = x2.shape[0]
    pw, pb = _vec("layer_norm", weight, "weight", D, x2), _vec("layer_norm", bias, "bias", D, x2)
    y = _new(x2)
    st = torch.empty((2, M), dtype=_F32, device=x2.device) if keep else None
    ps = st.data_ptr() if keep else None
    _call("layer_norm", load().mis_layernorm_fwd, x2, code, x2.data_ptr(), _ld(x2), M, D, eps, pw, pb, y.data_ptr(), D, ps, ps + 4 * M if keep else None)
    return x2, y if x.dim() == 2 else y.view(x.shape), st


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2, y, st = _norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, st)
        ctx.shape = x.shape
        return y

    @_once
    def backward(ctx, dy):
        x, weight, st = ctx.saved_tensors
        x, weight, st = _saved(x), _whole(weight), _whole(st)
        M, D = x.shape
        code = MIS_BF16 if x.dtype is _BF16 else MIS_F32
        nx, nw, nb, _ = ctx.needs_input_grad
        dy = _rows("layer_norm (backward)", dy, D, "dy")
        dx = _new(x) if nx else None
        dw = torch.empty_like(weight) if nw else None
        db = torch.empty((D,), dtype=_F32, device=x.device) if nb else None
        lib = load()
        n = lib.mis_layernorm_bwd_workspace_bytes(code, M, D) if nw or nb else 0
        ws, ps = _scratch(n, x), st.data_ptr()
        _call("layer_norm (backward)", lib.mis_layernorm_bwd, x, code, dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), M, D, _ptr(weight), ps, ps + 4 * M, _ptr(dx), D, _ptr(dw), _ptr(db),
              _ptr(ws), n)
        return dx if dx is None or len(ctx.shape) == 2 else dx.view(ctx.shape), dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension; weight, bias (width,) float32 or None"""
    if _wanted("layer_norm", x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm_fwd(x, weight, bias, float(eps), False)[1]


# ---- matrix product with bias, activation and residual ------------------------------------------------------------------------------------------
def _linear_fwd(x, weight, bias, act, residual, keep):
    w = _weight("linear", weight, "weight")
    N, K = w.shape
    if type(K) is not int or (N | K) > _WIDEST:
        _no_width("linear", weight, "weight", K)
    x2, code = _tokens("linear", x, K)
    _like("linear", w, "weight", x2)
    M = x2.shape[0]
    shape = (M, N) if x.dim() == 2 else x.shape[:-1] + (N,)
    pr = ldr = None
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != shape:
            _refuse("linear", f"residual must have the result's shape {tuple(shape)}, got {_say(residual)}")
        r2 = _rows("linear", residual, N, "residual")
        _like("linear", r2, "residual", x2)
        pr, ldr = r2.data_ptr(), _ld(r2)
    pb = _vec("linear", bias, "bias", N, x2)
    y = torch.empty((M, N), dtype=x2.dtype, device=x2.device)
    d = LinearDesc(code, act, M, N, K, x2.data_ptr(), _ld(x2), w.data_ptr(), _ld(w), pb, pr, ldr or 0, y.data_ptr(), N)
    lib = load()
    kept = _scratch(lib.mis_linear_kept_bytes(C.byref(d)), x2) if keep and act else None
    d.kept = _ptr(kept)
    ws = _scratch(lib.mis_linear_fwd_workspace_bytes(C.byref(d)), x2) if M > _FEW else None
    if ws is not None:
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
    _call("linear", lib.mis_linear_fwd, x2, C.byref(d))
    return x2, w, y if x.dim() == 2 else y.view(shape), kept


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        x2, w, y, kept = _linear_fwd(x, weight, bias, act, residual, True)
        ctx.save_for_backward(x2, w, bias, kept)
        ctx.act, ctx.shape = act, x.shape
        return y

    @_once
    def backward(ctx, dy):
        nx, nw, nb, _, nr = ctx.needs_input_grad
        dres = dy if nr else None
        if not (nx or nw or nb):
            return None, None, None, None, dres
        x, w, bias, kept = ctx.saved_tensors
        x, w, kept = _saved(x), _saved(w), _whole(kept)
        M, K = x.shape
        N = w.shape[0]
        d2 = _rows("linear (backward)", dy, N, "dy")
        dx = _new(x) if nx else None
        dw = _new(w) if nw else None
        db = torch.empty_like(bias) if nb else None
        d = LinearDesc(MIS_BF16 if x.dtype is _BF16 else MIS_F32, ctx.act, M, N, K, x.data_ptr(), _ld(x), w.data_ptr(), _ld(w), _ptr(bias), None, 0, None, 0, _ptr(kept),
                       d2.data_ptr(), _ld(d2), _ptr(dx), K, _ptr(dw), K, _ptr(db))
        lib = load()
        ws = _scratch(lib.mis_linear_bwd_workspace_bytes(C.byref(d)), x)
        if ws is not None:
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        _call("linear (backward)", lib.mis_linear_bwd, x, C.byref(d))
        return dx if dx is None or len(ctx.shape) == 2 else dx.view(ctx.shape), dw, db, None, dres


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual; activation None | 'relu' | 'gelu' | 'gelu_tanh' | 'silu' | 'sigmoid', residual with the result's shape"""
    act = token_act(activation)
    if _wanted("linear", x, weight, bias, residual):
        return _Linear.apply(x, weight, bias, act, residual)
    return _linear_fwd(x, weight, bias, act, residual, False)[2]


# ---- gated feed-forward block ---------------------------------------------------------------------------------------------------------------
def _gated_fwd(x, w_gate, w_up, b_gate, b_up, act, keep):
    wg, wu = _weight("gated_ffn", w_gate, "w_gate"), _weight("gated_ffn", w_up, "w_up")
    F, K = wg.shape
    if type(K) is not int or (F | K) > _WIDEST:
        _no_width("gated_ffn", w_gate, "w_gate", K)
    if wu.shape != wg.shape:
        _refuse("gated_ffn", f"w_gate and w_up must have one shape, got {_say(w_gate)} and {_say(w_up)}")
    if F > 1 and wg.stride(0) != wu.stride(0):
        wg, wu = wg.contiguous(), wu.contiguous()
    x2, code = _tokens("gated_ffn", x, K)
    _like("gated_ffn", wg, "w_gate", x2)
    _like("gated_ffn", wu, "w_up", x2)
    M = x2.shape[0]
    pg, pu = _vec("gated_ffn", b_gate, "b_gate", F, x2), _vec("gated_ffn", b_up, "b_up", F, x2)
    h = torch.empty((M, F), dtype=x2.dtype, device=x2.device)
    d = GatedDesc(code, act, M, F, K, x2.data_ptr(), _ld(x2), wg.data_ptr(), wu.data_ptr(), _ld(wg), pg, pu, h.data_ptr(), F)
    lib = load()
    kept = _scratch(lib.mis_gated_ffn_kept_bytes(C.byref(d)), x2) if keep else None
    d.kept = _ptr(kept)
    ws = _scratch(lib.mis_gated_ffn_fwd_workspace_bytes(C.byref(d)), x2) if M > _FEW else None
    if ws is not None:
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
    _call("gated_ffn", lib.mis_gated_ffn_fwd, x2, C.byref(d))
    return x2, wg, wu, h if x.dim() == 2 else h.view(x.shape[:-1] + (F,)), kept


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        x2, wg, wu, h, kept = _gated_fwd(x, w_gate, w_up, b_gate, b_up, act, True)
        ctx.save_for_backward(x2, wg, wu, b_gate, b_up, kept)
        ctx.act, ctx.shape = act, x.shape
        return h

    @_once
    def backward(ctx, dh):
        x, wg, wu, bg, bu, kept = ctx.saved_tensors
        x, wg, wu, kept = _saved(x), _saved(wg), _saved(wu), _whole(kept)
        if _ld(wg) != _ld(wu):
            wg, wu = wg.contiguous(), wu.contiguous()
        nx, ng, nu, nbg, nbu, _ = ctx.needs_input_grad
        M, K = x.shape
        F = wg.shape[0]
        d2 = _rows("gated_ffn (backward)", dh, F, "dh")
        dx = _new(x) if nx else None
        dwg, dwu = (_new(wg), _new(wu)) if ng or nu else (None, None)
        dbg = torch.empty_like(bg) if nbg else None
        dbu = torch.empty_like(bu) if nbu else None
        d = GatedDesc(MIS_BF16 if x.dtype is _BF16 else MIS_F32, ctx.act, M, F, K, x.data_ptr(), _ld(x), wg.data_ptr(), wu.data_ptr(), _ld(wg), _ptr(bg), _ptr(bu), None, 0, _ptr(kept),
                      d2.data_ptr(), _ld(d2), _ptr(dx), K, _ptr(dwg), _ptr(dwu), K, _ptr(dbg), _ptr(dbu))
        lib = load()
        ws = _scratch(lib.mis_gated_ffn_bwd_workspace_bytes(C.byref(d)), x)
        if ws is not None:
            d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel()
        _call("gated_ffn (backward)", lib.mis_gated_ffn_bwd, x, C.byref(d))
        return dx if dx is None or len(ctx.shape) == 2 else dx.view(ctx.shape), dwg if ng else None, dwu if nu else None, dbg, dbu, None


def gated_ffn(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """activation(x w_gate^T + b_gate) * (x w_up^T + b_up); w_gate, w_up (features, width), activation 'silu' | 'gelu' | 'gelu_tanh' | 'relu' | 'sigmoid' | None"""
    act = token_act(activation)
    if _wanted("gated_ffn", x, w_gate, w_up, b_gate, b_up):
        return _GatedFFN.apply(x, w_gate, w_up, b_gate, b_up, act)
    return _gated_fwd(x, w_gate, w_up, b_gate, b_up, act, False)[3]
