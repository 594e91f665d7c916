"""Token operators without a GPU: what the Python and the C entries refuse, and the oracle against torch's own differentiation in 64 bits."""
import ctypes as C

import pytest
import torch

from mdeical_image_segmentation_amd import _lib, ops, tokens
from mdeical_image_segmentation_amd._lib import MisError
from oracle import tokens_oracle as O


def test_cpu_tensors_are_refused():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    for call in (lambda: tokens.layer_norm(x), lambda: tokens.linear(x, w), lambda: tokens.gated_ffn(x, w, w), lambda: ops.layernorm_fwd(x, x), lambda: ops.linear_fwd(x, w, x)):
        with pytest.raises(MisError, match="MI355X"):
            call()


@pytest.mark.parametrize("call", [
    lambda x, w: tokens.linear(x, w[:, :7]), lambda x, w: tokens.linear(x, w[0]), lambda x, w: tokens.linear(x, w, residual=x), lambda x, w: tokens.gated_ffn(x[..., :0], w, w),
    lambda x, w: tokens.linear(torch.tensor(1.0), w), lambda x, w: ops.token_act("swish"), lambda x, w: ops.token_act(["gelu"])])
def test_wrong_shapes_and_names_are_refused(call):
    with pytest.raises(MisError):
        call(torch.randn(4, 8), torch.randn(6, 8))


@pytest.mark.parametrize("call", [
    lambda x, w: tokens.layer_norm(3.0), lambda x, w: tokens.linear([1.0], w), lambda x, w: tokens.linear(x, 2), lambda x, w: tokens.gated_ffn(x, w, None), lambda x, w: tokens.gated_ffn(None, w, w),
    lambda x, w: ops.linear_fwd("x", w, w), lambda x, w: ops.layernorm_bwd(x, None, x, x)])
def test_what_is_no_tensor_is_refused(call):
    with pytest.raises(MisError):
        call(torch.randn(4, 8, requires_grad=True), torch.randn(6, 8))


@pytest.mark.parametrize("M", [1 << 31, (1 << 40) - 1])
def test_more_rows_than_an_int_holds_are_refused(M):
    lib = _lib.load()
    for d, f in ((_lin(M=M, N=1, K=1), lib.mis_linear_fwd), (_lin(M=M, N=1, K=1), lib.mis_linear_bwd), (_gat(M=M, F=1, K=1), lib.mis_gated_ffn_fwd), (_gat(M=M, F=1, K=1), lib.mis_gated_ffn_bwd)):
        assert f(C.byref(d), None) < 0 and b"too many" in lib.mis_last_error()


def _lin(**kw):
    d = _lib.LinearDesc()
    d.dtype, d.M, d.N, d.K = _lib.MIS_F32, 4, 6, 8
    d.ldx = d.ldw = d.lddx = d.lddw = 8
    d.ldy = d.lddy = d.ldres = 6
    d.x = d.w = d.y = d.dy = d.kept = d.dx = 4096          # never reached: each call below is refused before a launch
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _gat(**kw):
    d = _lib.GatedDesc()
    d.dtype, d.act, d.M, d.F, d.K = _lib.MIS_BF16, 4, 4, 6, 8
    d.ldx = d.ldw = d.lddx = d.lddw = 8
    d.ldh = d.lddh = 6
    d.x = d.wg = d.wu = d.h = d.dh = d.kept = d.dx = 4096
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw, word", [({"dtype": 2}, b"dtype"), ({"act": 6}, b"activation"), ({"act": -1}, b"activation"), ({"M": -1}, b"rows"), ({"N": 0}, b"width"), ({"K": 0}, b"width"),
                                      ({"x": None}, b"null"), ({"w": None}, b"null"), ({"y": None}, b"null"), ({"ldx": 7}, b"stride"), ({"ldw": 7}, b"stride"), ({"ldy": 5}, b"stride"),
                                      ({"kept": 4100}, b"aligned"), ({"res": 4096, "ldres": 5}, b"stride"), ({"M": 1 << 60}, b"too many")])
def test_linear_fwd_refuses(kw, word):
    lib = _lib.load()
    assert lib.mis_linear_fwd(C.byref(_lin(**kw)), None) < 0
    assert word in lib.mis_last_error()


@pytest.mark.parametrize("kw, word", [({"dtype": 9}, b"dtype"), ({"dy": None}, b"null"), ({"lddy": 5}, b"stride"), ({"lddx": 7}, b"stride"), ({"dw": 4096, "lddw": 7}, b"stride"),
                                      ({"dw": 4096, "x": None}, b"null"), ({"act": 2, "kept": None}, b"keeps"), ({"act": 2, "kept": 4104}, b"aligned"), ({"dtype": 1, "act": 2, "dbias": 4096}, b"without"), ({"act": 2}, b"workspace"), ({"dbias": 4096}, b"workspace"),
                                      ({"act": 2, "workspace": 4096, "workspace_bytes": 64}, b"workspace")])
def test_linear_bwd_refuses(kw, word):
    lib = _lib.load()
    assert lib.mis_linear_bwd(C.byref(_lin(**kw)), None) < 0
    assert word in lib.mis_last_error()


@pytest.mark.parametrize("kw, word", [({"dtype": 2}, b"dtype"), ({"act": 9}, b"activation"), ({"F": 0}, b"width"), ({"wu": None}, b"null"), ({"h": None}, b"null"), ({"ldh": 5}, b"stride"),
                                      ({"kept": 4104}, b"aligned")])
def test_gated_fwd_refuses(kw, word):
    lib = _lib.load()
    assert lib.mis_gated_ffn_fwd(C.byref(_gat(**kw)), None) < 0
    assert word in lib.mis_last_error()


@pytest.mark.parametrize("kw, word", [({"dh": None}, b"null"), ({"kept": None}, b"keeps"), ({"kept": 4104}, b"aligned"), ({"dbg": 4096}, b"without"), ({"dwg": 4096}, b"together"), ({"lddh": 5}, b"stride"), ({}, b"workspace")])
def test_gated_bwd_refuses(kw, word):
    lib = _lib.load()
    assert lib.mis_gated_ffn_bwd(C.byref(_gat(**kw)), None) < 0
    assert word in lib.mis_last_error()


def test_layernorm_refuses():
    lib = _lib.load()
    p = 4096
    assert lib.mis_layernorm_fwd(5, p, 8, 4, 8, 1e-5, None, None, p, 8, None, None, None) < 0 and b"dtype" in lib.mis_last_error()
    assert lib.mis_layernorm_fwd(0, p, 8, 4, 0, 1e-5, None, None, p, 8, None, None, None) < 0 and b"width" in lib.mis_last_error()
    assert lib.mis_layernorm_fwd(0, p, 7, 4, 8, 1e-5, None, None, p, 8, None, None, None) < 0 and b"stride" in lib.mis_last_error()
    assert lib.mis_layernorm_fwd(0, None, 8, 4, 8, 1e-5, None, None, p, 8, None, None, None) < 0 and b"null" in lib.mis_last_error()
    assert lib.mis_layernorm_fwd(0, p, 8, 1 << 40, 8, 1e-5, None, None, p, 8, None, None, None) < 0 and b"grid" in lib.mis_last_error()
    assert lib.mis_layernorm_fwd(0, p, 1 << 23, 4, 1 << 23, 1e-5, None, None, p, 1 << 23, None, None, None) < 0 and b"2^22" in lib.mis_last_error()
    assert lib.mis_layernorm_bwd(0, p, 8, p, 8, 4, 8, None, p, None, p, 8, p, p, p, 1 << 20, None) < 0 and b"null" in lib.mis_last_error()
    assert lib.mis_layernorm_bwd(0, p, 8, p, 8, 4, 8, None, p, p, p, 8, p, p, p, 16, None) < 0 and b"workspace" in lib.mis_last_error()


def test_null_descriptors_are_refused():
    lib = _lib.load()
    for f in (lib.mis_linear_fwd, lib.mis_linear_bwd, lib.mis_gated_ffn_fwd, lib.mis_gated_ffn_bwd):
        assert f(None, None) < 0 and b"null" in lib.mis_last_error()
    assert lib.mis_linear_bwd_workspace_bytes(None) == 0 and lib.mis_gated_ffn_bwd_workspace_bytes(None) == 0


def test_forward_workspaces():
    lib = _lib.load()
    assert lib.mis_linear_fwd_workspace_bytes(None) == 0 and lib.mis_gated_ffn_fwd_workspace_bytes(None) == 0
    for M, some in ((1, False), (32, False), (33, True), (100, True), (0, False)):          # few tiles and 128 steps: cut along the width, but not where the rows are few enough for the weights' kernel
        assert (lib.mis_linear_fwd_workspace_bytes(C.byref(_lin(M=M, N=256, K=8192))) > 0) == some
        assert (lib.mis_gated_ffn_fwd_workspace_bytes(C.byref(_gat(M=M, F=256, K=8192))) > 0) == some
    assert lib.mis_linear_fwd_workspace_bytes(C.byref(_lin(M=16384, N=8192, K=512))) == 0          # enough tiles
    assert lib.mis_linear_fwd_workspace_bytes(C.byref(_lin(M=100, N=256, K=0))) == 0


def test_empty_batches_are_no_error():
    lib = _lib.load()
    assert lib.mis_linear_fwd(C.byref(_lin(M=0)), None) == 0
    assert lib.mis_gated_ffn_fwd(C.byref(_gat(M=0)), None) == 0
    assert lib.mis_layernorm_fwd(0, None, 8, 0, 8, 1e-5, None, None, None, 8, None, None, None) == 0


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
def test_oracle_gradients_are_torchs(name):
    g = torch.Generator().manual_seed(5)
    x, w, v, b, c, r, dy = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((7, 5), (6, 5), (6, 5), (6,), (6,), (7, 6), (7, 6)))
    f = {"none": lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"),
         "silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid}[name]
    y = f(x @ w.t() + b) + r
    o = O.linear(x, w, b, name, r, dy)
    for got, want in zip((y, *torch.autograd.grad(y, (x, w, b), dy.detach())), (o["y"], o["dx"], o["dw"], o["db"])):
        torch.testing.assert_close(want[0], got.detach(), rtol=1e-12, atol=1e-12)
    y = f(x @ w.t() + b) * (x @ v.t() + c)
    o = O.gated(x, w, v, b, c, name, dy)
    for got, want in zip((y, *torch.autograd.grad(y, (x, w, v, b, c), dy.detach())), (o["y"], o["dx"], o["dwg"], o["dwu"], o["dbg"], o["dbu"])):
        torch.testing.assert_close(want[0], got.detach(), rtol=1e-12, atol=1e-12)
    gam, bet = w[:, 0].detach().clone().requires_grad_(), b
    dz = torch.randn(7, 6, generator=g, dtype=torch.float64)
    y = torch.nn.functional.layer_norm(r, (6,), gam, bet, 1e-5)
    o = O.layer_norm(r, gam, bet, 1e-5, dz)
    for got, want in zip((y, *torch.autograd.grad(y, (r, gam, bet), dz)), (o["y"], o["dx"], o["dw"], o["db"])):
        torch.testing.assert_close(want[0], got.detach(), rtol=1e-12, atol=1e-12)


# a tangent would vanish behind the data pointers: refused, with gradients on or off, for every argument that may carry one
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call", [
    lambda x, w, b, d: tokens.layer_norm(d(x)), lambda x, w, b, d: tokens.layer_norm(x, d(x[0])), lambda x, w, b, d: tokens.layer_norm(x, None, d(x[0])), lambda x, w, b, d: tokens.linear(d(x), w),
    lambda x, w, b, d: tokens.linear(x, d(w)), lambda x, w, b, d: tokens.linear(x, w, d(b)), lambda x, w, b, d: tokens.linear(x, w, residual=d(x @ w.t())), lambda x, w, b, d: tokens.gated_ffn(d(x), w, w),
    lambda x, w, b, d: tokens.gated_ffn(x, d(w), w), lambda x, w, b, d: tokens.gated_ffn(x, w, d(w)), lambda x, w, b, d: tokens.gated_ffn(x, w, w, d(b)), lambda x, w, b, d: tokens.gated_ffn(x, w, w, None, d(b))])
def test_forward_mode_tangents_are_refused(call, grad):
    import torch.autograd.forward_ad as fw
    x, w, b = torch.randn(4, 8), torch.randn(6, 8), torch.randn(6)
    with torch.set_grad_enabled(grad), fw.dual_level():
        with pytest.raises(MisError, match="tangent"):
            call(x, w, b, lambda t: fw.make_dual(t, torch.ones_like(t)))
        with pytest.raises(MisError, match="MI355X"):           # without one: the ordinary checks
            call(x, w, b, lambda t: t)


def test_jvp_of_a_token_operator_is_refused():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    with pytest.raises(MisError, match="tangent"):
        torch.func.jvp(lambda t: tokens.linear(t, w), (x,), (torch.ones_like(x),))


# the C descriptors hold widths in 32 bits, and ctypes would cut a longer one to its low bits
@pytest.mark.parametrize("call", [
    lambda t: tokens.layer_norm(t(2, 1 << 32 | 64)), lambda t: tokens.linear(t(2, 1 << 32 | 64), t(4, 1 << 32 | 64)), lambda t: tokens.linear(t(2, 8), t(1 << 32 | 4, 8)),
    lambda t: tokens.gated_ffn(t(2, 1 << 31), t(4, 1 << 31), t(4, 1 << 31)), lambda t: tokens.gated_ffn(t(2, 8), t(1 << 32 | 4, 8), t(1 << 32 | 4, 8))])
def test_widths_that_an_int_does_not_hold_are_refused(call):
    with pytest.raises(MisError, match="2\\^31"):
        call(lambda *shape: torch.empty(*shape, device="meta"))


def test_rows_with_a_pending_negation_are_resolved():
    # the imaginary part of a conjugate is a view whose sign torch flips when it reads it; one column of it has rows that look like the kernels' own
    z = torch.complex(torch.randn(5, 1), torch.randn(5, 1)).conj().imag
    assert z.is_neg()
    for t in (z, z[:1]):
        r = tokens._rows("test", t, 1)
        assert not r.is_neg() and torch.equal(r, t)
        w = tokens._weight("test", t, "weight")
        assert not w.is_neg() and torch.equal(w, t)
    with pytest.raises(MisError, match="bias"):
        tokens._vec("test", z[0], "bias", 1, z)


# a trace would record the outputs' allocation and lose the kernels
@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    for f in (lambda t: tokens.layer_norm(t), lambda t: tokens.linear(t, w), lambda t: tokens.gated_ffn(t, w, w)):
        with pytest.raises(MisError, match="traced"):
            torch.jit.trace(f, (x,), check_trace=False)
