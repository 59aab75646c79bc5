"""Layer norm, 8-bit checkpoints and the many-class loss reject malformed calls on the host, before any launch."""
import ctypes

import pytest
import torch

from super_gnn_b200 import _cabi
from super_gnn_b200 import supergnn_ops as ops

P = 4096  # a pointer that is never followed
F32, BF16, F16 = 0, 1, 2


def norm_fwd(l, dtype=F32, x=P, ldx=8, pdt=F32, gamma=P, eps=1e-5, y=P, ldy=8, stats=P, codes=None, ldc=0, params=None, n=4, H=8):
    return l.sgnn_layer_norm_forward(dtype, x, ldx, pdt, gamma, None, eps, y, ldy, stats, codes, ldc, params, n, H, None)


def norm_bwd(l, dtype=F32, gy=P, x=P, codes=None, params=None, gg=P, n=4, H=8, ld=8, part=P):
    return l.sgnn_layer_norm_backward(dtype, gy, ld, x, ld, codes, ld, params, P, F32, P, P, ld, gg, P, part, n, H, None)


def nll(l, dtype=F32, x=P, w=P, bdt=F32, bias=P, labels=P, n=4, K=8, C=300, loss=P, gx=None, gw=None, gb=None, ws=None, nb=0,
        ldw=8, inv=1.0, ldg=8):
    return l.sgnn_linear_nll_loss(dtype, x, 8, w, ldw, bdt, bias, labels, None, inv, n, K, C, loss, None, gx, ldg, gw, ldg, gb,
                                  ws, nb, None)


def grad(l, dtype=F32, g=P, codes=P, params=P, n=4, M=8, F=8, ldo=8, out=P, ws=None, nb=0, beta=0.0, ldg=8):
    return l.sgnn_checkpoint_weight_grad(dtype, g, ldg, codes, 8, params, n, M, F, beta, out, ldo, ws, nb, None)


@pytest.mark.parametrize("call,needle", [
    (lambda l: norm_fwd(l, dtype=3), "unknown element type"),
    (lambda l: norm_fwd(l, dtype=BF16, pdt=F16), "gamma and beta"),
    (lambda l: norm_fwd(l, n=-1), "bad size"),
    (lambda l: norm_fwd(l, H=0), "bad size"),
    (lambda l: norm_fwd(l, H=16385, ldx=20000, ldy=20000), "at most 16384"),
    (lambda l: norm_fwd(l, eps=-1.0), "eps"),
    (lambda l: norm_fwd(l, eps=float("nan")), "eps"),
    (lambda l: norm_fwd(l, x=None), "null pointer"),
    (lambda l: norm_fwd(l, stats=None), "null pointer"),
    (lambda l: norm_fwd(l, ldx=7), "leading dimension"),
    (lambda l: norm_fwd(l, codes=P, ldc=8), "belong together"),
    (lambda l: norm_fwd(l, codes=P, ldc=7, params=P), "leading dimension"),
    (lambda l: norm_fwd(l, x=P + 2), "aligned"),
    (lambda l: norm_fwd(l, stats=P + 4), "aligned"),
    (lambda l: norm_bwd(l, codes=P, params=P), "exactly one"),
    (lambda l: norm_bwd(l, x=None), "exactly one"),
    (lambda l: norm_bwd(l, gg=None), "null pointer"),
    (lambda l: norm_bwd(l, part=None), "null pointer"),
    (lambda l: norm_bwd(l, ld=7), "leading dimension"),
    (lambda l: l.sgnn_checkpoint_pack_rows(7, P, 8, P, 8, P, 4, 8, None), "unknown element type"),
    (lambda l: l.sgnn_checkpoint_pack_rows(F32, P, 7, P, 8, P, 4, 8, None), "leading dimension"),
    (lambda l: l.sgnn_checkpoint_pack_rows(F32, P, 8, P, 8, P + 4, 4, 8, None), "aligned"),
    (lambda l: l.sgnn_checkpoint_unpack_rows(None, 8, P, F32, P, 8, 4, 8, None), "null pointer"),
    (lambda l: l.sgnn_checkpoint_unpack_rows(P, 8, P, F32, P, 8, 4, 1 << 30, None), "too large"),
    (lambda l: grad(l, dtype=-1), "unknown element type"),
    (lambda l: grad(l, n=1 << 31), "too large"),
    (lambda l: grad(l, beta=float("nan")), "NaN"),
    (lambda l: grad(l, ldo=7), "bad output"),
    (lambda l: grad(l, g=None), "null pointer"),
    (lambda l: grad(l, ldg=7), "leading dimension"),
    (lambda l: grad(l), "workspace"),
    (lambda l: nll(l, dtype=F16), "fp32 or bf16"),
    (lambda l: nll(l, bdt=BF16), "the bias"),
    (lambda l: nll(l, C=0), "bad size"),
    (lambda l: nll(l, K=16385), "too large"),
    (lambda l: nll(l, inv=float("nan")), "NaN"),
    (lambda l: nll(l, loss=None), "null output"),
    (lambda l: nll(l, gx=P), "belong together"),
    (lambda l: nll(l, gx=P, gw=P, gb=P, bias=None), "belong together"),
    (lambda l: nll(l, gx=P, gw=P, ldg=7), "leading dimension"),
    (lambda l: nll(l, ldw=7), "leading dimension"),
    (lambda l: nll(l, labels=None), "null pointer"),
    (lambda l: nll(l), "workspace"),
])
def test_malformed_calls_are_rejected(call, needle):
    lib = _cabi.lib()
    assert call(lib) != 0
    assert needle in _cabi.last_error(), _cabi.last_error()


def test_workspace_queries():
    lib = _cabi.lib()
    need = ctypes.c_size_t(0)
    assert lib.sgnn_checkpoint_weight_grad_workspace_bytes(F32, 0, 4, 4, ctypes.byref(need)) == 0 and need.value == 0
    assert lib.sgnn_checkpoint_weight_grad_workspace_bytes(F32, 1000, 256, 512, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.sgnn_checkpoint_weight_grad_workspace_bytes(F32, 10, 4, 4, None) == 1
    assert lib.sgnn_linear_nll_workspace_bytes(F32, 10, 16, 300, 0, ctypes.byref(need)) == 0
    loss_only = need.value
    assert lib.sgnn_linear_nll_workspace_bytes(F32, 10, 16, 300, 1, ctypes.byref(need)) == 0 and need.value > loss_only
    assert lib.sgnn_linear_nll_workspace_bytes(F32, 10, 16, 300, 1, None) == 1
    # a full-batch call does not ask for a matrix of n x C
    assert lib.sgnn_linear_nll_workspace_bytes(BF16, 1 << 20, 256, 1 << 17, 1, ctypes.byref(need)) == 0
    assert need.value < (1 << 20) * (1 << 17) // 8


@pytest.mark.parametrize("call", [
    lambda t: ops.layer_norm_forward(t),
    lambda t: ops.layer_norm_backward(t, t, t),
    lambda t: ops.layer_norm_backward_checkpoint(t, t, t, t),
    lambda t: ops.checkpoint_pack_rows(t),
    lambda t: ops.checkpoint_unpack_rows(t.byte(), t),
    lambda t: ops.checkpoint_weight_grad(t, t.byte(), t),
    lambda t: ops.linear_nll_loss(t, t, None, torch.zeros(4, dtype=torch.int64), None, 1.0),
    lambda t: ops.linear_nll_loss_grad(t, t, None, torch.zeros(4, dtype=torch.int64), None, 1.0),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        call(torch.zeros(4, 8))
