"""What the encoder's operators refuse, without a GPU: arguments are checked before anything is launched."""
import ctypes

import pytest
import torch

from spion_b200 import _lib
from spion_b200._lib import SpionError
from spion_b200.quant import quantize_rows
from spion_b200.rmsnorm import rms_norm, rms_norm_e4m3


def test_rows_on_the_cpu_are_refused():
    x, w = torch.randn(4, 8), torch.ones(8)
    for call in (lambda: rms_norm(x, w), lambda: rms_norm(x, w, res=x), lambda: rms_norm_e4m3(x, w), lambda: quantize_rows(x)):
        with pytest.raises(SpionError, match="CUDA"):
            call()


def test_norm_arguments_at_the_c_boundary():
    L, d = _lib.lib, ctypes.c_void_p(4096)
    F32, BF16, F16, E4M3 = _lib.F32, _lib.BF16, _lib.F16, _lib.E4M3

    def forward(x=d, ldx=8, xt=F32, res=None, ldr=0, rt=F32, w=d, wt=F32, s=None, y=d, ldy=8, yt=F32, scale=None, M=4, N=8, norm=1):
        return L.spion_rmsnorm_forward(x, ldx, xt, res, ldr, rt, w, wt, s, y, ldy, yt, scale, None, M, N, 1e-6, norm, None)

    assert forward(M=0) == 0
    assert forward(M=-1) == -1 and forward(N=0) == -1 and forward(xt=E4M3) == -1 and forward(wt=E4M3) == -1
    assert forward(x=None) == -1 and forward(y=None) == -1 and forward(ldy=7) == -1 and forward(ldx=-1) == -1
    assert forward(res=d, ldr=8) == -1                                       # nowhere to put the sum
    assert forward(yt=E4M3) == -1 and forward(scale=d) == -1                 # 8 bits have scales, others none
    assert forward(norm=0) == -1 and forward(norm=0, w=None) == -1           # without a norm: to e4m3 only
    assert forward(xt=BF16, yt=F32) == -5 and forward(xt=BF16, yt=F16) == -5
    assert forward(xt=BF16, res=d, rt=F32, s=d, ldr=8, yt=BF16) == -5

    def backward(s=d, st=F32, dy=d, dt=F32, w=d, rho=d, dx=d, dr=None, rt=F32, dw=d, ws=d, M=4, N=8):
        return L.spion_rmsnorm_backward(s, 8, st, dy, dt, None, w, F32, rho, dx, dr, rt, dw, ws, M, N, None)

    assert backward(M=-1) == -1 and backward(N=0) == -1 and backward(s=None) == -1 and backward(dy=None) == -1 and backward(rho=None) == -1
    assert backward(ws=None) == -1 and backward(w=None) == -1 and backward(dr=d, rt=F32) == -1 and backward(dt=E4M3) == -1
    assert backward(st=BF16, dt=F32) == -5
    assert L.spion_rmsnorm_workspace_floats(0, 8) == 0 and L.spion_rmsnorm_workspace_floats(3, 8) == 24
    assert L.spion_rmsnorm_workspace_floats(10 ** 9, 8) <= 8 * 2048


def test_optimizer_arguments_at_the_c_boundary_and_in_the_module():
    from spion_b200.optim import AdamW, adamw_step, places
    L, d = _lib.lib, ctypes.c_void_p(4096)

    def step(tensors=((4096, 4096, None, 10, 0, 0),), type=_lib.F32, bits=32, m=d, v=d, sm=None, sv=None, steps=d, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0,
             copy_type=_lib.BF16, ws=d):
        table = (_lib.AdamwTensor * len(tensors))(*tensors)
        return L.spion_adamw_step(table, len(tensors), type, bits, m, v, sm, sv, steps, None, lr, b1, b2, eps, wd, -1.0, 0, copy_type, ws, None)

    assert step(tensors=()) == 0
    assert step(bits=16) == -1 and step(m=None) == -1 and step(v=None) == -1 and step(steps=None) == -1 and step(ws=None) == -1 and step(bits=8) == -1 and step(sm=d, sv=d) == -1
    assert step(lr=-1.0) == -1 and step(b1=1.0) == -1 and step(b2=-0.1) == -1 and step(eps=float("nan")) == -1 and step(wd=-1.0) == -1
    assert step(m=ctypes.c_void_p(4100)) == -1
    assert step(tensors=((None, 4096, None, 10, 0, 0),)) == -1 and step(tensors=((4096, None, None, 10, 0, 0),)) == -1
    assert step(tensors=((4096, 4096, None, -1, 0, 0),)) == -1 and step(tensors=((4096, 4096, None, 10, 100, 0),)) == -1
    assert step(tensors=((4096, 4096, 4096, 10, 0, 0),), copy_type=_lib.F32) == -1
    assert step(type=_lib.E4M3) == -5
    w = torch.zeros(3)
    with pytest.raises(SpionError, match="CUDA"):
        adamw_step([w], [w], w, w, w)
    with pytest.raises(SpionError, match="GPU"):
        AdamW([torch.nn.Parameter(w)]).step()
    for bad in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(clip_value=-1.0)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(w)], **bad)
    assert places([torch.zeros(1), torch.zeros(0), torch.zeros(257)]) == ([0, 256, 256], 768)


def test_8_bit_linear_arguments_at_the_c_boundary():
    from spion_b200.quant import Rows8, linear_e4m3
    L, d = _lib.lib, ctypes.c_void_p(4096)

    def linear(x=d, ldx=16, sx=d, w=d, ldw=16, sw=d, bias=None, bt=_lib.F32, y=d, ldy=8, yt=_lib.BF16, T=4, K=10, N=8):
        return L.spion_linear_e4m3(x, ldx, sx, w, ldw, sw, bias, bt, y, ldy, yt, T, K, N, None)

    assert linear(T=0) == 0
    assert linear(T=-1) == -1 and linear(K=0) == -1 and linear(N=0) == -1 and linear(ldy=7) == -1
    assert linear(x=None) == -1 and linear(w=None) == -1 and linear(sx=None) == -1 and linear(sw=None) == -1 and linear(y=None) == -1
    assert linear(ldx=17) == -1 and linear(ldw=24) == -1 and linear(K=17) == -1 and linear(x=ctypes.c_void_p(4097)) == -1
    assert linear(bias=d, bt=_lib.E4M3) == -1 and linear(yt=_lib.E4M3) == -5 and linear(T=2 ** 31) == -2
    x = torch.zeros(3, 16)
    with pytest.raises(SpionError, match="CUDA"):
        linear_e4m3(x, Rows8(x.to(torch.float8_e4m3fn), torch.ones(3)))


def test_states_of_other_algorithms_are_refused():
    from spion_b200.optim import AdamW
    w = torch.nn.Parameter(torch.zeros(3))
    for kw, match in ((dict(amsgrad=True), "amsgrad"), (dict(maximize=True), "maximize")):
        with pytest.raises(ValueError, match=match):
            AdamW([w]).load_state_dict(torch.optim.AdamW([w], **kw).state_dict())
    with pytest.raises(ValueError, match="decoupled"):
        AdamW([w]).load_state_dict(torch.optim.Adam([w], weight_decay=0.1).state_dict())
