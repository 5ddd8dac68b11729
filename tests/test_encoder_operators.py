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
