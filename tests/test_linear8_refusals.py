"""What the entry points of the 8-bit linear layer refuse.  Arguments are checked before a device is looked for, so this runs
without one; the addresses are never read."""
import ctypes

import pytest

from nncv_b200 import _lib
from nncv_b200._lib import BF16, E4M3, F16, F32, lib

EINVAL = 1
P = 1 << 20   # an address on every boundary


def norm(x=P, ldx=0, res=2 * P, w=3 * P, eps=1e-6, sum_=4 * P, out=5 * P, out_dt=E4M3, scale=6 * P, dt=BF16, m=4, k=256):
    return lib().nncv_b200_rmsnorm(x, ldx, res, w, eps, sum_, out, out_dt, scale, dt, m, k, None)


def gated(gate=P, up=2 * P, ld=0, out=3 * P, out_dt=E4M3, scale=4 * P, dt=BF16, m=4, k=256, act=5):
    return lib().nncv_b200_gated_activation(gate, up, ld, out, out_dt, scale, dt, m, k, act, None)


def quantize(x=P, ldx=0, dt=BF16, q=2 * P, scale=3 * P, m=4, k=256, rows=1):
    return lib().nncv_b200_quantize_e4m3(x, ldx, dt, q, scale, m, k, rows, None)


def matmul(a=P, sa=2 * P, b=3 * P, sb=4 * P, c=5 * P, m=4, n=8, k=256, cdt=BF16, bias=6 * P, relu=0):
    return lib().nncv_b200_matmul_e4m3(a, sa, b, sb, c, m, n, k, cdt, bias, relu, None)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(m=-1), dict(k=0), dict(k=-8), dict(dt=3), dict(dt=-1), dict(eps=-1e-6), dict(eps=float("nan")),
    dict(ldx=255), dict(ldx=-1), dict(m=1 << 30, k=1 << 10), dict(m=1, k=(1 << 30) + 16), dict(out_dt=F16, scale=None), dict(out_dt=4), dict(scale=None), dict(out_dt=BF16), dict(x=P + 1), dict(res=P + 1),
    dict(sum_=P + 1), dict(w=P + 2), dict(scale=P + 2), dict(dt=F32, x=P + 2), dict(out_dt=BF16, scale=None, out=P + 1),
    dict(sum_=P, ldx=264), dict(out=4 * P), dict(out=P), dict(out=2 * P), dict(out=P, ldx=264, out_dt=BF16, scale=None)])
def test_rmsnorm_refuses(bad):
    assert norm(**bad) == EINVAL and b"rmsnorm" in lib().nncv_b200_last_error()


@pytest.mark.parametrize("bad", [
    dict(gate=None), dict(out=None), dict(m=-1), dict(k=0), dict(dt=3), dict(act=6), dict(act=-1), dict(ld=255), dict(m=1 << 30, k=1 << 10), dict(m=1, k=(1 << 30) + 16), dict(out_dt=F32, scale=None),
    dict(scale=None), dict(out_dt=BF16), dict(gate=P + 1), dict(up=P + 1), dict(scale=P + 1), dict(out=P), dict(out=2 * P),
    dict(out=P, out_dt=BF16, scale=None, ld=512)])
def test_gated_activation_refuses(bad):
    assert gated(**bad) == EINVAL and b"gated_activation" in lib().nncv_b200_last_error()


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(q=None), dict(scale=None), dict(m=-1), dict(k=0), dict(dt=3), dict(ldx=100), dict(m=1 << 30, k=1 << 10), dict(m=1, k=(1 << 30) + 16), dict(m=1 << 30, k=1 << 10, rows=128), dict(rows=0), dict(rows=64), dict(rows=256),
    dict(x=P + 1), dict(scale=P + 2), dict(q=P)])
def test_quantize_refuses(bad):
    assert quantize(**bad) == EINVAL and b"quantize_e4m3" in lib().nncv_b200_last_error()


@pytest.mark.parametrize("bad", [
    dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(c=None), dict(m=-1), dict(n=0), dict(k=0), dict(k=8), dict(k=250), dict(cdt=3),
    dict(cdt=-1), dict(a=P + 8), dict(b=P + 1), dict(c=P + 1), dict(cdt=F32, c=P + 2), dict(sa=P + 2), dict(sb=P + 1), dict(bias=P + 2), dict(m=1 << 30, n=1 << 20), dict(m=(1 << 30) + 1), dict(n=(1 << 30) + 1), dict(k=(1 << 30) + 16)])
def test_matmul_refuses(bad):
    assert matmul(**bad) == EINVAL and b"matmul_e4m3" in lib().nncv_b200_last_error()


def test_without_a_device_they_fail_loudly():
    import torch
    if torch.cuda.is_available():
        pytest.skip("checks the no-GPU behaviour")
    for call in (norm, gated, quantize, matmul):
        assert call() == 3 and b"no CPU fallback" in lib().nncv_b200_last_error()
        assert call(m=0) == 3
    assert ctypes.sizeof(ctypes.c_void_p) == 8 and _lib.E4M3 == 3 and F16 == 1
