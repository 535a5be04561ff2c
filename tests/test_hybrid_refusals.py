"""What the dense and state-space entry points refuse, before any CUDA call."""

from __future__ import annotations

import ctypes

import pytest
import torch

from ervf_b200 import GPUKernels, _lib

P = ctypes.addressof(ctypes.create_string_buffer(256)) & ~63
Q = P + 4096


def linear(W=P, x=P, xs=64, b=None, r=None, rs=0, out=Q, os=32, ty=0, rows=32, cols=64, t=4, act=0):
    return _lib.load().ervf_linear_bf16(W, x, xs, b, r, rs, out, os, ty, rows, cols, t, act, None)


def test_linear():
    assert linear(W=None) == linear(x=None) == linear(out=None) == _lib.ERR_NULL
    assert linear(rows=0) == linear(cols=0) == linear(t=-1) == linear(cols=60, xs=64) == _lib.ERR_SHAPE
    assert linear(xs=56) == linear(os=31) == linear(r=P, rs=31) == _lib.ERR_SHAPE
    assert linear(ty=2) == linear(act=4) == linear(act=-1) == linear(out=P) == _lib.ERR_ARG
    assert linear(r=Q, rs=40) == _lib.ERR_ARG
    assert linear(W=P + 2) == linear(x=P + 8) == linear(xs=68) == linear(out=Q + 2) == linear(b=P + 2) == _lib.ERR_ALIGN
    assert linear(t=0, x=None, out=None) == _lib.OK


def test_linear_sizes_that_tiles_cannot_count():
    most, over = 0x7fffff00, 0x7fffff01
    big = dict(xs=2 ** 31, os=2 ** 31)
    assert linear(rows=over, **big) == linear(t=over, **big) == linear(cols=0x7ffffff8, **big) == _lib.ERR_SHAPE
    assert linear(rows=most, t=0, **big) == _lib.OK


def conv(x=P, xs=8, w=P, b=None, st=None, ns=0, sl=None, has=None, cu=P, s=1, out=Q, os=8, ty=0, t=4, ch=8, k=4, silu=1):
    return _lib.load().ervf_conv1d_prompt(x, xs, w, b, st, ns, sl, has, cu, s, out, os, ty, t, ch, k, silu, None)


def test_conv():
    assert conv(x=None) == conv(w=None) == conv(out=None) == _lib.ERR_NULL
    assert conv(t=-1) == conv(ch=0) == conv(k=1) == conv(k=5) == conv(xs=7) == conv(os=7) == _lib.ERR_SHAPE
    assert conv(s=-1) == conv(ns=-1) == _lib.ERR_SHAPE
    assert conv(cu=None, s=2) == conv(ty=3) == conv(silu=2) == conv(out=P) == _lib.ERR_ARG
    assert conv(x=P + 2) == conv(cu=P + 2) == conv(sl=P + 2) == conv(st=P + 2) == _lib.ERR_ALIGN
    assert conv(s=0) == _lib.OK


def scan(x=P, xs=16, dt=P, ds=2, A=P, B=P, bs=8, C=P, cs=8, st=None, ns=0, sl=None, has=None, cu=P, s=1, y=Q, ys=16,
         ty=0, t=4, h=2, p=8, g=1, n=8, scr=None, nb=0):
    return _lib.load().ervf_ssm_prompt(x, xs, dt, ds, A, B, bs, C, cs, None, None, st, ns, sl, has, cu, s, y, ys, ty,
                                       t, h, p, g, n, scr, nb, None)


def test_scan():
    assert scan(x=None) == scan(dt=None) == scan(A=None) == scan(B=None) == scan(C=None) == scan(y=None) == _lib.ERR_NULL
    assert scan(h=0) == scan(g=0) == scan(h=3, g=2) == scan(p=257, xs=999, ys=999) == scan(n=257) == _lib.ERR_SHAPE
    assert scan(xs=15) == scan(ys=15) == scan(ds=1) == scan(bs=7) == scan(cs=7) == scan(t=-1) == _lib.ERR_SHAPE
    assert scan(cu=None, s=2) == scan(ty=2) == scan(y=P) == _lib.ERR_ARG
    assert scan(x=P + 2) == scan(A=P + 2) == scan(st=P + 2) == _lib.ERR_ALIGN
    assert scan(s=0) == _lib.OK


def test_scan_scratch_is_checked():
    dims = (4096, 1, 64, 64, 8, 128)
    need = _lib.load().ervf_ssm_prompt_scratch_bytes(_lib.BF16, *dims)
    big = dict(xs=4096, ys=4096, ds=64, bs=1024, cs=1024, ty=1, t=4096, h=64, p=64, g=8, n=128)
    if need:
        assert scan(**big) == _lib.ERR_NULL
        assert scan(scr=P, nb=need - 1, **big) == _lib.ERR_ARG
        assert scan(scr=P + 4, nb=need, **big) == _lib.ERR_ALIGN
    assert _lib.load().ervf_ssm_prompt_scratch_bytes(7, *dims) == 0
    assert _lib.load().ervf_ssm_prompt_scratch_bytes(_lib.BF16, 4096, 1, 64, 64, 7, 128) == 0


def token(x=P, xs=32, dt=P, ds=2, z=None, zs=0, cw=P, cst=P, A=P, eps=1e-5, st=P, ns=1, sl=None, out=Q, os=16, ty=0,
          s=1, h=2, p=8, g=1, n=8, k=4):
    return _lib.load().ervf_ssm_token(x, xs, dt, ds, z, zs, cw, None, cst, A, None, None, None, eps, st, ns, sl, out,
                                      os, ty, s, h, p, g, n, k, None)


def test_token():
    assert token(x=None) == token(dt=None) == token(cw=None) == token(cst=None) == token(A=None) == _lib.ERR_NULL
    assert token(st=None) == token(out=None) == _lib.ERR_NULL
    assert token(h=3, g=2) == token(n=6) == token(n=260) == token(k=1) == token(k=5) == token(p=300) == _lib.ERR_SHAPE
    assert token(h=129, p=256, xs=40000, os=40000, ds=200) == _lib.ERR_SHAPE
    assert token(xs=31) == token(ds=1) == token(os=15) == token(z=P, zs=15) == token(s=-1) == _lib.ERR_SHAPE
    assert token(ty=2) == token(out=P) == token(eps=-1.0) == token(eps=float("nan")) == _lib.ERR_ARG
    assert token(st=P + 4) == token(x=P + 2) == token(sl=P + 2) == _lib.ERR_ALIGN
    assert token(s=0) == _lib.OK


def norm(y=P, ys=16, z=None, zs=0, w=P, eps=1e-5, out=Q, os=16, ty=0, t=2, g=2, n=8):
    return _lib.load().ervf_gated_norm(y, ys, z, zs, w, eps, out, os, ty, t, g, n, None)


def test_norm():
    assert norm(y=None) == norm(w=None) == norm(out=None) == _lib.ERR_NULL
    assert norm(t=-1) == norm(g=0) == norm(n=0) == norm(ys=15) == norm(os=15) == norm(z=P, zs=15) == _lib.ERR_SHAPE
    assert norm(ty=2) == norm(eps=-1.0) == norm(out=P, os=17) == _lib.ERR_ARG
    assert norm(y=P + 2) == norm(w=P + 2) == _lib.ERR_ALIGN
    assert norm(t=0, y=None, out=None) == _lib.OK


def test_sizes_that_a_grid_or_an_index_cannot_hold():
    wide = 2 ** 33
    assert conv(ch=65535 * 128 + 1, xs=wide, os=wide) == conv(s=2 ** 27) == scan(s=2 ** 27) == _lib.ERR_SHAPE
    assert token(h=2 ** 24, g=2 ** 24, p=256, xs=wide, os=wide, ds=2 ** 24) == _lib.ERR_SHAPE
    assert token(s=2 ** 20, h=2 ** 9, g=2 ** 9, p=1, xs=wide, os=wide, ds=2 ** 9) == _lib.ERR_SHAPE
    assert norm(g=1, n=0x7fffff01, ys=wide, os=wide) == _lib.ERR_SHAPE


@pytest.fixture()
def k():
    return GPUKernels(device="cuda:0")


def test_python_refuses_tensors_of_another_device_type_or_size(k):
    a = torch.zeros(4, 64)
    for call in (lambda: k.linear_bf16(a, a.bfloat16(), a.bfloat16(), 64, 64, 4),
                 lambda: k.gated_norm(a, a, a, a[0], 4, 1, 64),
                 lambda: k.conv1d_prompt(a, a, a, None, None, None, 1, 4, 64, 4),
                 lambda: k.linear_bf16(a.half(), a, a, 64, 64, 4),
                 lambda: k.linear_bf16(P, P, P, 64, 64, 4),          # an address needs dtype
                 lambda: k.linear_bf16(P, P, P, 64, 64, 4, act="swish", dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()
