"""Refusals of the 8-bit activation operators, without a GPU: the C entry points check before any
launch, the Python ones before the library."""

from __future__ import annotations

import pytest
import torch

A, B, C, D = 0x10000, 0x40000000, 0x80000000, 0xC0000000  # addresses that are never followed


def _refused(pkg, rc, words):
    assert rc == pkg._lib.MOE_EINVAL
    assert words in pkg._lib.load().moe_last_error(), pkg._lib.load().moe_last_error()


def test_quantize_rows_refusals(pkg):
    f = pkg._lib.load().moe_quantize_rows
    for n in (0, -8, 12, 8200):
        _refused(pkg, f(A, 4, n, B, C, None), b"multiple of 8")
    _refused(pkg, f(A, -1, 64, B, C, None), b"multiple of 8")
    _refused(pkg, f(None, 4, 64, B, C, None), b"null")
    _refused(pkg, f(A, 4, 64, None, C, None), b"null")
    _refused(pkg, f(A, 4, 64, B, None, None), b"null")
    _refused(pkg, f(A + 8, 4, 64, B, C, None), b"aligned")
    _refused(pkg, f(A, 4, 64, B + 4, C, None), b"aligned")
    _refused(pkg, f(A, 4, 64, A + 256, C, None), b"overlap")
    _refused(pkg, f(A, 4, 64, B, B + 252, None), b"overlap")
    _refused(pkg, f(A, 2**26, 64, B, C, None), b"rows")
    assert f(None, 0, 64, None, None, None) == 0


def test_add_rms_fp8_refusals(pkg):
    f = pkg._lib.load().moe_add_rmsnorm_fp8
    _refused(pkg, f(A, None, B, 4, 60, 1e-6, None, C, D, None, None), b"multiple of 8")
    _refused(pkg, f(A, None, B, 4, 64, -1.0, None, C, D, None, None), b"eps")
    _refused(pkg, f(A, None, B, 4, 64, float("nan"), None, C, D, None, None), b"eps")
    _refused(pkg, f(A, B, B, 4, 64, 1e-6, None, C, D, None, None), b"null")
    _refused(pkg, f(A, None, None, 4, 64, 1e-6, None, C, D, None, None), b"null")
    _refused(pkg, f(A, None, B + 2, 4, 64, 1e-6, None, C, D, None, None), b"aligned")
    _refused(pkg, f(A, None, B, 4, 64, 1e-6, None, A, D, None, None), b"overlap")
    _refused(pkg, f(A, None, B, 4, 64, 1e-6, None, C, D, C + 128, None), b"overlap")
    assert f(None, None, None, 0, 64, 1e-6, None, None, None, None, None) == 0


def test_linear_refusals(pkg):
    f = pkg._lib.load().moe_linear

    def call(x=A, ldx=64, xs=None, w=B, ldw=64, ws=None, dtype=0, M=4, K=64, N=8, bias=None, f32=0, act=0,
             mul=None, res=None, out=C):
        return f(x, ldx, xs, w, ldw, ws, dtype, M, K, N, bias, f32, act, mul, res, out, None)

    _refused(pkg, call(dtype=2), b"dtype")
    _refused(pkg, call(M=-1), b">= 0")
    _refused(pkg, call(N=-1), b">= 0")
    for K in (0, 4, 12, -8):
        _refused(pkg, call(K=K), b"multiple of 8")
    for K in (0, 8, 24):
        _refused(pkg, call(K=K, dtype=1, xs=D, ws=D), b"multiple of 16")
    for act in (-1, 5):
        _refused(pkg, call(act=act), b"activation")
    _refused(pkg, call(x=None), b"null")
    _refused(pkg, call(out=None), b"null")
    _refused(pkg, call(xs=D), b"scale")
    _refused(pkg, call(ws=D), b"scale")
    _refused(pkg, call(dtype=1, xs=D), b"scale")
    _refused(pkg, call(ldx=56), b"ldx")
    _refused(pkg, call(ldw=68), b"ldw")
    _refused(pkg, call(x=A + 8), b"16 bytes")
    _refused(pkg, call(w=B + 2), b"16 bytes")
    _refused(pkg, call(out=C + 4), b"aligned")
    _refused(pkg, call(res=D + 2), b"aligned")
    _refused(pkg, call(bias=D + 2, f32=1), b"aligned")
    _refused(pkg, call(out=A), b"overlap")
    _refused(pkg, call(res=C + 8), b"overlap")
    _refused(pkg, call(N=2**31 - 1), b"M and N")
    _refused(pkg, call(M=2**31 - 512), b"M and N")
    assert call(M=0, x=None) == 0 and call(N=0, w=None) == 0


def test_experts_fp8_refusals(pkg):
    lib = pkg._lib.load()
    f = lib.moe_experts_fp8_forward
    need = lib.moe_experts_fp8_workspace_bytes(4, 64, 8, 2, 32)
    assert 0 < need < lib.moe_experts_fp8_workspace_bytes(400, 64, 8, 2, 32)
    assert lib.moe_experts_fp8_workspace_bytes(-1, 64, 8, 2, 32) == 0

    def call(q=A, xs=B, T=4, H=64, E=8, k=2, I=32, idx=B, wts=B, gu=B, gus=B, dn=B, dns=B, out=C, ws=D, n=need,
             sh=None, gate=None, ld=1, res=None):
        return f(q, xs, T, H, E, k, I, idx, wts, gu, gus, dn, dns, sh, gate, ld, res, out, ws, n, None)

    _refused(pkg, call(H=40), b"hidden")
    _refused(pkg, call(I=48), b"intermediate")
    _refused(pkg, call(E=1025), b"experts")
    _refused(pkg, call(k=9), b"top_k")
    _refused(pkg, call(T=-1), b"T must")
    _refused(pkg, call(T=1 << 30), b"too many")
    for name in ("q", "xs", "idx", "wts", "gu", "gus", "dn", "dns", "out"):
        _refused(pkg, call(**{name: None}), b"null")
    _refused(pkg, call(q=A + 8), b"aligned")
    _refused(pkg, call(n=need - 1), b"workspace")
    _refused(pkg, call(ws=None), b"workspace")
    _refused(pkg, call(sh=B), b"gate")
    _refused(pkg, call(sh=B, gate=B, ld=-1), b"gate")
    _refused(pkg, call(sh=B + 4, gate=B), b"aligned")
    _refused(pkg, call(res=B + 8), b"aligned")
    _refused(pkg, call(res=C), b"overlap")
    _refused(pkg, call(sh=C + 64, gate=B), b"overlap")
    for name in ("q", "gu", "dn"):
        _refused(pkg, call(**{name: D + 64}), b"overlap")
    _refused(pkg, call(out=D + 128), b"overlap")
    assert call(T=0, q=None) == 0


def test_cpu_tensors_fail_loudly(pkg):
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    q, s = torch.zeros(2, 64).to(torch.float8_e4m3fn), torch.ones(2)
    for call in (lambda: pkg.ops.quantize_rows(x), lambda: pkg.ops.add_rms_fp8(x, None, w, 1e-6),
                 lambda: pkg.ops.linear(x, x), lambda: pkg.ops.experts_fp8(
                     q, s, None, None, None, None, gate_up_scale=None, down_scale=None)):
        with pytest.raises(pkg.MoeLibraryError, match="no CPU path"):
            call()
