"""Rows in 8 bits (ops.quantize_rows, ops.add_rms_fp8): values and scales against torch and
against 64 bits, non-finite and empty rows, views, streams, graphs."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16

pytestmark = pytest.mark.gpu

EPS = 1e-6
SHAPES = [(1, 8), (1, 512), (3, 40), (4, 520), (5, 1000), (130, 2048), (7, 4096), (2, 8192), (1, 8192)]


def _bytes(q):
    return q.cpu().view(torch.uint8)


@pytest.mark.parametrize("T,n", SHAPES)
def test_quantize_rows_is_torchs_division_and_rounding(pkg, dev, T, n):
    x = torch.randn(T, n, generator=torch.Generator().manual_seed(T + n)).to(BF16)
    x[0] = torch.arange(n).remainder(97).to(BF16) * 17  # many quotients midway between two values
    q, s = pkg.ops.quantize_rows(x.to(dev))
    want, ws = ref.rows(x)
    assert q.dtype == ref.FP8 and q.shape == x.shape and s.shape == (T,)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(_bytes(q), _bytes(want))


def test_quantize_rows_zero_tiny_huge_and_non_finite(pkg, dev):
    x = torch.randn(8, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    x[1] = 0
    x[2] *= 2.0**-130  # below the smallest amax
    x[3] = torch.where(x[3] > 0, 3.0e38, -3.3e38).to(BF16)
    x[4, 5], x[4, 9] = float("nan"), float("inf")
    x[5, 0] = float("-inf")
    x[6] = float("nan")
    x[7] = -0.0
    q, s = pkg.ops.quantize_rows(x.to(dev))
    q, s, f = q.float().cpu(), s.cpu(), x.float()
    fine = torch.isfinite(f)
    assert torch.equal(torch.isnan(q), ~fine)
    amax = torch.where(fine, f.abs(), 0).amax(-1)
    want = torch.where(amax > 0, amax.clamp_min(2.0**-100) / 448.0, 1.0)
    assert torch.equal(s, want)
    clean = torch.where(fine, f, 0)
    assert torch.equal(torch.where(fine, q, 0), (clean / want[:, None]).to(ref.FP8).float())
    assert torch.equal(q[1], torch.zeros(64)) and s[1] == 1 and s[6] == 1 and s[7] == 1


def test_quantize_rows_views_and_empty(pkg, dev):
    x = torch.randn(6, 5, 72, device=dev).to(BF16)
    q, s = pkg.ops.quantize_rows(x)
    assert q.shape == x.shape and s.shape == (6, 5)
    for view in (x[:, 1:4], x.transpose(0, 1), x[2:, :, 3:67]):  # strided, and at odd addresses
        a, b = pkg.ops.quantize_rows(view)
        c, d = pkg.ops.quantize_rows(view.clone(memory_format=torch.contiguous_format))
        assert a.shape == view.shape and torch.equal(_bytes(a), _bytes(c)) and torch.equal(b, d)
    q, s = pkg.ops.quantize_rows(x[:0])
    assert q.shape == (0, 5, 72) and s.shape == (0, 5)


@pytest.mark.parametrize("T,n", SHAPES)
@pytest.mark.parametrize("with_h", [True, False])
def test_add_rms_fp8_against_64_bits(pkg, dev, T, n, with_h):
    """total bit for bit, norm that of add_rms, the 8-bit rows within half a step of the norm in
    64 bits. The fp32 norm is off by at most (n / 64 + 40) 2^-24: 64 lanes' sums of n / 64
    squares, joined, then rsqrt and three products."""
    g = torch.Generator().manual_seed(T * 7 + n)
    x, w = torch.randn(T, n, generator=g).to(BF16), (torch.randn(n, generator=g) * 0.2).to(BF16)
    h = torch.randn(T, n, generator=g).to(BF16) if with_h else None
    hd = None if h is None else h.to(dev)
    total, q, s, norm = pkg.ops.add_rms_fp8(x.to(dev), hd, w.to(dev), EPS, return_norm=True)
    t0, q0, s0 = pkg.ops.add_rms_fp8(x.to(dev), hd, w.to(dev), EPS)
    total1, norm1 = pkg.ops.add_rms(x.to(dev), hd, w.to(dev), EPS)
    assert torch.equal(total, total1) and torch.equal(norm, norm1) and torch.equal(t0, total)
    assert torch.equal(_bytes(q), _bytes(q0)) and torch.equal(s, s0)
    t64 = total.double().cpu()
    y = t64 / (t64.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + w.double())
    rel = (n / 64 + 40) * 2.0**-24
    amax = y.abs().amax(-1)
    assert ((s.double().cpu() - amax / 448).abs() <= amax / 448 * 2 * rel).all()
    sd = s.double().cpu()[:, None]
    off = (q.double().cpu() * sd - y).abs()
    assert (off <= y.abs() * (2.0**-4 + 4 * rel) + sd * 2.0**-10 * (1 + rel)).all()


def test_add_rms_fp8_empty_masked_and_non_finite_rows(pkg, dev):
    """A row of zeros gives zeros and scale 1; a row with a NaN or an infinity is NaN where add_rms
    makes it so, and leaves the other rows alone."""
    x = torch.randn(5, 256, generator=torch.Generator().manual_seed(3)).to(BF16)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 7] = float("inf")
    w = torch.zeros(256, dtype=BF16)
    total, q, s, norm = pkg.ops.add_rms_fp8(x.to(dev), None, w.to(dev), EPS, return_norm=True)
    alone = pkg.ops.add_rms_fp8(x[4:].to(dev), None, w.to(dev), EPS)
    assert torch.equal(torch.isnan(q.float()), torch.isnan(norm))
    assert torch.equal(q[1].float().cpu(), torch.zeros(256)) and s[1] == 1
    assert torch.isnan(q[2].float()).all() and torch.isnan(q[3, 7].float())
    assert torch.equal(_bytes(q[4:]), _bytes(alone[1]))
    assert total.data_ptr() != 0 and torch.equal(torch.isnan(total).cpu(), torch.isnan(x))
    empty = pkg.ops.add_rms_fp8(x[:0].to(dev), x[:0].to(dev), w.to(dev), EPS, return_norm=True)
    assert [e.shape for e in empty] == [(0, 256), (0, 256), (0,), (0, 256)]


def test_rows_write_nothing_behind_the_last_row(pkg, dev):
    x = torch.randn(5, 72, device=dev).to(BF16)
    q = torch.full((8, 72), 0x55, dtype=torch.uint8, device=dev)
    s = torch.full((8,), -7.0, device=dev)
    lib = pkg._lib.load()
    pkg._lib.check(lib.moe_quantize_rows(x.data_ptr(), 5, 72, q.data_ptr(), s.data_ptr(),
                                         pkg._lib.stream_of(x)), "quantize_rows")
    want = pkg.ops.quantize_rows(x)
    assert torch.equal(q[:5].cpu(), _bytes(want[0])) and torch.equal(s[:5], want[1])
    assert (q[5:] == 0x55).all() and (s[5:] == -7).all()


def test_rows_on_another_stream_and_in_a_graph(pkg, dev):
    x, h = torch.randn(33, 512, device=dev).to(BF16), torch.randn(33, 512, device=dev).to(BF16)
    w = torch.randn(512, device=dev).to(BF16)
    want = pkg.ops.add_rms_fp8(x, h, w, EPS, return_norm=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.ops.add_rms_fp8(x, h, w, EPS, return_norm=True)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.float(), b.float())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pkg.ops.add_rms_fp8(x, h, w, EPS, return_norm=True)
        rows = pkg.ops.quantize_rows(got[3])
    for i in range(3):
        x.copy_(torch.randn(33, 512, device=dev))
        graph.replay()
        want = pkg.ops.add_rms_fp8(x, h, w, EPS, return_norm=True)
        w2 = pkg.ops.quantize_rows(want[3])
        torch.cuda.synchronize()
        for a, b in zip((*want, *w2), (*got, *rows)):
            assert torch.equal(a.float(), b.float()), i
