"""ops.linear on e4m3 rows whose scales are views: strided, expanded, of other shapes."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16

pytestmark = pytest.mark.gpu


def _operands(M, K, N, dev):
    g = torch.Generator().manual_seed(M + N)
    (x, xs), (w, ws) = ref.rows(torch.randn(M, K, generator=g).to(BF16)), ref.rows(torch.randn(N, K, generator=g).to(BF16))
    # sizes that tell one scale from another
    xs, ws = xs * torch.exp2(torch.arange(M) % 5.0), ws * torch.exp2(-(torch.arange(N) % 7.0))
    bias, mul, res = torch.randn(N, generator=g), torch.randn(M, N, generator=g).to(BF16), torch.randn(M, N, generator=g).to(BF16)
    return [t.to(dev) for t in (x, w, xs, ws, bias, mul, res)]


def _spread(t):
    """``t`` as every other element (or column) of a tensor whose others are large."""
    wide = torch.full((*t.shape, 2), 1e6, dtype=t.dtype, device=t.device)
    wide[..., 0] = t
    return wide[..., 0]


@pytest.mark.parametrize("M,N", [(5, 5), (96, 96), (7, 300), (300, 7), (256, 512)])
def test_linear_strided_scales(pkg, dev, M, N):
    """Copies of strided scales are made before the call and read in it: none may be the place of another
    copy or of the output."""
    x, w, xs, ws, bias, mul, res = _operands(M, 64, N, dev)
    lin = pkg.ops.linear
    want = lin(x, w, x_scale=xs, w_scale=ws)
    full = lin(x, w, x_scale=xs, w_scale=ws, bias=bias, mul=mul, residual=res)
    xv, wv = _spread(xs), _spread(ws)
    assert not xv.is_contiguous() and not wv.is_contiguous()
    for a, b in ((xv, ws), (xs, wv), (xv, wv)):
        assert torch.equal(lin(x, w, x_scale=a, w_scale=b), want)
        assert torch.equal(lin(x, w, x_scale=a, w_scale=b, bias=_spread(bias), mul=_spread(mul), residual=_spread(res)),
                           full)


@pytest.mark.parametrize("M,N", [(6, 6), (200, 130)])
def test_linear_one_scale_expanded(pkg, dev, M, N):
    x, w, _, _, _, mul, _ = _operands(M, 64, N, dev)
    one, two = torch.tensor(0.25, device=dev), torch.tensor(3.0, device=dev)
    want = pkg.ops.linear(x, w, x_scale=one.repeat(M), w_scale=two.repeat(N), mul=mul)
    assert torch.equal(pkg.ops.linear(x, w, x_scale=one.expand(M), w_scale=two.expand(N), mul=_spread(mul)), want)


def test_linear_strided_scales_in_a_graph(pkg, dev):
    x, w, xs, ws, _, mul, _ = _operands(40, 64, 40, dev)
    xv, wv, mv = _spread(xs), _spread(ws), _spread(mul)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.ops.linear(x, w, x_scale=xv, w_scale=wv, mul=mv)
    for i in range(4):
        xv.mul_(2.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, pkg.ops.linear(x, w, x_scale=xv.contiguous(), w_scale=ws, mul=mul)), i
        torch.cuda.synchronize()


def test_scales_of_another_shape_are_refused(pkg, dev):
    """As many values in another order would be taken for the wrong rows; one dimension, and dimensions
    of one, leave the order as it is."""
    x, w, xs, ws, bias, _, _ = _operands(6, 64, 8, dev)
    lin, x3 = pkg.ops.linear, x.view(2, 3, 64)
    want = lin(x, w, x_scale=xs, w_scale=ws)
    for a, b in ((xs.view(2, 3), ws), (xs, ws), (xs.view(2, 3, 1), ws.view(8, 1)), (xs.view(1, 6), ws.view(1, 8))):
        assert torch.equal(lin(x3, w, x_scale=a, w_scale=b).view(6, 8), want)
    one = lin(x[0], w, x_scale=xs[0], w_scale=ws)
    assert torch.equal(one, want[0]) and torch.equal(lin(x[:1], w, x_scale=xs[:1, None], w_scale=ws)[0], one)
    for bad in (dict(x_scale=xs.view(3, 2), w_scale=ws), dict(x_scale=xs.view(2, 3), w_scale=ws.view(2, 4)),
                dict(x_scale=xs.view(2, 3).t(), w_scale=ws), dict(x_scale=xs, w_scale=ws, bias=bias.view(4, 2))):
        with pytest.raises(ValueError):
            lin(x3, w, **bad)


def test_expert_scales_of_another_shape_are_refused(pkg, dev):
    T, H, E, I = 5, 64, 8, 32
    g = torch.Generator().manual_seed(0)
    q, xs = ref.rows(torch.randn(T, H, generator=g).to(BF16))
    gu, gus = ref.rows(torch.randn(E, 2 * I, H, generator=g).to(BF16))
    dn, dns = ref.rows(torch.randn(E, H, I, generator=g).to(BF16))
    idx, wts = torch.randint(E, (T, 2), generator=g), torch.rand(T, 2, generator=g).to(BF16)
    q, xs, gu, gus, dn, dns, idx, wts = (t.to(dev) for t in (q, xs, gu, gus, dn, dns, idx, wts))

    def call(scale=xs, gate_up_scale=gus, down_scale=dns):
        return pkg.ops.experts_fp8(q, scale, idx, wts, gu, dn, gate_up_scale=gate_up_scale, down_scale=down_scale)

    want = call()
    for good in (dict(scale=xs[:, None]), dict(gate_up_scale=gus.flatten()), dict(down_scale=dns[..., None]),
                 dict(gate_up_scale=_spread(gus), down_scale=_spread(dns), scale=_spread(xs))):
        assert torch.equal(call(**good), want)
    for bad in (dict(gate_up_scale=gus.t()), dict(gate_up_scale=gus.t().contiguous()), dict(down_scale=dns.t()),
                dict(gate_up_scale=gus.view(2 * E, I)), dict(down_scale=dns.view(E, 2, H // 2))):
        with pytest.raises(ValueError):
            call(**bad)
