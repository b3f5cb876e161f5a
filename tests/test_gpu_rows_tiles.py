"""Every tile that ops.linear and ops.experts_fp8 choose from: more tiles than workgroups that the chip
holds, ragged edges, rows past 2^31 bytes, in sums that are exact or against copies of the same token."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16, routing

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def _small(dev, g, *shape, e4m3=False):
    """Integers up to 8: products of up to 2^6, sums of up to 2^6 K, exact in fp32 in any order, and no
    product under 2^-6 of another (the e4m3 instruction cuts none)."""
    t = torch.randint(-8, 9, shape, generator=g, device=dev).to(BF16)
    return t.to(FP8) if e4m3 else t



# 256 x 256 tiles: one round of workgroups, two; 128: few, more than two a unit; 64: few, more than two a
# unit, either way round; 128 x 64
TILES = [(4096, 4096, 48), (7700, 4000, 32), (7700, 4001, 448), (1100, 2100, 200), (4200, 4000, 48), (300, 520, 328),
         (40, 66001, 80), (66001, 40, 144), (33, 77, 16), (1111, 1537, 328), (250, 8000, 104)]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("M,N,K", TILES)
def test_linear_tiles_exactly(pkg, dev, M, N, K, e4m3):
    K -= K % 16 if e4m3 else 0  # e4m3 rows are multiples of 16 bytes
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    x, w = _small(dev, g, M, K, e4m3=e4m3), _small(dev, g, N, K, e4m3=e4m3)
    kw = {}
    if e4m3:
        kw = dict(x_scale=torch.exp2(torch.randint(-3, 4, (M,), generator=g, device=dev).float()),
                  w_scale=torch.exp2(torch.randint(-3, 4, (N,), generator=g, device=dev).float()))
    bias = torch.randint(-8, 9, (N,), generator=g, device=dev).float()
    mul, res = _small(dev, g, M, N), _small(dev, g, M, N)
    plain = pkg.ops.linear(x, w, **kw)
    full = pkg.ops.linear(x, w, bias=bias, activation="relu", mul=mul, residual=res, **kw)
    xf, wf = x.float().double(), w.float().double()
    for r0 in range(0, M, 4096):
        v = xf[r0 : r0 + 4096] @ wf.t()
        if e4m3:
            v *= kw["x_scale"][r0 : r0 + 4096, None].double() * kw["w_scale"].double()
        rows = slice(r0, r0 + 4096)
        assert torch.equal(plain[rows], v.to(BF16))
        v = (v + bias.double()).clamp_min(0) * mul[rows].double() + res[rows].double()
        assert torch.equal(full[rows], v.to(BF16))


@pytest.mark.parametrize("e4m3", [False, True])
def test_linear_past_31_bits(pkg, dev, e4m3):
    """Rows of x, residual and output that lie more than 2^31 elements behind the first (67000 x 32768),
    and weight rows more than 2^31 bytes behind theirs."""
    M, N, K = 67000, 32768, 32
    g = torch.Generator(device=dev).manual_seed(5)
    wide = torch.empty(M, N, dtype=BF16, device=dev)
    step = 4096
    for r in range(0, M, step):
        wide[r : r + step] = _small(dev, g, min(step, M - r), N)
    x = wide[:, 64 : 64 + K] if not e4m3 else wide.view(torch.uint8)[:, :K].view(FP8)
    if e4m3:
        x.view(torch.uint8).copy_(_small(dev, g, M, K, e4m3=True).view(torch.uint8))
    w = _small(dev, g, N, K, e4m3=e4m3)
    kw = dict(x_scale=torch.ones(M, device=dev), w_scale=torch.ones(N, device=dev)) if e4m3 else {}
    got = pkg.ops.linear(x, w, residual=None if e4m3 else wide, **kw)
    for r in range(0, M, step):
        want = x[r : r + step].float().double() @ w.float().double().t()
        if not e4m3:
            want += wide[r : r + step].double()
        assert torch.equal(got[r : r + step], want.to(BF16)), r
    del got
    # the same rows as weights: their outputs lie across
    y = _small(dev, g, 40, K, e4m3=e4m3)
    kw = dict(x_scale=torch.ones(40, device=dev), w_scale=torch.ones(M, device=dev)) if e4m3 else {}
    for rows in (40, 3):
        got = pkg.ops.linear(y[:rows], x, **({**kw, "x_scale": kw["x_scale"][:rows]} if e4m3 else {}))
        want = y[:rows].float().double() @ x.float().double().t()
        assert torch.equal(got, want.to(BF16))


def _layer(dev, T, H, E, I, seed):
    g = torch.Generator().manual_seed(seed)
    q, xs = ref.rows(torch.randn(T, H, generator=g).to(BF16))
    gu, gus = ref.rows((torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(BF16))
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5).to(BF16))
    return (q, xs, gu, gus, dn, dns), g


# pairs an expert: 4, 20 (more than two workgroups a unit in the down product), 64, 112 and 128 (more than
# one), 300 of few experts, one expert
BATCHES = [(64, 96, 64, 160, 4, "uniform"), (160, 4096, 16, 96, 2, "uniform"), (512, 2080, 32, 416, 4, "uniform"),
           (896, 160, 64, 160, 8, "skewed"), (1024, 2080, 32, 800, 4, "uniform"), (600, 96, 4, 224, 2, "sparse"),
           (700, 64, 1, 96, 1, "uniform"), (1024, 64, 32, 544, 4, "one")]


@pytest.mark.parametrize("T,H,E,I,k,mode", BATCHES)
def test_experts_tiles(pkg, dev, T, H, E, I, k, mode):
    """Copies of 12 tokens at every place of the batch: each as the first, and the first within its bound."""

    (q, xs, gu, gus, dn, dns), g = _layer(dev, 12, H, E, I, T + H)
    idx, wts = routing(12, E, k, mode, g)
    at = torch.randint(12, (T,), generator=g)
    at[:12] = torch.arange(12)
    d = lambda t: t.to(dev)  # noqa: E731
    take = lambda t: t.view(torch.uint8)[at].view(t.dtype) if t.dtype == FP8 else t[at]  # noqa: E731
    got = pkg.ops.experts_fp8(*(d(take(t)) for t in (q, xs, idx, wts)), d(gu), d(dn), gate_up_scale=d(gus),
                              down_scale=d(dns))
    want, bound = ref.experts(q, xs, idx, wts, gu, gus, dn, dns)
    assert ref.inside(got[:12], want, bound) <= 1
    assert torch.equal(got, got[:12][at.to(dev)])


@pytest.mark.parametrize("T", [3, 40, 600])
def test_experts_outputs_of_very_different_size(pkg, dev, T):
    """Outputs whose size differs by 2^100 from one 32 columns to the next, and one that is infinite, keep
    their digits; columns of zeros stay zeros."""
    (q, xs, gu, gus, dn, dns), g = _layer(dev, 12, 192, 4, 96, T)
    dns[:] *= torch.exp2(torch.tensor([-80.0, 20.0, 0.0, -40.0, 60.0, 10.0]).repeat_interleave(32))
    dns[:, 64:96] = 0
    idx, wts = routing(12, 4, 2, "uniform", g)
    want, bound = ref.experts(q, xs, idx, wts, gu, gus, dn, dns)
    dns[:, 161] = torch.inf
    at = torch.arange(T) % 12
    d = lambda t: t.to(dev)  # noqa: E731
    got = pkg.ops.experts_fp8(d(q.view(torch.uint8)[at].view(FP8)), d(xs[at]), d(idx[at]), d(wts[at]), d(gu),
                              d(dn), gate_up_scale=d(gus), down_scale=d(dns))
    assert not torch.isfinite(got[:, 161]).any()
    got[:, 161] = want.to(dev)[at.to(dev), 161].to(BF16)
    assert ref.inside(got, want[at], bound[at]) <= 1
    assert (got[:, 64:96] == 0).all()


def test_experts_more_pairs_than_a_grid_has_rows(pkg, dev):
    """2^20 and some tokens of 2048 columns: past 2^31 bytes, where the kernel of few rows takes all, in
    more tiles than one launch has."""
    T, H, E, I = (1 << 20) + 70000, 2048, 8, 32
    (q, xs, gu, gus, dn, dns), g = _layer(dev, 12, H, E, I, 1)
    idx, wts = routing(12, E, 1, "uniform", g)
    at = torch.randint(12, (T,), generator=g).to(dev)
    at[:12] = torch.arange(12, device=dev)
    d = lambda t: t.to(dev)  # noqa: E731
    got = pkg.ops.experts_fp8(d(q).view(torch.uint8)[at].view(FP8), d(xs)[at], d(idx)[at], d(wts)[at], d(gu), d(dn),
                              gate_up_scale=d(gus), down_scale=d(dns))
    want, bound = ref.experts(q, xs, idx, wts, gu, gus, dn, dns)
    assert ref.inside(got[:12], want, bound) <= 1
    for r in range(0, T, 1 << 17):
        assert torch.equal(got[r : r + (1 << 17)], got[:12][at[r : r + (1 << 17)]])
