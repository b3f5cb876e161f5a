"""The experts' tiles of 16, 64, 128 and 192 pairs with scales that differ from group to group and from row to
row, and with rows that are not finite."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16, routing

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn

# tokens, hidden, experts, intermediate, top_k: pairs by themselves; tiles of 16, 64, 128 and 192; the last with
# several of them and ragged ends
SIZES = [(3, 96, 8, 160, 4), (20, 96, 32, 160, 4), (200, 96, 32, 160, 4), (512, 96, 32, 416, 4), (1024, 96, 32, 800, 4),
         (1000, 160, 32, 416, 4), (1100, 2080, 16, 1056, 5)]


def _layer(T, H, E, I, k, seed):
    """Twelve tokens at every place of a batch of T. Between the products group c of 32 columns is 2^up(c) times
    as large as it would be, and the down weights of its columns 2^-up(c) as large: each group counts alike
    in the outputs, so that a scale taken from another group, step or row is off by a power of two of them."""
    g = torch.Generator().manual_seed(seed)
    q, xs = ref.rows(torch.randn(12, H, generator=g).to(BF16))
    xs = xs * torch.exp2(torch.randint(-2, 3, (12,), generator=g))
    gu, gus = ref.rows((torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(BF16))
    up = torch.randint(-3, 4, (I // 32,), generator=g).repeat_interleave(32)
    gus[:, I:] *= torch.exp2(up)
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5 * torch.exp2(-up)).to(BF16))
    idx, wts = routing(12, E, k, "uniform", g)
    at = torch.randint(12, (T,), generator=g)
    at[: min(T, 12)] = torch.arange(min(T, 12))
    return (q, xs, idx, wts, gu, gus, dn, dns), at


def _run(pkg, dev, at, q, xs, idx, wts, gu, gus, dn, dns):
    args = (q.view(torch.uint8)[at].view(FP8), xs[at], idx[at], wts[at], gu, dn)
    return pkg.ops.experts_fp8(*(t.to(dev) for t in args), gate_up_scale=gus.to(dev), down_scale=dns.to(dev))


@pytest.mark.parametrize("T,H,E,I,k", SIZES)
def test_experts_groups_and_rows_of_different_size(pkg, dev, T, H, E, I, k):
    case, at = _layer(T, H, E, I, k, T + I)
    got = _run(pkg, dev, at, *case)
    want, bound = ref.experts(*case)
    n = min(T, 12)
    share = ref.inside(got[:n], want[:n], bound[:n])
    print(f"experts_fp8 {T} x {H}, {E} experts of {I}: {share:.3f} of the bound", flush=True)
    assert share <= 1
    assert torch.equal(got, got[:n][at.to(dev)])


@pytest.mark.parametrize("T,H,E,I,k", SIZES)
def test_experts_non_finite_rows_in_every_tile(pkg, dev, T, H, E, I, k):
    case, at = _layer(T, H, E, I, k, T + I + 1)
    clean = _run(pkg, dev, at, *case)
    assert torch.isfinite(clean).all()
    case[0].view(torch.uint8)[1, 5] = 0x7F  # a NaN in the rows of one token, another's scale infinite
    case[1][2] = torch.inf
    got = _run(pkg, dev, at, *case)
    bad = ((at == 1) | (at == 2)).to(dev)
    assert torch.isnan(got[bad]).all()
    assert torch.equal(got[~bad], clean[~bad])
