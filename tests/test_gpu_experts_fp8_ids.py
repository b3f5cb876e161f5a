"""ops.experts_fp8 with expert indices outside [0, E): the nearest expert, in each of its kernels."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16, routing

pytestmark = pytest.mark.gpu


# pairs by themselves (up to 16, up to E / 4), tiles of 16, 64 and 128
@pytest.mark.parametrize("T,E", [(1, 8), (4, 8), (12, 200), (20, 8), (70, 8), (700, 8)])
@pytest.mark.parametrize("far", [1, 2**31, 2**40])
def test_experts_fp8_indices_outside_count_as_the_nearest(pkg, dev, T, E, far):
    H, I, k = 96, 64, 4
    g = torch.Generator().manual_seed(T + E)
    q, xs = ref.rows(torch.randn(T, H, generator=g).to(BF16))
    gu, gus = ref.rows((torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(BF16))
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5).to(BF16))
    idx, wts = routing(T, E, k, "uniform", g)
    idx[0, 0], idx[T // 2, 1], idx[T - 1, 3] = -far, E - 1 + far, -1
    d = lambda t: t.to(dev)  # noqa: E731
    call = lambda i, w: pkg.ops.experts_fp8(d(q), d(xs), d(i), d(w), d(gu), d(dn), gate_up_scale=d(gus),  # noqa: E731
                                            down_scale=d(dns))
    assert torch.equal(call(idx, wts), call(idx.clamp(0, E - 1), wts))
    # a masked slot, weight 0, leaves the sum of the others
    masked = wts.clone()
    masked[(idx < 0) | (idx >= E)] = 0
    inside = idx.clamp(0, E - 1)
    want, bound = ref.experts(q, xs, inside, masked, gu, gus, dn, dns)
    assert ref.inside(call(idx, masked), want, bound) <= 1
