"""ops.experts_fp8 on each way that its kernels take, with that way's own bound: products that are cut or kept,
pair outputs in fp32 or through fp16."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_kept_ref as kept
from tests import fp8_ref as ref
from tests.helpers import BF16, routing

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


# pairs by themselves; tiles of 16, 64, 128 and 192
CASES = [(1, 64, 8, 4, 64), (8, 96, 8, 2, 96), (14, 64, 256, 4, 64), (20, 96, 8, 4, 64), (90, 64, 8, 1, 160),
         (120, 96, 8, 4, 96), (700, 64, 8, 2, 64), (300, 96, 32, 8, 416), (512, 64, 32, 8, 800)]


@pytest.mark.parametrize("T,H,E,k,I", CASES)
def test_experts_fp8_each_way_within_its_own_bound(pkg, dev, T, H, E, k, I):
    g = torch.Generator().manual_seed(T + H + I)
    n = min(T, 24)  # copies of 24 tokens at every place
    q, xs = ref.rows(torch.randn(n, H, generator=g).to(BF16))
    gu, gus = ref.rows((torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(BF16))
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5).to(BF16))
    idx, wts = routing(n, E, k, "uniform", g)
    at = torch.arange(T) % n
    args = (q.view(torch.uint8)[at].view(FP8), xs[at], idx[at], wts[at])
    got = pkg.ops.experts_fp8(*(t.to(dev) for t in (*args, gu, dn)), gate_up_scale=gus.to(dev), down_scale=dns.to(dev))
    assert torch.equal(got, got[:n][at.to(dev)])
    # the way is chosen by all tokens: the reference of the first n is of as many copies as it needs
    want, bound = kept.experts(*args, gu, gus, dn, dns)
    share = ref.inside(got, want, bound)
    print(f"experts_fp8 {T} x {H}, {E} experts of {I}: {share:.3f} of the bound", flush=True)
    assert share <= 1
