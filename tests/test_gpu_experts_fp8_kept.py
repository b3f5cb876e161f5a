"""ops.experts_fp8 and ops.linear on few e4m3 rows: small products beside large ones that cancel are kept."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_kept_ref as kept
from tests import fp8_ref as ref
from tests.helpers import BF16, routing

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def _cancelling(g, rows, weights, K):
    """x [rows, K] and w [..., K] of whole numbers: in each eight neighbours 256 * 256 - 256 * 256 and six
    products of up to 7, whose sums are what is left."""
    x = torch.randint(1, 8, (rows, K // 8, 8), generator=g).float()
    w = torch.randint(0, 2, (*weights, K // 8, 8), generator=g).float()
    x[..., :2] = 256
    w[..., 0], w[..., 1] = 256, -256
    return x.reshape(rows, K).to(FP8), w.reshape(*weights, K).to(FP8)


@pytest.mark.parametrize("M,N,K", [(1, 40, 64), (5, 2048, 208), (16, 300, 2048), (3, 4100, 80), (16, 5000, 144)])
def test_linear_few_rows_keep_small_products(pkg, dev, M, N, K):
    """Up to 16 rows: sums of whole numbers below 2^24, exact, whose large products cancel."""
    g = torch.Generator().manual_seed(M + N + K)
    x, w = _cancelling(g, M, (N,), K)
    xs, ws = torch.exp2(torch.randint(-4, 5, (M,), generator=g)), torch.exp2(torch.randint(-4, 5, (N,), generator=g))
    got = pkg.ops.linear(x.to(dev), w.to(dev), x_scale=xs.to(dev), w_scale=ws.to(dev))
    want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    assert want.count_nonzero() == want.numel()
    assert torch.equal(got.cpu(), want.to(BF16))


# pairs by themselves; up to 12 pairs an expert
@pytest.mark.parametrize("T,E,k", [(1, 8, 4), (8, 8, 2), (12, 200, 4), (20, 8, 4), (40, 16, 4)])
def test_experts_few_rows_keep_small_products(pkg, dev, T, E, k):
    H, I = 96, 64
    g = torch.Generator().manual_seed(T + E)
    q, gu = _cancelling(g, T, (E, 2 * I), H)
    xs, gus = torch.exp2(torch.randint(-3, 1, (T,), generator=g)), torch.exp2(torch.randint(-6, -3, (E, 2 * I), generator=g))
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5).to(BF16))
    idx, wts = routing(T, E, k, "uniform", g)
    assert kept.kept(idx, E)
    got = pkg.ops.experts_fp8(*(t.to(dev) for t in (q, xs.float(), idx, wts, gu, dn)), gate_up_scale=gus.float().to(dev),
                              down_scale=dns.to(dev))
    want, bound = kept.experts(q, xs.float(), idx, wts, gu, gus.float(), dn, dns, whole=True)
    share = ref.inside(got, want, bound)
    print(f"experts_fp8 {T} tokens, cancelling: {share:.3f} of the bound", flush=True)
    assert share <= 1
