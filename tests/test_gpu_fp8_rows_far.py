"""ops.add_rms_fp8 where its norm is next to the ends of fp32: q and scale are those of the norm itself."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16

pytestmark = pytest.mark.gpu


def _norm64(x, w, eps):
    return x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt() * (1 + w.double())


@pytest.mark.parametrize("eps", [0.3, 0.7, 1.0, 3.0])
@pytest.mark.parametrize("n", [8, 520])
def test_add_rms_fp8_tiny_rows(pkg, dev, eps, n):
    """A largest value under 2^-100 counts as 2^-100, whatever the reciprocal root is. The scale has a few
    roundings of 2^-24, the quotient some more; q is off by half a step, 2^-4 of a value and 2^-10 at the least."""
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(6, n, generator=g) * torch.exp2(torch.tensor([-99.0, -101, -103, -106, -109, -112]))[:, None]).to(BF16)
    w = (torch.randn(n, generator=g) * 0.2).to(BF16)
    _, q, s = pkg.ops.add_rms_fp8(x.to(dev), None, w.to(dev), eps)
    y = _norm64(x, w, eps)
    want = y.abs().amax(-1).clamp_min(2.0**-100) / 448
    assert ((s.double().cpu() - want).abs() <= want * 64 * 2.0**-24).all(), s.double().cpu() / want
    v = y / want[:, None]
    off = (q.double().cpu() - v).abs()
    assert (off <= v.abs() * (2.0**-4 + 2.0**-16) + 2.0**-10 * (1 + 2.0**-16)).all()


@pytest.mark.parametrize("n", [264, 1032, 4096])
@pytest.mark.parametrize("with_h", [False, True])
def test_add_rms_fp8_values_past_fp32_are_nan(pkg, dev, n, with_h):
    """Where the norm is infinite its 8 bits are NaN, and the scale is of the row's finite values."""
    g = torch.Generator().manual_seed(n)
    x, w = torch.randn(40, n, generator=g).to(BF16), torch.zeros(n).to(BF16)
    far = [3, 100, n // 2, n - 1]
    w[far] = 3.0e38
    x[:20, far] *= 0.25
    h = torch.randn(40, n, generator=g).to(BF16) * 0.125 if with_h else None
    total, q, s, norm = pkg.ops.add_rms_fp8(x.to(dev), None if h is None else h.to(dev), w.to(dev), 1e-6, return_norm=True)
    y = _norm64(total.cpu(), w, 1e-6)
    top = torch.finfo(torch.float32).max
    past = y.abs() > top
    # no value so near to the end that fp32's roundings decide, and rows of either kind
    assert ((y.abs() / top - 1).abs() > 2.0**-18).all() and 4 < past.any(-1).sum() < 40
    assert torch.equal(torch.isnan(q.float().cpu()), past)
    assert torch.isinf(norm.float().cpu()[past]).all()
    want = torch.where(past, 0.0, y.abs()).amax(-1) / 448
    assert ((s.double().cpu() - want).abs() <= want * 64 * 2.0**-24).all()
    fine = torch.where(past, 0.0, y / want[:, None])
    off = torch.where(past, 0.0, (q.double().cpu() - fine).abs())
    assert (off <= fine.abs() * (2.0**-4 + 2.0**-16) + 2.0**-10 * (1 + 2.0**-16)).all()
