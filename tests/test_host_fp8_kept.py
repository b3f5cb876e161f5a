"""The bounds of fp8_kept_ref see what they are for: mistakes planted in the reference, on the CPU."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_kept_ref as kept
from tests import fp8_ref as ref
from tests.helpers import BF16, routing


def _case(T, H, E, k, I):
    g = torch.Generator().manual_seed(T + E)
    q, xs = ref.rows(torch.randn(T, H, generator=g).to(BF16))
    gu, gus = ref.rows((torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(BF16))
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5).to(BF16))
    idx, wts = routing(T, E, k, "uniform", g)
    return q, xs, idx, wts, gu, gus, dn, dns


def _fp16_groups(y, low=0):
    """y through fp16 with a power of two per 32 columns, ``low`` binary places under the kernels'."""
    g = y.reshape(y.shape[0], -1, 32)
    two = torch.exp2(torch.floor(torch.log2(g.abs().amax(-1, keepdim=True).clamp_min(2.0**-100))) - 14 + low)
    return ((g / two).to(torch.float16).double() * two).reshape(y.shape)


@pytest.mark.parametrize("T,E", [(16, 8), (130, 8)])
def test_bound_holds_for_fp16_pairs_and_not_for_bf16_ones(T, E):
    case = _case(T, 96, E, 4, 64)
    want, bound = kept.experts(*case)
    assert not kept.few(case[2], E)
    share = lambda plant: ref.inside(kept.experts(*case, plant=plant)[0].to(BF16), want, bound)  # noqa: E731
    assert share(_fp16_groups) <= 1
    assert share(lambda y: y.to(BF16).double()) > 1
    assert share(lambda y: _fp16_groups(y, low=36)) > 1


def test_bound_of_few_pairs_sees_fp16_pairs():
    # (the final rounding is as large as most of what fp16 loses: of many outputs some are near zero)
    case = _case(4, 512, 8, 4, 64)
    assert kept.few(case[2], 8)
    want, bound = kept.experts(*case)
    plain = ref.inside(want.to(BF16), want, bound)
    assert plain <= 1
    rough = kept.experts(*case, plant=lambda y: y.to(BF16).double())[0]
    assert ref.inside(rough.to(BF16), want, bound) > plain
