"""block.add_rms_moe_fp8: the 8-bit operators run together, against add_rms_moe (norm, routing), 64 bits
(the output), on streams and in graphs."""

from __future__ import annotations

import copy

import pytest
import torch

from oracle import moe_oracle as orc
from tests import fp8_ref as ref
from tests.helpers import BF16

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="module", params=[(256, 16, 96, 160), (384, 64, 128, 96)])
def layer(request, pkg, dev):
    import __graft_entry__

    H, E, I, S = request.param
    mlp = __graft_entry__._mlp_from_weights(orc.make_weights(H, E, I, S, seed=7), dev)
    return _fp8(pkg, mlp), mlp, H


def _fp8(pkg, mlp):
    m = copy.copy(mlp)
    m.experts = copy.copy(mlp.experts)
    for name in ("gate_up", "down"):
        q, s = pkg.fp8.quantize_rows(getattr(mlp.experts, name + "_proj"))
        setattr(m.experts, name + "_proj", q)
        setattr(m.experts, name + "_scale", s)
    return m


def _inputs(T, H, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(T, H, generator=g) * 2).to(BF16).to(dev), torch.randn(T, H, generator=g).to(BF16).to(dev),
            (torch.randn(H, generator=g) * 0.1).to(BF16).to(dev))


def _want(mlp, q, scale, total, norm, idx, wts, logits):
    """The block's output in 64 bits from its norm and routing, and the bound on what the roundings on the
    way can do: each product's bound (fp8_ref.linear, fp8_ref.experts) carried through the next."""
    c = lambda t: t.detach().cpu()  # noqa: E731
    sh, ex = mlp.shared_expert, mlp.experts
    norm, sg, su, sd = c(norm), c(sh.gate_proj.weight), c(sh.up_proj.weight), c(sh.down_proj.weight)
    gate, gate_off = ref.linear(norm, sg, activation="silu")
    up, up_off = ref.linear(norm, su)
    act, off = ref.linear(norm, su, mul=gate)
    off = (off + gate_off * (up.abs() + up_off)) * 1.01
    y, y_off = ref.linear(act, sd.double())
    y_off = (y_off + off @ sd.double().abs().t()) * 1.01
    s = torch.sigmoid(c(logits)[:, ex.gate_up_proj.shape[0], None].double())
    y_off = s * y_off + s * 2.0**-7 * (y.abs() + y_off)  # the gate's rounding and the product's
    routed, r_off = ref.experts(c(q), c(scale), c(idx), c(wts), c(ex.gate_up_proj), c(ex.gate_up_scale),
                                c(ex.down_proj), c(ex.down_scale))
    both, b_off = routed + s * y, r_off + y_off
    out = both + c(total).double()
    return out, b_off * 1.01 + (both.abs() + b_off) * 2.0**-8 + (out.abs() + b_off) * 2.0**-8


@pytest.mark.parametrize("T", [1, 3, 16, 70, 300])
@pytest.mark.parametrize("with_h", [True, False])
def test_block_fp8_against_64_bits(pkg, dev, layer, T, with_h):
    mlp, _, H = layer
    x, h, w = _inputs(T, H, T, dev)
    h = h if with_h else None
    out, total, norm, idx, wts, logits = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4, return_norm=True,
                                                                   return_routing=True)
    b_total, b_norm = pkg.ops.add_rms(x, h, w, EPS)
    b_wts, b_idx, _ = pkg.ops.route(logits, 4, mlp.experts.gate_up_proj.shape[0])
    b_logits = pkg.ops.router_logits(norm, pkg.pack_router(mlp))
    for got, same in ((total, b_total), (norm, b_norm), (idx, b_idx), (wts, b_wts), (logits, b_logits)):
        assert torch.equal(got, same)
    assert torch.equal(pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4), out)
    _, q, scale = pkg.ops.add_rms_fp8(x, h, w, EPS)
    want, bound = _want(mlp, q, scale, total, norm, idx, wts, logits)
    share = ref.inside(out, want, bound)
    print(f"add_rms_moe_fp8 {T}: {share:.3f} of the bound", flush=True)
    assert share <= 1


@pytest.mark.parametrize("T", [1, 20, 200])
def test_block_fp8_routes_as_the_bf16_block(pkg, dev, T):
    import __graft_entry__

    mlp = _fp8(pkg, __graft_entry__._mlp_from_weights(orc.make_weights(512, 32, 128, 128, seed=8), dev))
    x, h, w = _inputs(T, 512, T, dev)
    ours = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4, return_norm=True, return_routing=True)
    bf16 = pkg.block.add_rms_moe(x, h, w, EPS, mlp, 4, return_norm=True, return_routing=True)
    for got, same in zip(ours[1:], bf16[1:]):
        assert torch.equal(got, same)
    # (The outputs themselves have their 64-bit bound above. Against each other they have no small one: the
    # total here is about ten times the block's share, and each output's own last roundings, 2^-8 of its
    # size each, are already several percent of that share.)


def test_block_fp8_shapes_and_refusals(pkg, dev, layer):
    mlp, bf16, H = layer
    x, h, w = _inputs(6, H, 1, dev)
    base = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 2)
    assert torch.equal(pkg.block.add_rms_moe_fp8(x.view(2, 3, H), h.view(2, 3, H), w, EPS, mlp, 2),
                       base.view(2, 3, H))
    out, total, norm = pkg.block.add_rms_moe_fp8(x[:0], h[:0], w, EPS, mlp, 2, return_norm=True)
    assert out.shape == total.shape == norm.shape == (0, H)
    with pytest.raises(ValueError):
        pkg.block.add_rms_moe_fp8(x, h, w, EPS, bf16, 2)
    with pytest.raises(ValueError):
        pkg.block.add_rms_moe_fp8(x.float(), h, w, EPS, mlp, 2)
    with pytest.raises(ValueError):
        pkg.block.add_rms_moe_fp8(x, h, w[:-1], EPS, mlp, 2)
    with pytest.raises((ValueError, pkg.MoeLibraryError)):
        pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, mlp.experts.gate_up_proj.shape[0] + 1)


def test_block_fp8_masked_tokens(pkg, dev, layer):
    """Padding rows of zeros, and a row that is not finite, change no other row."""
    mlp, _, H = layer
    x, h, w = _inputs(50, H, 2, dev)
    base = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4)
    x[40:], h[40:] = 0, 0
    x[3, 5] = torch.nan
    got = pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4)
    keep = torch.ones(50, dtype=torch.bool, device=dev)
    keep[40:], keep[3] = False, False
    assert torch.equal(got[keep], base[keep])
    assert (got[40:] == 0).all() and torch.isnan(got[3, 5])


@pytest.mark.parametrize("T", [1, 60])
def test_block_fp8_streams_and_graphs(pkg, dev, layer, T):
    mlp, _, H = layer
    ins = [_inputs(T, H, 20 + i, dev)[:2] for i in range(2)]
    w = _inputs(1, H, 3, dev)[2]
    call = lambda x, h: pkg.block.add_rms_moe_fp8(x, h, w, EPS, mlp, 4)  # noqa: E731
    want = [call(*i) for i in ins]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(8):
        with torch.cuda.stream(side[i % 2]):
            got.append(call(*ins[i % 2]))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i % 2]) for i, t in enumerate(got))
    x, h = (t.clone() for t in ins[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side[0]):
        out = call(x, h)
    for i in (1, 0, 0, 1):
        x.copy_(ins[i][0]), h.copy_(ins[i][1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
        call(*ins[1 - i])
        torch.cuda.synchronize()
