"""ops.experts_fp8 against 64 bits, over shapes and routings."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16, routing

pytestmark = pytest.mark.gpu


def _layer(T, H, E, I, seed):
    g = torch.Generator().manual_seed(seed)
    q, xs = ref.rows(torch.randn(T, H, generator=g).to(BF16))
    gu, gus = ref.rows((torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(BF16))
    dn, dns = ref.rows((torch.randn(E, H, I, generator=g) * I**-0.5).to(BF16))
    return q, xs, gu, gus, dn, dns, g


def _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns):
    return pkg.ops.experts_fp8(*(t.to(dev) for t in (q, xs, idx, wts, gu, dn)), gate_up_scale=gus.to(dev),
                               down_scale=dns.to(dev))


CASES = [(1, 64, 8, 2, 32, "uniform"), (1, 2048, 16, 8, 512, "uniform"), (2, 96, 8, 8, 64, "uniform"),
         (5, 160, 16, 1, 96, "uniform"), (4, 256, 8, 3, 128, "one"), (17, 32, 4, 2, 224, "skewed"),
         (33, 256, 16, 4, 96, "uniform"), (64, 512, 16, 8, 256, "skewed"), (70, 128, 8, 4, 64, "sparse"),
         (130, 96, 8, 8, 160, "uniform"), (300, 128, 8, 6, 128, "skewed"), (257, 64, 2, 1, 32, "one"),
         (700, 256, 16, 8, 64, "uniform"), (900, 160, 4, 2, 352, "sparse")]


@pytest.mark.parametrize("T,H,E,k,I,mode", CASES)
def test_experts_fp8_against_64_bits(pkg, dev, T, H, E, k, I, mode):
    q, xs, gu, gus, dn, dns, g = _layer(T, H, E, I, T + H + I)
    idx, wts = routing(T, E, k, mode, g)
    got = _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns)
    assert got.shape == (T, H) and got.dtype == BF16
    assert torch.equal(got, _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns))
    want, bound = ref.experts(q, xs, idx, wts, gu, gus, dn, dns)
    share = ref.inside(got, want, bound)
    rel = ((got.double().cpu() - want).norm() / want.norm()).item()
    print(f"experts_fp8 {T} tokens: {share:.3f} of the bound, rel {rel:.2g}", flush=True)
    assert share <= 1
    # two roundings to bf16 in a row, each at most 2^-8 of its value
    assert rel <= 2 * 2.0**-8


def test_experts_fp8_groups_of_very_different_size(pkg, dev):
    """Columns whose activations differ by 2^40 from group to group (and groups of zeros) keep their own
    scale."""
    q, xs, gu, gus, dn, dns, g = _layer(40, 128, 4, 160, 3)
    gus[:, :] *= torch.exp2(torch.arange(320).remainder(160).div(32, rounding_mode="floor") * 10.0 - 20.0)
    gus[:, 64:96] = 0
    dns[:, :] *= 2.0**-10
    idx, wts = routing(40, 4, 2, "uniform", g)
    got = _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns)
    want, bound = ref.experts(q, xs, idx, wts, gu, gus, dn, dns)
    assert ref.inside(got, want, bound) <= 1


def test_experts_fp8_non_finite_rows_stay_theirs(pkg, dev):
    q, xs, gu, gus, dn, dns, g = _layer(50, 128, 8, 64, 4)
    idx, wts = routing(50, 8, 2, "uniform", g)
    clean = _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns)
    q.view(torch.uint8)[7, 5] = 0x7F
    got = _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns)
    assert torch.isnan(got[7]).all()
    got[7] = clean[7]
    assert torch.equal(got, clean)


def test_experts_fp8_empty_same_expert_twice_and_zero_weights(pkg, dev):
    q, xs, gu, gus, dn, dns, g = _layer(6, 64, 8, 32, 9)
    idx, wts = routing(6, 8, 2, "uniform", g)
    assert _run(pkg, dev, q[:0], xs[:0], idx[:0], wts[:0], gu, gus, dn, dns).shape == (0, 64)
    idx[2] = idx[2, 0]  # both of a token's slots name one expert
    wts[3] = 0
    got = _run(pkg, dev, q, xs, idx, wts, gu, gus, dn, dns)
    want, bound = ref.experts(q, xs, idx, wts, gu, gus, dn, dns)
    assert ref.inside(got, want, bound) <= 1
    assert (got[3] == 0).all()


@pytest.mark.parametrize("T", [1, 3, 40, 600])
def test_experts_fp8_streams_and_graphs(pkg, dev, T):
    """Two streams at once; two graphs of one capture stream, replayed in turn and with other inputs."""
    q, xs, gu, gus, dn, dns, g = _layer(2 * T, 128, 8, 64, 11)
    idx, wts = routing(2 * T, 8, 4, "uniform", g)
    d = [t.to(dev) for t in (q, xs, idx, wts, gu, gus, dn, dns)]
    half = [[t[:T] for t in d[:4]], [t[T:] for t in d[:4]]]
    call = lambda a: pkg.ops.experts_fp8(*a, d[4], d[6], gate_up_scale=d[5], down_scale=d[7])  # noqa: E731
    want = [call(a) for a in half]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            got.append(call(half[i % 2]))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        assert torch.equal(t, want[i % 2])
    graphs = []
    for i in range(2):
        static = [t.clone() for t in half[i]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[0]):
            out = call(static)
        graphs.append((graph, static, out))
    for i in range(4):
        for j, (graph, static, out) in enumerate(graphs):
            for s, h in zip(static, half[(i + j) % 2]):
                s.view(torch.uint8).copy_(h.contiguous().view(torch.uint8))
        torch.cuda.synchronize()
        for j, (graph, _, _) in enumerate(graphs):  # both at once
            with torch.cuda.stream(side[j]):
                graph.replay()
        torch.cuda.synchronize()
        for j, (_, _, out) in enumerate(graphs):
            assert torch.equal(out, want[(i + j) % 2]), (i, j)
        call(half[0])
        torch.cuda.synchronize()


def test_experts_fp8_refusals(pkg, dev):
    q, xs, gu, gus, dn, dns, g = _layer(4, 64, 8, 32, 2)
    idx, wts = routing(4, 8, 2, "uniform", g)
    good = dict(q=q, scale=xs, top_k_index=idx, top_k_weights=wts, gate_up=gu, down=dn, gate_up_scale=gus,
                down_scale=dns)
    good = {k: v.to(dev) for k, v in good.items()}
    pkg.ops.experts_fp8(**good)
    bf = lambda t: t.float().to(BF16)  # noqa: E731
    for name, t in (("q", bf(good["q"])), ("q", good["q"][None]), ("q", good["q"][:, :32]), ("scale", good["scale"][:3]),
                    ("scale", None), ("top_k_index", good["top_k_index"].int()), ("top_k_index", good["top_k_index"][:3]),
                    ("top_k_weights", good["top_k_weights"][:, :1]), ("gate_up", bf(good["gate_up"])),
                    ("gate_up", good["gate_up"].transpose(1, 2)), ("down", bf(good["down"])), ("down", good["down"][:7]),
                    ("gate_up_scale", good["gate_up_scale"][:, :60]), ("gate_up_scale", None),
                    ("down_scale", good["down_scale"].double()), ("scale", good["scale"].cpu())):
        with pytest.raises((ValueError, pkg.MoeLibraryError)):
            pkg.ops.experts_fp8(**{**good, name: t})


@pytest.mark.parametrize("E", [8, 200])
@pytest.mark.parametrize("T", [1, 5, 40, 300])
def test_experts_fp8_with_shared_and_residual_is_combine(pkg, dev, T, E):
    q, xs, gu, gus, dn, dns, g = _layer(T, 96, E, 64, T + 20)
    idx, wts = routing(T, E, 4, "uniform", g)
    shared, res = (torch.randn(T, 96, generator=g).to(BF16).to(dev) for _ in range(2))
    gate = (torch.randn(T, 7, generator=g) * 4).to(BF16).to(dev)[:, 3]
    args = [t.to(dev) for t in (q, xs, idx, wts, gu, dn)]
    call = lambda **kw: pkg.ops.experts_fp8(*args, gate_up_scale=gus.to(dev), down_scale=dns.to(dev), **kw)  # noqa: E731
    routed, one = call(), torch.ones(T, 1, dtype=BF16, device=dev)
    for s, r in ((None, res), (shared, None), (shared, res)):
        want = pkg.ops.combine(routed, one, shared=s, shared_gate_logit=None if s is None else gate, residual=r)
        kw = {} if s is None else dict(shared=s, shared_gate_logit=gate)
        assert torch.equal(call(residual=r, **kw), want)
    wide = torch.zeros(T, 200, dtype=BF16, device=dev)  # views, one at an odd address
    wide[:, 5:101], wide[:, 104:] = shared, res
    assert torch.equal(call(shared=wide[:, 5:101], shared_gate_logit=gate.contiguous(), residual=wide[:, 104:]),
                       call(shared=shared, shared_gate_logit=gate, residual=res))
    for bad in (dict(shared=shared), dict(shared=shared, shared_gate_logit=gate[:-1]), dict(residual=res[:, :64]),
                dict(shared=shared[:, :64], shared_gate_logit=gate), dict(residual=res.float()),
                dict(shared=shared, shared_gate_logit=gate.float()), dict(shared=shared, shared_gate_logit=gate[:, None]),
                dict(residual=res.cpu())):
        with pytest.raises((ValueError, pkg.MoeLibraryError)):
            call(**bad)
