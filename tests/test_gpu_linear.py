"""ops.linear against 64 bits: sizes, types, every operand of the epilogue, views, rows that are
not finite, streams and graphs."""

from __future__ import annotations

import pytest
import torch

from tests import fp8_ref as ref
from tests.helpers import BF16

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def _operands(M, K, N, e4m3, seed):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(M, K, generator=g).to(BF16), (torch.randn(N, K, generator=g) * K**-0.5).to(BF16)
    if not e4m3:
        return x, w, None, None
    (x, xs), (w, ws) = ref.rows(x), ref.rows(w)
    return x, w, xs, ws


def _epilogue(M, N, bias, mul, residual, seed):
    g = torch.Generator().manual_seed(seed + 99)
    b = torch.randn(N, generator=g)
    m, r = torch.randn(M, N, generator=g).to(BF16), torch.randn(M, N, generator=g).to(BF16)
    return (None if not bias else b.to(BF16) if bias == "bf16" else b, m if mul else None,
            r if residual else None)


def _check(pkg, dev, M, K, N, e4m3, act=None, bias=None, mul=False, residual=False, seed=0):
    x, w, xs, ws = _operands(M, K, N, e4m3, seed)
    b, m, r = _epilogue(M, N, bias, mul, residual, seed)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = pkg.ops.linear(to(x), to(w), x_scale=to(xs), w_scale=to(ws), bias=to(b), activation=act,
                         mul=to(m), residual=to(r))
    again = pkg.ops.linear(to(x), to(w), x_scale=to(xs), w_scale=to(ws), bias=to(b), activation=act,
                           mul=to(m), residual=to(r))
    assert got.shape == (M, N) and got.dtype == BF16 and torch.equal(got, again)
    want, bound = ref.linear(x, w, xs, ws, b, act, m, r)
    share = ref.inside(got, want, bound)
    print(f"linear {M}x{K}x{N} e4m3={e4m3}: {share:.3f} of the bound", flush=True)
    assert share <= 1


SIZES = [(1, 16, 1), (1, 48, 5), (2, 2048, 33), (15, 144, 16), (16, 4096, 40), (17, 80, 31), (31, 272, 96),
         (64, 128, 64), (65, 176, 257), (100, 1040, 130), (129, 512, 512), (200, 96, 1000), (257, 1184, 300),
         (513, 64, 129), (1, 8192, 1000), (300, 4096, 264), (600, 640, 520)]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_sizes(pkg, dev, M, K, N, e4m3):
    _check(pkg, dev, M, K, N, e4m3, seed=M + K + N)
    _check(pkg, dev, M, K, N, e4m3, "silu", "bf16", True, True, seed=M + K + N + 1)


@pytest.mark.parametrize("K", [8, 24, 40, 56, 72, 136, 2040])
def test_linear_bf16_rows_of_odd_multiples_of_eight(pkg, dev, K):
    _check(pkg, dev, 5, K, 37, False, seed=K)
    _check(pkg, dev, 150, K, 150, False, seed=K + 1)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,e4m3", [(3, 50, False), (140, 132, False), (140, 133, True), (700, 513, True)])
def test_linear_epilogues(pkg, dev, act, M, N, e4m3):
    for i, (bias, mul, residual) in enumerate([(None, False, False), ("bf16", False, True), ("fp32", True, False),
                                               ("fp32", True, True)]):
        _check(pkg, dev, M, 192, N, e4m3, act, bias, mul, residual, seed=i)


def test_linear_activation_far_from_zero(pkg, dev):
    """Results that are tiny next to their inputs (gelu and silu at -3 .. -12) keep their digits: half a
    bf16 step of a value computed to 2^-19 or better of itself."""
    v = torch.linspace(-12, 12, 512).to(BF16)
    x, w = torch.zeros(1, 16, dtype=BF16), torch.zeros(512, 16, dtype=BF16)
    for act in ACTS[1:]:
        got = pkg.ops.linear(x.to(dev), w.to(dev), bias=v.to(dev), activation=act)[0].double().cpu()
        want = ref.act(v.double(), act)
        tail = 2.0**-17 if act.startswith("gelu") else 2.0**-19  # exp's argument reaches -90
        assert ((got - want).abs() <= want.abs() * (2.0**-8 + tail) + 2.0**-133).all(), act


@pytest.mark.parametrize("e4m3", [False, True])
def test_linear_leading_dimensions_and_views(pkg, dev, e4m3):
    x, w, xs, ws = (None if t is None else t.to(dev) for t in _operands(60, 256, 96, e4m3, 5))
    base = pkg.ops.linear(x, w, x_scale=xs, w_scale=ws)
    kw = dict(x_scale=None if xs is None else xs.view(3, 4, 5), w_scale=ws)
    res = torch.randn(3, 4, 5, 96, device=dev).to(BF16)
    assert torch.equal(pkg.ops.linear(x.view(3, 4, 5, 256), w, **kw), base.view(3, 4, 5, 96))
    got = pkg.ops.linear(x.view(3, 4, 5, 256), w, residual=res, **kw)
    assert torch.equal(got, pkg.ops.linear(x, w, x_scale=xs, w_scale=ws, residual=res.view(60, 96)).view_as(got))
    # rows inside wider ones (aligned: in place), every other row, columns first, odd addresses
    u8 = torch.uint8 if e4m3 else BF16
    wide = torch.zeros(60, 512, dtype=u8, device=dev)
    wide[:, 64:320] = x.view(u8)
    assert torch.equal(pkg.ops.linear(wide[:, 64:320].view(x.dtype), w, x_scale=xs, w_scale=ws), base)
    packed = torch.zeros(96, 320, dtype=u8, device=dev)
    packed[:, 32:288] = w.view(u8)
    assert torch.equal(pkg.ops.linear(x, packed[:, 32:288].view(w.dtype), x_scale=xs, w_scale=ws), base)
    odd = torch.zeros(60 * 256 + 1, dtype=u8, device=dev)
    odd[1:] = x.reshape(-1).view(u8)
    assert torch.equal(pkg.ops.linear(odd[1:].view(60, 256).view(x.dtype), w, x_scale=xs, w_scale=ws), base)
    if not e4m3:
        assert torch.equal(pkg.ops.linear(x.t().contiguous().t(), w), base)
        assert torch.equal(pkg.ops.linear(x[::2], w), base[::2])
        one = pkg.ops.linear(x[0], w)
        assert one.shape == (96,) and torch.equal(one, pkg.ops.linear(x[:1], w)[0])
        assert torch.equal(pkg.ops.linear(x[:1].expand(60, 256), w)[59:], pkg.ops.linear(x[:1].expand(60, 256), w)[:1])
        assert torch.equal(pkg.ops.linear(x, w, mul=res.view(60, 96).t().contiguous().t()),
                           pkg.ops.linear(x, w, mul=res.view(60, 96)))


def test_linear_empty(pkg, dev):
    x, w = torch.randn(4, 64, device=dev).to(BF16), torch.randn(6, 64, device=dev).to(BF16)
    assert pkg.ops.linear(x[:0], w).shape == (0, 6)
    assert pkg.ops.linear(x, w[:0]).shape == (4, 0)
    assert pkg.ops.linear(x.view(2, 2, 64)[:, :0], w).shape == (2, 0, 6)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("M,N", [(20, 70), (300, 300)])
def test_linear_non_finite_rows_stay_in_their_row(pkg, dev, M, N, e4m3):
    x, w, xs, ws = _operands(M, 208, N, e4m3, 8)
    clean = pkg.ops.linear(*(t.to(dev) for t in (x, w)), x_scale=None if xs is None else xs.to(dev),
                           w_scale=None if ws is None else ws.to(dev)).cpu()
    nan = 0x7F if e4m3 else 0x7FC0
    view = torch.uint8 if e4m3 else torch.int16
    x.view(view)[3, 207] = nan
    w.view(view)[N - 1, 0] = nan
    got = pkg.ops.linear(*(t.to(dev) for t in (x, w)), x_scale=None if xs is None else xs.to(dev),
                         w_scale=None if ws is None else ws.to(dev)).cpu()
    bad = torch.isnan(got)
    assert bad[3].all() and bad[:, N - 1].all() and bad.sum() == N + M - 1
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("M,N", [(3, 17), (130, 131), (300, 520)])
def test_linear_writes_nothing_behind_its_rows(pkg, dev, M, N, e4m3):
    x, w, xs, ws = (None if t is None else t.to(dev) for t in _operands(M, 64, N, e4m3, 6))
    out = torch.full((M * N + 4096,), 7.0, dtype=BF16, device=dev)
    p = pkg._lib.ptr
    rc = pkg._lib.load().moe_linear(p(x), 64, p(xs), p(w), 64, p(ws), int(e4m3), M, 64, N, None, 0, 0, None, None,
                                    p(out), pkg._lib.stream_of(x))
    pkg._lib.check(rc, "linear")
    assert torch.equal(out[:M * N].view(M, N), pkg.ops.linear(x, w, x_scale=xs, w_scale=ws))
    assert (out[M * N:] == 7).all()


@pytest.mark.parametrize("M,N,e4m3", [(4, 512, False), (200, 300, True), (1000, 700, False)])
def test_linear_streams_and_graphs(pkg, dev, M, N, e4m3):
    """Two streams at once, and one graph replayed with other inputs."""
    x, w, xs, ws = (None if t is None else t.to(dev) for t in _operands(M, 512, N, e4m3, 4))
    x2 = x.flip(0).contiguous() if not e4m3 else x.view(torch.uint8).flip(0).contiguous().view(x.dtype)
    xs2 = None if xs is None else xs.flip(0).contiguous()
    want, want2 = (pkg.ops.linear(a, w, x_scale=s, w_scale=ws, activation="gelu") for a, s in ((x, xs), (x2, xs2)))
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            got.append(pkg.ops.linear((x, x2)[i % 2], w, x_scale=(xs, xs2)[i % 2], w_scale=ws, activation="gelu"))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        assert torch.equal(t, (want, want2)[i % 2])
    u8 = torch.uint8
    static, sscale = x.clone(), None if xs is None else xs.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.ops.linear(static, w, x_scale=sscale, w_scale=ws, activation="gelu")
    for i in range(4):
        static.view(u8).copy_((x, x2)[i % 2].view(u8))
        if xs is not None:
            sscale.copy_((xs, xs2)[i % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, (want, want2)[i % 2]), i
        pkg.ops.linear(x, w, x_scale=xs, w_scale=ws)
        torch.cuda.synchronize()


def test_linear_refusals(pkg, dev):
    lin = pkg.ops.linear
    x, w = torch.zeros(4, 64, device=dev, dtype=BF16), torch.zeros(6, 64, device=dev, dtype=BF16)
    q, s = pkg.ops.quantize_rows(x)
    wq, ws = pkg.ops.quantize_rows(w)
    for bad in (lambda: lin(x, w, activation="tanh"), lambda: lin(x, wq), lambda: lin(x.float(), w.float()),
                lambda: lin(x, w[:, :32]), lambda: lin(x, w.view(2, 3, 64)), lambda: lin(x, w, x_scale=s),
                lambda: lin(q, wq), lambda: lin(q, wq, x_scale=s, w_scale=ws[:5]),
                lambda: lin(q, wq, x_scale=s.double(), w_scale=ws), lambda: lin(x, w.t().contiguous().t()),
                lambda: lin(x, torch.zeros(6 * 64 + 1, device=dev, dtype=BF16)[1:].view(6, 64)),
                lambda: lin(x, w, bias=torch.zeros(5, device=dev)), lambda: lin(x, w, bias=s[:4].half()),
                lambda: lin(x, w, mul=torch.zeros(4, 5, device=dev, dtype=BF16)),
                lambda: lin(x, w, residual=torch.zeros(4, 6, device=dev)), lambda: lin(x[:, :4], w[:, :4]),
                lambda: lin(x, w, bias=torch.zeros(6))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("M,K", [(1, 40), (20, 200), (70, 72), (300, 2056)])
def test_linear_infinite_weights_and_rows_stay_infinite(pkg, dev, M, K):
    """An infinity in the last columns, beside bytes past a row's end, is no NaN: positive rows times a
    weight of plus and one of minus infinity, and the other way round."""
    g = torch.Generator().manual_seed(K)
    x, w = (torch.rand(M, K, generator=g) + 0.5).to(BF16), (torch.rand(40, K, generator=g) + 0.5).to(BF16)
    w[3, K - 1], w[5, K - 8], w[39, 0] = torch.inf, -torch.inf, torch.inf
    got = pkg.ops.linear(x.to(dev), w.to(dev)).float().cpu()
    for n, sign in ((3, 1), (5, -1), (39, 1)):
        assert (got[:, n] == sign * torch.inf).all(), n
    rest = [n for n in range(40) if n not in (3, 5, 39)]
    assert torch.isfinite(got[:, rest]).all()
    x[0, K - 1] = -torch.inf
    got = pkg.ops.linear(x.to(dev), w.to(dev)).float().cpu()
    assert (got[0, rest] == -torch.inf).all() and torch.isfinite(got[1:, rest]).all()


def test_linear_activations_of_huge_values(pkg, dev):
    """Values whose square leaves fp32, and infinity: the identity above zero, zero below (bf16 of a finite
    value up to its largest is itself)."""
    v = torch.tensor([1e19, 1e20, 3e38, 1e30], dtype=BF16)
    x, w = torch.zeros(1, 16, dtype=BF16), torch.zeros(8, 16, dtype=BF16)
    for act in ACTS[1:]:
        got = pkg.ops.linear(x.to(dev), w.to(dev), bias=torch.cat([v, -v]).to(dev), activation=act)[0].cpu()
        assert torch.equal(got[:4], v), act
        assert (got[4:] == 0).all(), act
        inf = torch.full((8,), torch.inf, dtype=BF16, device=dev)
        assert (pkg.ops.linear(x.to(dev), w.to(dev), bias=inf, activation=act) == torch.inf).all(), act


def test_rows_and_linear_of_no_columns_are_refused(pkg, dev):
    w, scalar = torch.zeros(0, dtype=BF16, device=dev), torch.zeros((), dtype=BF16, device=dev)
    for x in (torch.zeros(3, 0, dtype=BF16, device=dev), scalar):
        for call in (lambda: pkg.ops.quantize_rows(x), lambda: pkg.ops.add_rms_fp8(x, None, w, 1e-6),
                     lambda: pkg.ops.linear(x, torch.zeros(4, 0, dtype=BF16, device=dev))):
            with pytest.raises(ValueError):
                call()
