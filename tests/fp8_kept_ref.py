"""experts_fp8 in 64 bits with a bound for each way that its kernels take, on the CPU (test infrastructure).

- ``kept``: every product counts in the fp32 sums (few rows); else the e4m3 matrix instruction cuts some
  (``fp8_ref.dropped``).
- ``stored``: the pairs' outputs go to the weighted sum as fp16 with a power of two per 32 columns; else
  (as many pairs as 16, or a quarter of the experts) in fp32.
- ``whole``: the operands' sums of products are whole numbers below 2^24, exact in any order.
"""

from __future__ import annotations

import torch

from tests.fp8_ref import dropped, groups


def few(idx, experts):
    return idx.numel() <= max(16, experts // 4)


def kept(idx, experts):
    return idx.numel() <= 12 * experts


def as_stored(y):
    """By how much y [rows, n] may change on its way through fp16: half a step of 2^-10 of a value (2^-11 of
    it), at the least half of fp16's last place, 2^-25, where the largest of 32 columns lies between 2^14
    and 2^15: 2^-39 of that largest."""
    amax = y.abs().reshape(y.shape[0], -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(y.shape)
    return torch.maximum(y.abs() * 2.0**-11, amax * 2.0**-39) + 2.0**-145


def experts(q, xs, idx, wts, gu, gus, dn, dns, whole=False, plant=None):
    """(result [T, H], bound) in float64. fp32 sums as in fp8_ref.linear; a value of the 8-bit product in
    between may fall to its neighbour where that bound reaches the middle; the pairs' outputs as stored;
    the weighted sum in fp32, and one rounding of the result to bf16 (2^-8). ``plant``: a mistake
    to be seen by the bound, applied to each pair's output."""
    tokens, hidden = q.shape
    k, inter, count = idx.shape[1], gu.shape[1] // 2, gu.shape[0]
    out = torch.zeros(tokens, hidden, dtype=torch.float64)
    off = torch.zeros_like(out)
    cut = (lambda x, w: 0.0) if kept(idx, count) else dropped
    for e in torch.unique(idx).tolist():
        t, j = torch.nonzero(idx == e, as_tuple=True)
        x, w = q[t].double(), gu[e].double()
        both, s = x @ w.t(), xs[t].double()[:, None] * gus[e].double()
        eb = cut(x, w) + (0.0 if whole else (x.abs() @ w.abs().t()) * (hidden + 8) * 2.0**-23)
        both, eb = both * s, (eb + both.abs() * 2.0**-22) * s
        g, u, eg, eu = both[:, :inter], both[:, inter:], eb[:, :inter], eb[:, inter:]
        s = g * torch.sigmoid(g)
        a = s * u
        ea = 1.1 * eg * (u.abs() + eu) + s.abs() * eu + a.abs() * 2.0**-19 + 2.0**-126
        b, slack = groups(a, ea)
        w = dn[e].double()
        size = b.abs() @ w.abs().t()
        y, ey = b @ w.t(), slack @ w.abs().t() + cut(b, w) + size * (inter + 8) * 2.0**-23
        y, ey = y * dns[e].double(), ey * dns[e].double()
        if not few(idx, count):
            ey = ey + as_stored(y) * 1.01
        if plant is not None:
            y = plant(y)
        ww = wts.double()[t, j][:, None]
        out.index_add_(0, t, y * ww)
        off.index_add_(0, t, (ey + (y.abs() + ey) * (k + 2) * 2.0**-23) * ww.abs())
    return out, off + (out.abs() + off) * 2.0**-8 + 2.0**-133
