"""fp64 statements of the serving operators on the CPU, and the error bounds
the tests hold the kernels to.

Bounds (u = the output type's unit roundoff):
* rope: one rounding of the result, u |y|, and the fp32 products and sum,
  3 * 2^-24 (|x1 c| + |x2 s|).
* attention: rounding of the result, u |o|; rounding of the softmax weights
  to the element type, u sum w |v| (fp16 weights below 2^-14 of the row's
  largest lose up to 2^-25 each: n 2^-25 max|v|); the fp32 score sum over D
  terms, off by at most e = (D + 2) 2^-23 scale max_j sum_d |q_d k_jd|, which
  moves the weights by 2e relative; and 2^-20 for exp2 and the fp32 row sums.
* lse: e + 2^-20 (1 + |lse|).
"""
import math

import torch

ROUNDOFF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def rotate(x, pos, table, interleaved=False, inverse=False):
    """(y, bound) of the rotation of x [tokens, heads, D] in fp64."""
    u = ROUNDOFF[x.dtype]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    x = x.double()
    rot = table.shape[1]
    t = table.double()[pos.long()][:, None]
    c, s = t[..., :rot // 2], t[..., rot // 2:] * (-1.0 if inverse else 1.0)
    y = x.clone()
    b = torch.zeros_like(x)
    i = torch.arange(rot // 2)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    x1, x2 = x[..., first], x[..., second]
    y[..., first], y[..., second] = x1 * c - x2 * s, x2 * c + x1 * s
    b[..., first] = 3 * 2.0 ** -24 * ((x1 * c).abs() + (x2 * s).abs())
    b[..., second] = 3 * 2.0 ** -24 * ((x2 * c).abs() + (x1 * s).abs())
    return y, b + u * y.abs() + tiny


def attend(q, k, v, seen, scale=None):
    """(o, lse, o's bound, lse's bound) of one sequence: q [n, Hq, D], k/v [m, Hk, D], seen bool [n, m]."""
    u = ROUNDOFF[q.dtype]
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    n, hq, d = q.shape
    m, hk, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    k, v = (x.repeat_interleave(hq // hk, dim=1) for x in (k, v))
    live = seen.any(1)
    hide = ~seen[None]
    s = (torch.einsum("nhd,mhd->hnm", q, k) * scale).masked_fill(hide, -math.inf)
    size = (torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()) * scale).masked_fill(hide, 0.0)
    e = (d + 2) * 2.0 ** -23 * (size.amax(2) if m else torch.zeros(hq, n, dtype=torch.float64))
    lse = torch.logsumexp(s, 2) if m else torch.full((hq, n), -math.inf, dtype=torch.float64)
    w = torch.exp(s - torch.where(live, lse, torch.zeros_like(lse))[..., None]).masked_fill(hide, 0.0)
    o = torch.einsum("hnm,mhd->nhd", w, v)
    mass = torch.einsum("hnm,mhd->nhd", w, v.abs())
    most = v.abs().amax(0)[None] if m else 0.0  # [1, Hq, D]
    e = e.T[..., None]
    bound = u * o.abs() + (u + 2 * e + 2.0 ** -20) * mass + tiny * m * most + 1e-30
    bound = bound + tiny  # fp16 results below 2^-14
    lse_bound = e[..., 0] + 2.0 ** -20 * (1 + lse.T.abs().nan_to_num(posinf=0.0))
    return o, lse.T, bound, lse_bound


def causal(n, m):
    i, j = torch.arange(n)[:, None], torch.arange(m)[None]
    return j <= i + m - n


def tree_seen(ctx, parents):
    """bool [nodes, ctx + nodes] from the parents of one tree."""
    n = len(parents)
    seen = torch.zeros(n, ctx + n, dtype=torch.bool)
    seen[:, :ctx] = True
    for i in range(n):
        j = i
        while j >= 0:
            seen[i, ctx + j] = True
            j = parents[j]
    return seen


def bits_of(seen_nodes, words):
    """int32 words of a bool [nodes, nodes] matrix."""
    rows = []
    for r in seen_nodes.tolist():
        v = sum(1 << j for j, on in enumerate(r) if on)
        w = [(v >> (32 * i)) & 0xFFFFFFFF for i in range(words)]
        rows.append([x - (1 << 32) if x >> 31 else x for x in w])
    return torch.tensor(rows, dtype=torch.int32).view(len(rows), words)


def assert_within(got, want, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    ok = ~nan & ~inf
    over = ((got - want).abs() - bound.expand_as(want))[ok]
    assert over.numel() == 0 or over.max() <= 0, \
        f"{what}: {(over > 0).sum().item()} of {over.numel()} values off by up to {over.max().item():.3g} past the bound"
