"""Plain 64-bit attention of packed rows and of pages, and the tolerance of the tests that compare with it.

For output o = sum_j p_j v_j with A = sum_j p_j |v_j| and S the row's largest sum of |q k| products in units of log2:
  2^-8 A    P (E4M3: P times its key's scale) rounded to bf16 before the product with V, half a step of each weight
            (the sum l is not rounded)
  2^-12 A   the exponentials' relative error (below 2^-13), once in the weights and once in their sum
  2^-16 S A a score is D <= 128 products added in fp32, each addition off by at most 2^-23 of the largest partial sum:
            128 2^-23 S = 2^-16 S in the exponent, times ln 2 for the weight, once in the weights and once in the sum
  2^-8 |o|  the output rounded to bf16
and 2^-20 A for the fp32 sums over the keys and the joined parts.

Where the scores are exact (one product each), S counts as min(S, 2^12) / 2^5 instead: what is left is the rounding of
score times scale, of the reference maximum times scale and of the polynomial's argument, 3 2^-24 of scores below 2^12
(past that the difference to the maximum is taken first), 6 ln 2 2^-24 < 2^-21 in the weights and their sum.
"""

from __future__ import annotations

import math

import torch

LOG2E = 1.0 / math.log(2.0)


def plain_attention(q, k, v, limit, scale, exact=False):
    """q (n, H, D), k and v (T, KV, D), limit (n,) visible keys of each row.  Returns (out, tolerance) in float64, rows
    without a key zero.  Values behind a row's limit are never used; an infinity or a NaN within it counts."""
    n, H, D = q.shape
    T, KV = k.shape[:2]
    rep = H // KV
    q, k, v = q.double(), k.double(), v.double()
    see = (torch.arange(T, device=q.device)[None, :] < limit[:, None].to(q.device))[:, None]  # n, 1, T
    qg = q.view(n, KV, rep, D)
    s = torch.einsum("nkrd,tkd->nkrt", qg, k).reshape(n, H, T) * scale
    s = torch.where(see, s, -math.inf)
    S = torch.einsum("nkrd,tkd->nkrt", qg.abs(), k.abs()).reshape(n, H, T) * (scale * LOG2E)
    S = torch.where(see & S.isfinite(), S, 0.0).amax(-1, keepdim=True)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l == 0, 0.0, p / l)
    fine = torch.where(v.isfinite(), v, 0.0)
    pg = p.view(n, KV, rep, T)
    out = torch.einsum("nkrt,tkd->nkrd", pg, fine).reshape(n, H, D)
    A = torch.einsum("nkrt,tkd->nkrd", pg, fine.abs()).reshape(n, H, D)
    for t in (~v.isfinite()).any(-1).any(-1).nonzero().flatten().tolist():
        add = torch.where(v[t].isfinite(), 0.0, v[t]).repeat_interleave(rep, 0)  # H, D
        out = torch.where((limit > t)[:, None, None].to(q.device), out + add, out)
    if exact:
        S = S.clamp(max=2.0**12) / 2**5
    tol = A * (2.0**-8 + 2.0**-12 + 2.0**-20 + 2.0**-16 * S) + out.abs() * 2.0**-8 + 1e-30
    return out, tol


def assert_rows(got, want, tol, what=""):
    got = got.double()
    strange = ~want.isfinite()
    same = torch.where(want.isnan(), got.isnan(), got == want)
    assert same[strange].all(), f"{what}: infinities and NaNs differ"
    err = torch.where(strange, 0.0, (got - want).abs())
    assert not err.isnan().any(), f"{what}: {int(err.isnan().sum())} NaNs where there is a value"
    over = err - torch.where(strange, math.inf, tol)
    worst = int(over.argmax())
    assert over.max() <= 0, (f"{what}: |err| {float(err.flatten()[worst]):.3e} over {float(tol.flatten()[worst]):.3e} at "
                             f"{[int(i) for i in torch.unravel_index(torch.tensor(worst), over.shape)]}, "
                             f"{int((over > 0).sum())} of {over.numel()} values")


def packed_case(lens, H, KV, D, seed, *, gap=0, extra=None):
    """Packed prompts: ``lens`` new tokens of each sequence, ``extra`` keys before them, ``gap`` rows of nobody's between
    sequences.  Returns q, k, v (cuda bf16), row0, kv0 and the contexts."""
    extra = extra or [0] * len(lens)
    g = torch.Generator().manual_seed(seed)
    row0, kv0, r, c = [], [], gap, gap
    for n, e in zip(lens, extra):
        row0.append(r)
        kv0.append(c)
        r += n + gap
        c += n + e + gap
    q = torch.randn(max(r, 1), H, D, generator=g).to(torch.bfloat16).cuda()
    k = torch.randn(max(c, 1), KV, D, generator=g).to(torch.bfloat16).cuda()
    v = torch.randn(max(c, 1), KV, D, generator=g).to(torch.bfloat16).cuda()
    return q, k, v, row0, kv0, [n + e for n, e in zip(lens, extra)]


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def make_batch(row0, lens, ctx, rows, q_max=None):
    from specdec_b200.kernels import ops

    return ops.RaggedBatch(i32(row0), i32(lens), i32(ctx), len(lens), q_max or max(max(lens), 1), rows, max(ctx))


def check_packed(out, fill, q, k, v, row0, kv0, lens, ctx, scale=None, what="", skip=(), exact=False):
    """Every sequence's rows against the plain form; the rows of nobody's (and of ``skip``) still hold ``fill``."""
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    left = torch.ones(out.shape[0], dtype=torch.bool)
    for b, (r, c, n, t) in enumerate(zip(row0, kv0, lens, ctx)):
        if n == 0 or b in skip:
            continue
        left[r:r + n] = False
        limit = torch.arange(n) + (t - n + 1)
        want, tol = plain_attention(q[r:r + n], k[c:c + t], v[c:c + t], limit, scale, exact)
        assert_rows(out[r:r + n], want, tol, f"{what} sequence {b}")
    assert torch.equal(out[left.cuda()], torch.full_like(out[left.cuda()], fill)), f"{what}: rows of no sequence changed"


class Pages:
    """A cache with random pages and a table in which the members of a group share their first pages."""

    def __init__(self, ctx, groups, KV, D, v8, seed, *, layers=1, max_pages=None, spare=8):
        from specdec_b200.engine.paged_cache import PagedKVCache

        g = torch.Generator().manual_seed(seed)
        B = len(ctx)
        need = [(-(-t // 16)) for t in ctx]
        mp = max_pages or max(max(need), 1)
        total = B * mp + spare
        free = torch.randperm(total, generator=g).tolist()
        pt = torch.full((B, mp), -1, dtype=torch.int32)
        shared = {}
        for seqs, n in groups:
            ids = None
            for b in seqs:
                if ids is None:
                    ids = [free.pop() for _ in range(min(n // 16, mp))]
                shared[b] = ids
        for b in range(B):
            ids = list(shared.get(b, []))[:need[b]]
            while len(ids) < need[b]:
                ids.append(free.pop())
            pt[b, :need[b]] = torch.tensor(ids, dtype=torch.int32)
        ks = [torch.randn(total, KV, 16 * D, generator=g).to(torch.bfloat16).cuda() for _ in range(layers)]
        vs = [torch.randn(total, KV, 16 * D, generator=g) for _ in range(layers)]
        if v8:
            sc = [(torch.rand(total, KV, 16, generator=g) + 0.25).cuda() for _ in range(layers)]
            vs = [(20 * v).to(torch.float8_e4m3fn).view(torch.uint8).cuda() for v in vs]
        else:
            sc, vs = None, [v.to(torch.bfloat16).cuda() for v in vs]
        self.cache = PagedKVCache.from_pools(ks, vs, sc, pt.cuda(), i32(ctx), D)
        self.ctx, self.KV, self.D, self.v8, self.free = list(ctx), KV, D, v8, free

    def kv(self, b, layer=0, length=None):
        """(k, v) (T, KV, D) of sequence b as the attention sees them."""
        length = self.ctx[b] if length is None else length
        d = self.cache.gather_layer(layer, b, length)
        k, v = d["k"][0].transpose(0, 1), d["v"][0].transpose(0, 1)
        if self.v8:
            v = v.double() * d["v_scale"][0].transpose(0, 1).double()
        return k, v


def check_pages(out, fill, q, pages, row0, lens, ctx, scale=None, layer=0, what="", skip=()):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    left = torch.ones(out.shape[0], dtype=torch.bool)
    for b, (r, n, t) in enumerate(zip(row0, lens, ctx)):
        if n == 0 or b in skip:
            continue
        left[r:r + n] = False
        k, v = pages.kv(b, layer, t)
        want, tol = plain_attention(q[r:r + n], k, v, torch.arange(n) + (t - n + 1), scale)
        assert_rows(out[r:r + n], want, tol, f"{what} sequence {b}")
    assert torch.equal(out[left.cuda()], torch.full_like(out[left.cuda()], fill)), f"{what}: rows of no sequence changed"
