"""Plain 64-bit forms of the attention operators over a paged cache, and how far a kernel may be from them.

The bounds follow from the roundings the operators state (include/vwsampler.h).  With u = 2^-8 (bf16: 8
significant bits) and w = 2^-24 (fp32) as the largest relative error of one rounding to nearest:

* a score is an fp32 sum of D products: off by at most d = (D + 4) w scale sum|q k|; the largest over a row's keys bounds
  the relative error of every probability;
* a probability is rounded to bf16 (u), its exponential and the sums are fp32; so an output is off by at most
  u |out| (its own rounding) + (u + 2 d + n w + 2^-20) A, A the same average of |v| (n keys, 2^-20 for two exponentials
  of 2^-22 each and the rescaling of running sums);
* lse is off by at most d + n w + 2^-20 + 4 w |lse|.
"""

import torch

U, W = 2.0 ** -8, 2.0 ** -24


def keys_of(cache, table_row, n):
    """The first n rows of a sequence's pages, [n, heads, dim] in 64 bits."""
    size = cache.shape[1]
    j = torch.arange(n, device=cache.device)
    return cache[table_row.long()[j // size], j % size].double()


def attend(q, k, v, scale, limit=None):
    """q [r, H, D] over k, v [n, Hkv, D]; row i sees keys j < limit[i] (None: all).  out, lse and their bounds."""
    r, H, D = q.shape
    n, kv = k.shape[0], k.shape[1]
    q = q.double()
    kk, vv = (x.repeat_interleave(H // kv, dim=1) for x in (k, v))
    z = torch.einsum("rhd,nhd->rhn", q, kk) * scale
    seen = torch.ones((r, n), dtype=torch.bool, device=q.device)
    if limit is not None:
        seen = torch.arange(n, device=q.device)[None] < limit[:, None]
    z = torch.where(seen[:, None], z, torch.full_like(z, -float("inf")))
    d = torch.einsum("rhd,nhd->rhn", q.abs(), kk.abs()) * abs(scale) * (D + 4) * W
    d = torch.where(seen[:, None], d, torch.zeros_like(d)).amax(-1) if n else torch.zeros((r, H), device=q.device).double()
    lse = torch.logsumexp(z, dim=-1) if n else torch.full((r, H), -float("inf"), device=q.device).double()
    p = torch.exp(z - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None])
    vv = torch.where(seen.any(0)[:, None, None], vv, torch.zeros_like(vv)) if r else vv
    out = torch.einsum("rhn,nhd->rhd", p, vv)
    mean = torch.einsum("rhn,nhd->rhd", p, vv.abs())
    out_bound = U * out.abs() + (U + 2 * d + n * W + 2.0 ** -20)[..., None] * mean
    lse_bound = d + n * W + 2.0 ** -20 + 4 * W * torch.where(torch.isinf(lse), torch.zeros_like(lse), lse).abs()
    return out, lse, out_bound, lse_bound


def check(got, want, bound, what):
    """got within bound of want, with a rounding's slack on the bound itself; not-finite values equal."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"{what}: finite where the formula is not, or the other way round"
    assert torch.equal(got[~fine], want[~fine]), f"{what}: infinities differ"
    if fine.any():
        over = ((got - want).abs() - 1.01 * bound - 1e-30)[fine]
        assert bool((over <= 0).all()), f"{what}: off by up to {float((got - want).abs()[fine].max()):.3e}, " \
                                        f"{int((over > 0).sum())} of {over.numel()} over the bound"


def rope(x, weight, eps, cos, sin, interleaved):
    """x [n, H, D] normalised and turned in 64 bits (cos, sin [n, R / 2]), and the bound of an fp32 pass rounded to bf16."""
    x = x.double()
    D = x.shape[-1]
    if weight is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    y, size = x.clone(), x.abs()
    if cos is not None and cos.shape[-1]:
        half = cos.shape[-1]
        i = torch.arange(half, device=x.device)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos.double()[:, None], sin.double()[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        size = size.clone()
        size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
        size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, U * y.abs() + (D + 8) * W * size
