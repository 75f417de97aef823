"""Paged caches and the 64-bit forms that the tests of the drafted tokens' and
the selected blocks' attention compare with (CPU side)."""
import math

import torch

from oracle import exact, restate

ALPHA = math.sqrt(2.0 / math.pi) / 128


def codebooks(H, seed=11):
    """Ascending levels for N(0, 1), each head's times a factor of its own."""
    half = torch.tensor([0.1284, 0.3881, 0.6568, 0.9424, 1.2562, 1.6181, 2.0690, 2.7326])
    g = torch.Generator().manual_seed(seed)
    return torch.cat((-half.flip(0), half))[None, :] * (0.7 + 0.6 * torch.rand(H, 1, generator=g))


def packed(B, H, S, seed):
    """A contiguous packed cache of N(0, 1) keys and values: codes of the levels' bins, norms and signs of their residuals'
    sizes."""
    g = torch.Generator().manual_seed(seed)
    level = codebooks(1)[0] / codebooks(1)[0, -1] * 2.7326
    mid = (level[1:] + level[:-1]) / 2
    kc, vc = (torch.bucketize(torch.randn(B, H, S, 128, generator=g), mid).to(torch.uint8) for _ in range(2))
    kn, vn = (c[..., 0::2] | (c[..., 1::2] << 4) for c in (kc, vc))
    kq = torch.randint(0, 256, (B, H, S, 8), generator=g, dtype=torch.uint8)
    kr = 1.1 + 0.1 * torch.rand(B, H, S, generator=g)
    return kn, kq, kr, vn


def codes(nib):
    return torch.stack((nib & 15, nib >> 4), -1).flatten(-2).long()


def keys_values(kn, kq, kr, vn, cb, uid, with_qjl=True):
    """float64 K^ and V^ (B, H, S, 128)."""
    H = kn.shape[1]
    c = cb.double() if cb.dim() == 2 else cb.double()[None].expand(H, 16)
    k = torch.stack([c[h][codes(kn[:, h])] for h in range(H)], 1)
    v = torch.stack([c[h][codes(vn[:, h])] for h in range(H)], 1)
    if with_qjl:
        bits = ((kq[..., None] >> torch.arange(8, dtype=torch.uint8)) & 1).flatten(-2).double() * 2 - 1
        G = torch.stack([torch.as_tensor(exact.g_from_mt(restate.make_qjl_seed(uid, h), 128)) for h in range(H)]).double()
        k = k + (bits @ G[None]) * (kr.double() * ALPHA)[..., None]
    return k, v


def rotated(q, flip):
    """float64 rows times the signs and the normalized Hadamard matrix."""
    i = torch.arange(128)
    odd = sum(((i[:, None] & i[None, :]) >> b) & 1 for b in range(7)) % 2
    x = q.double() if flip is None else q.double() * flip.double()
    return x @ ((1.0 - 2.0 * odd.double()) / math.sqrt(128.0))


def attend(q, k, v, visible, scale, dtype, rounded):
    """One head's rows: float64 q (R, 128), k and v (S, 128), visible (R, S).
    Returns the result and how far an output of `dtype` may be off: the
    output's half step; P's, which counts in numerator and denominator (2^-11
    each way), and the centroids' of V (2^-11); the scores' error, which changes
    every weight by its size, in numerator and denominator: of the fp16 centroids
    and (`rounded`) of the fp16 rows 2^-11 of each product, of G q 2^-11 of the
    signs' part, which sum |q k| covers too; fp16 calls keep 22 bits instead;
    fp32 sums of 128 + 64 products 2^-16."""
    s = (q @ k.T) * scale
    s = torch.where(visible, s, -math.inf)
    p = torch.exp(s - s.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    o = p @ v
    per = 2.0 ** -11 * (2 if rounded else 1) if dtype == torch.bfloat16 else 3 * 2.0 ** -22
    size = (q.abs() @ k.abs().T) * abs(scale)
    # the signs' part of k^ can be smaller than the sum of its terms: norm alpha sum |G q| <= norm alpha 64 max |G q|
    err = torch.where(visible, size, 0.0).amax(1, keepdim=True) * (2 * per + 2.0 ** -16)
    bound = (p @ v.abs()) * (2 * err + 3 * 2.0 ** -11) + torch.finfo(dtype).eps / 2 * o.abs() + 1e-6
    return o, bound


def close(got, want, bound, tag=""):
    """NaN where wanted, and within the bound elsewhere."""
    got = got.double().cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{tag}: NaN in other places"
    off = torch.where(nan, 0.0, (got - want).abs() - bound)
    assert float(off.max()) <= 0.0, f"{tag}: {float((got - want).abs()[~nan].max()):.3e} off, by {float(off.max()):.3e} too much"


def paged(device, parts, page_size, lens=None, seed=0, spare=3, **kw):
    from omnistack_rs.cache import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    return PagedKVCache.from_contiguous(*(t.to(device) for t in parts), page_size=page_size, seq_lens=lens, spare_pages=spare,
                                        generator=g, **kw)


def random_parents(B, T, seed):
    g = torch.Generator().manual_seed(seed)
    back = torch.randint(1, 5, (B, T), generator=g)
    return (torch.arange(T)[None, :] - back).clamp_min(-1)
