"""Dropout, embedding and sampling from their definitions, on the CPU: random bits by whole numbers, PAM products in 64 bits, probabilities as whole numbers."""
import math

import numpy as np
import torch

from decoding_cases import INF, LOG2E, U, _split, pad, pam  # noqa: F401

F32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
MASK = 2 ** 32 - 1


def philox(counter, key):
    """Philox4x32-10 on Python integers: four words of the 128-bit counter under the 64-bit key."""
    a, b, c, d = (counter >> s & MASK for s in (0, 32, 64, 96))
    k, m = key & MASK, key >> 32 & MASK
    for _ in range(10):
        left, right = 0xD2511F53 * a, 0xCD9E8D57 * c
        a, b, c, d = right >> 32 ^ b ^ k, right & MASK, left >> 32 ^ d ^ m, left & MASK
        k, m = k + 0x9E3779B9 & MASK, m + 0xBB67AE85 & MASK
    return a, b, c, d


def kept(seed, first, last, p):
    """Which of the elements first .. last - 1 stay."""
    blocks = np.arange(first // 4, (last + 3) // 4, dtype=np.uint64)
    a, b = blocks & np.uint64(MASK), blocks >> np.uint64(32)
    c = d = np.zeros_like(a)
    k, m, low = seed & MASK, seed >> 32 & MASK, np.uint64(MASK)
    for _ in range(10):
        left, right = np.uint64(0xD2511F53) * a, np.uint64(0xCD9E8D57) * c
        a, b, c, d = right >> np.uint64(32) ^ b ^ np.uint64(k), right & low, left >> np.uint64(32) ^ d ^ np.uint64(m), left & low
        k, m = k + 0x9E3779B9 & MASK, m + 0xBB67AE85 & MASK
    words = np.stack([a, b, c, d], 1).reshape(-1)
    start = first // 4 * 4
    return torch.from_numpy(words[first - start:last - start] >= np.uint64(min(int(p * 2 ** 32 + 0.5), MASK)))


def scale_of(p):
    return F32(1 / (1 - p))


def slope(a, b):
    """d pam(a, b) / d a."""
    (_, fa, _), (sb, fb, eb) = _split(a), _split(torch.as_tensor(b, dtype=torch.float64))
    return sb * torch.exp2(eb + (fa + fb >= 1.0))


def dropped(x, p, seed):
    """(float64 value, mask) of dropout on the fp32 tensor x; the product is exact."""
    mask = kept(seed, 0, x.numel(), p).view(x.shape)
    return torch.where(mask, pam(x.double(), scale_of(p)), 0.0), mask


def dropped_grad(g, x, p, seed, approx):
    mask = kept(seed, 0, g.numel(), p).view(g.shape)
    s = scale_of(p)
    return torch.where(mask, pam(g.double(), s) if approx else g.double() * slope(x.double(), s), 0.0)


def embedded(tokens, weight, scale, positions, p, seed):
    """(x, y): the fp32 sum before the dropout and the float64 result; with positions the sum is rounded once."""
    rows = weight.double()[tokens]
    x = rows if scale is None else pam(rows, F32(scale))
    if positions is not None:
        x = x + positions.double()
    x = x.float()
    return x, x.double() if p == 0 else dropped(x, p, seed)[0]


def embedded_grad(g, tokens, weight, scale, positions, padding, p, seed, approx):
    """(d weight, its bound, d positions of one row for each place): float64.

    The terms are exact: PAM products, or products with powers of two.  A sum of n of them in any order is off by at most n - 1 roundings, each of at most
    u = 2^-24 of the sum of their magnitudes, to first order; n u covers the second."""
    x, _ = embedded(tokens, weight, scale, positions, p, seed)
    h = dropped_grad(g, x, p, seed, approx) if p else g.double()
    terms = h if scale is None else pam(h, F32(scale)) if approx else h * slope(weight.double()[tokens], F32(scale))
    live = torch.ones_like(tokens, dtype=torch.bool) if padding is None else tokens != padding
    d, size = torch.zeros(weight.shape, dtype=torch.float64), torch.zeros(weight.shape, dtype=torch.float64)
    d.index_put_((tokens[live],), terms[live], accumulate=True)
    size.index_put_((tokens[live],), terms[live].abs(), accumulate=True)
    count = torch.bincount(tokens[live].flatten(), minlength=weight.shape[0]).double()[:, None]
    return d, count * U * size, h


def _share(fraction, total):
    return int(math.floor(fraction * 2 ** 24)) * total


def sampled(logits, uniform, temperature, top_k, top_p, min_p, banned):
    """(token, score, bound) of one row: fp32 logits [vocabulary], numbers, banned bool [vocabulary] or None.

    The score is x minus a quotient: a sum that is exact but for terms below 2^-62 of the largest power (2^-44 of it together), a logarithm, a quotient and a difference
    with a rounding of 2^-53 each, 2^-40 together for |x| < 2^10, and the rounding to fp32."""
    n = logits.numel()
    masked = logits <= -1e30
    x = torch.where(masked, -1.0, pad(logits.double(), F32(temperature)))
    t = pam(x, LOG2E)
    banned = torch.zeros(n, dtype=torch.bool) if banned is None else banned
    live = ~masked & ~banned
    if bool((t.isnan() & ~masked).any()) or not bool(live.any()) or not 0 < temperature < INF:
        return -1, -INF, 0.0
    whole = torch.floor(t)
    steps = torch.floor((t - whole) * 2 ** 23).long() + 2 ** 23                     # (1 + f') 2^23
    below = (whole[live].max() - whole).clamp(max=200).long()
    weight = torch.where(below <= 21, steps << (21 - below).clamp(0, 63), steps >> (below - 21).clamp(0, 63))
    at = live.nonzero()[:, 0].numpy()
    order = at[np.lexsort((at, -steps[at].numpy(), below[at].numpy()))]
    if top_k > 0:
        order = order[:top_k]
    w = weight.numpy()[order]
    if top_p < 1.0:
        limit = max(-(-_share(F32(top_p), int(w.sum())) >> 24), 1)
        keep = int((np.cumsum(w) - w < limit).sum())
        order, w = order[:keep], w[:keep]
    least = -(-_share(F32(min_p), int(w[0])) >> 24)
    order, w = order[w >= least], w[w >= least]
    place = np.argsort(order)
    upto = np.cumsum(w[place])
    drawn = _share(float(uniform), int(upto[-1])) >> 24
    token = int(order[place][int((upto <= drawn).sum())])
    inside = ~masked
    top = whole[inside].max()
    total = (torch.exp2(whole[inside] - top) * (1 + (t - whole)[inside])).sum()
    _, f, e = _split(total)
    score = float(x[token] - pad(top + e + f, LOG2E))
    return token, score, U * abs(score) + 2.0 ** -40
