"""Plain 64-bit statements of the rotary, paged-cache and drafted-tree operators."""
import math

import torch


def half_step(dtype):
    """The most one rounding to `dtype` is off, relative to the value."""
    return torch.finfo(dtype).eps / 2


def rotate(x, positions, inv_freq, interleaved, scale=1.0, inverse=False):
    """[tokens, heads, dim] in 64 bits, pair by pair."""
    y = x.double().clone()
    r = 2 * inv_freq.numel()
    a = positions.double()[:, None] * inv_freq.double()[None, :]
    if inverse:
        a = -a
    c, s = (a.cos() * scale)[:, None], (a.sin() * scale)[:, None]
    if interleaved:
        x1, x2 = x[..., 0:r:2].double(), x[..., 1:r:2].double()
        y[..., 0:r:2], y[..., 1:r:2] = x1 * c - x2 * s, x2 * c + x1 * s
    else:
        x1, x2 = x[..., :r // 2].double(), x[..., r // 2:r].double()
        y[..., :r // 2], y[..., r // 2:r] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def rotate_bound(x, inv_freq, interleaved, scale, dtype, positions):
    """Elementwise bound on a computed rotation's distance from `rotate`.

    sin and cos: the angle in half turns is rounded to fp32 (2^-25, times pi as an
    angle), the function is good to 2 ulp (2^-23 of a value of at most 1), the step
    of a 64-bit fraction is good to 2^-53 of a turn's fraction per position and
    the 64-bit statement rounds its angle to 2^-53 relative: 2^-51 |position| for
    both.  Two products, a sum and the factor add four roundings of 2^-24 to terms
    that |x1| + |x2| bounds.  Then one rounding to the element type.
    """
    y = x.double().abs()
    r = 2 * inv_freq.numel()
    if interleaved:
        s = y[..., 0:r:2] + y[..., 1:r:2]
        both = torch.stack((s, s), -1).flatten(-2)
    else:
        s = y[..., :r // 2] + y[..., r // 2:r]
        both = torch.cat((s, s), -1)
    per = math.pi * 2.0 ** -25 + 2.0 ** -23 + 4 * 2.0 ** -24
    far = positions.double().abs()[:, None, None] * 2.0 ** -51
    out = torch.zeros_like(y)
    out[..., :r] = both * scale * (per + far)
    ref = torch.zeros_like(y)
    ref[..., :r] = both * scale
    return out + half_step(dtype) * ref + torch.finfo(dtype).tiny


def sees(tokens, mask=None):
    """[tokens, tokens] bool of one request; mask: bool [tokens, columns] or None (causal)."""
    if mask is None:
        return torch.ones(tokens, tokens, dtype=torch.bool).tril()
    m = torch.zeros(tokens, tokens, dtype=torch.bool)
    w = min(tokens, mask.shape[1])
    m[:, :w] = mask[:, :w]
    return m


def ancestors(parents):
    """Bool mask and depths of one tree from its parent list."""
    n = len(parents)
    m = torch.zeros(n, n, dtype=torch.bool)
    depth = []
    for i in range(n):
        j, d = i, -1
        while j >= 0:
            m[i, j] = True
            d += 1
            j = parents[j]
        depth.append(d)
    return m, depth


def gather(pages, table, n, head):
    """The first n rows of one request and head: [n, dim]."""
    page = pages.shape[2]
    return torch.stack([pages[int(table[j // page]), head, j % page] for j in range(n)]) if n else \
        pages.new_zeros(0, pages.shape[3])


def attention(q, k_pages, v_pages, table, ctx, counts, masks=None, scale=None):
    """out, lse and sum_j p_j |v_j| (what a rounding of p can move), all in 64 bits on the CPU.

    Keys that a row does not see do not take part, whatever they hold.
    """
    T, H, D = q.shape
    hk = k_pages.shape[1]
    g = H // hk
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, H, D, dtype=torch.float64)
    mag = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    smax = torch.zeros(T, H, dtype=torch.float64)
    first = 0
    for b, (c, m) in enumerate(zip(ctx, counts)):
        vis = sees(m, None if masks is None else masks[b])
        for h in range(hk):
            k = gather(k_pages, table[b], c + m, h).double()
            v = gather(v_pages, table[b], c + m, h).double()
            for t in range(m):
                idx = torch.cat((torch.arange(c), c + torch.nonzero(vis[t]).flatten()))
                if idx.numel() == 0:
                    continue
                qq = q[first + t, h * g:(h + 1) * g].double()
                s = qq @ k[idx].T * scale
                p = torch.softmax(s, -1)
                out[first + t, h * g:(h + 1) * g] = p @ v[idx]
                mag[first + t, h * g:(h + 1) * g] = p @ v[idx].abs()
                lse[first + t, h * g:(h + 1) * g] = torch.logsumexp(s, -1)
                smax[first + t, h * g:(h + 1) * g] = (qq.abs() @ k[idx].abs().T).amax(-1) * abs(scale)  # a size: a negative scale has one too
        first += m
    return out, lse, mag, smax


def attention_bound(out, mag, smax, dtype, keys, dim):
    """Elementwise bounds (out, lse) on the distance from `attention`.

    Products of two elements are exact in fp32 (or, for fp32 elements, off by
    2^-24); a score sums `dim` of them and is scaled: (dim + 2) 2^-24 of the sum of
    the products' sizes.  A weight exp(s - m) moves by that much relative, twice
    (its own and the maximum's), plus 2^-21 for the exponential; both the weighted
    sum and the normaliser carry it, and each sums `keys` terms in fp32.  A weight
    rounded to the element type for the product with V adds half a step; the
    result one more.
    """
    e = 2 * (dim + 2) * 2.0 ** -24 * smax + 2.0 ** -21 + (keys + 8) * 2.0 ** -24
    p_round = half_step(dtype) if dtype != torch.float32 else 0.0
    o = (2 * e[..., None] + p_round) * mag + half_step(dtype) * (out.abs() + 1e-30)
    return o * (1 + 2.0 ** -6), e + 2.0 ** -22 * 40
