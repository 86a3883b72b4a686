"""The rotation, the paged append and the paged decode in 64 bits, straight from their formulas, and how far a kernel may be off."""
import math

import torch

EPS = 2.0 ** -24  # half a step of fp32


def positions_of(new, held=None):
    held = new if held is None else held
    return torch.cat([torch.arange(b - a, b) for a, b in zip(new, held)]) if new else torch.zeros(0, dtype=torch.int64)


def rotate(x, cos, sin, pos, interleaved, back=False):
    """(rotated x, sum of the absolute products of each element), both float64."""
    x, c, s = x.detach().double(), cos.double()[pos][:, None], sin.double()[pos][:, None]
    s = -s if back else s
    R = 2 * cos.shape[1]
    out, mag = x.clone(), x.abs()
    first = torch.arange(0, R, 2, device=x.device) if interleaved else torch.arange(R // 2, device=x.device)
    second = first + 1 if interleaved else first + R // 2
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    mag[..., first], mag[..., second] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, mag


def store_error(ref, dtype):
    """Half a step of the type at each value (for fp16 no less than half its smallest one)."""
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return ref.abs() * (torch.finfo(dtype).eps / 2) + tiny


def rotation_error(ref, mag, dtype):
    """Two products and a sum of fp32, each off by half a step of at most the absolute sum, then the type's rounding of the
    value (once more for a value that the first errors moved across a power of two: counted by the factor)."""
    fp32 = 3 * EPS * mag
    return fp32 + store_error(ref.abs() + fp32, dtype)


def assert_within(got, ref, tol, what):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    both = torch.isnan(ref) & torch.isnan(got) | (ref == got)
    off = ((got - ref).abs() - tol)
    bad = ~(both | (off <= 0))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by {off[bad].max().item() if bad.any() else 0:.3g} over its bound"


def decode(q, k_cache, v_cache, table, lens, scale=None):
    """(o, lse, bound of o, bound of lse) in float64 for q [n, T, H, D] and host lists of lengths.

    Bounds.  A score is a sum of D products: each addend meets at most D + 2 roundings of fp32 (2^-23 each, as matrix
    units may cut instead of rounding), so it is off by e_s = scale (D + 2) 2^-23 sum|q k|, plus the scaling's own.  The exponent c s - m
    (in the log2 domain, |c s - m| <= 2 max|c s|) is rounded once, the exponential off by 2^-22, P as two 16-bit
    pieces by 2^-18 (bf16: 2^-9 of 2^-9; fp16 less, but no less than 2^-25 of the row's largest).  An addend of sum p v goes
    through the roundings of its block, of the blocks after it and of the joins: fewer than n / 32 + 80.  All of that is
    relative to sum p |v|, the denominator's share doubles it, and the type's rounding comes last."""
    n, T, H, D = q.shape
    page, H_kv = k_cache.shape[1], k_cache.shape[2]
    g = H // H_kv
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
    eo, el = torch.zeros_like(o), torch.zeros_like(lse)
    for i, L in enumerate(lens):
        pages = table[i, :-(-L // page)].long()
        k, v = (x[pages].flatten(0, 1)[:L].double() for x in (k_cache, v_cache))
        for t in range(T):
            e = L - T + t + 1
            if e <= 0:
                continue
            qq = q[i, t].double().view(H_kv, g, D)
            kk, vv = k[:e], v[:e]
            s = torch.einsum("hgd,jhd->hgj", qq, kk) * scale
            p = torch.softmax(s, -1)
            o[i, t] = torch.einsum("hgj,jhd->hgd", p, vv).reshape(H, D)
            lse[i, t] = torch.logsumexp(s, -1).view(H)
            mag = torch.einsum("hgd,jhd->hgj", qq.abs(), kk.abs()).amax(-1) * abs(scale)
            rel = mag * (D + 2) * 2.0 ** -23 + 4 * s.abs().amax(-1) * 2.0 ** -23 + 2.0 ** -22
            rel = rel + (e / 32 + 80) * 2.0 ** -23 + (0 if q.dtype == torch.float32 else 2.0 ** -18)
            floor = 2.0 ** -24 * p.amax(-1) if q.dtype == torch.float16 else 0.0
            pv = torch.einsum("hgj,jhd->hgd", p, vv.abs())
            eo[i, t] = (2 * rel[..., None] * pv + (torch.as_tensor(floor) * torch.ones_like(rel))[..., None] * vv.abs().sum(0)[:, None]).reshape(H, D)
            el[i, t] = (2 * rel + 2.0 ** -22 * (1 + lse[i, t].view(H_kv, g).abs())).view(H)
    return o, lse, eo + store_error(o.abs() + eo, q.dtype), el


def paged_cache(lens, H_kv, D, page, dtype, gen, spare=2, extra_cols=1, fill=float("nan"), layout="nhd"):
    """(k_cache, v_cache, table): pages in random order; what no token holds is `fill`."""
    dev = "cuda"
    need = [-(-n // page) for n in lens]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(need + [0]) + extra_cols, dtype=torch.int32, device=dev)
    if layout == "hnd":
        caches = [torch.empty(pool, H_kv, page, D, dtype=dtype, device=dev).transpose(1, 2) for _ in range(2)]
    elif layout == "halves":
        both = torch.empty(pool, 2, page, H_kv, D, dtype=dtype, device=dev)
        caches = [both[:, 0], both[:, 1]]
    else:
        caches = [torch.empty(pool, page, H_kv, D, dtype=dtype, device=dev) for _ in range(2)]
    for c in caches:
        c.fill_(fill)
    at = 0
    for i, n in enumerate(lens):
        ids = order[at:at + need[i]]
        at += need[i]
        table[i, :need[i]] = ids
        for c in caches:
            x = torch.full((need[i] * page, H_kv, D), fill, dtype=dtype, device=dev)
            x[:n] = torch.randn(n, H_kv, D, generator=gen, device=dev).to(dtype)
            c[ids.long()] = x.view(need[i], page, H_kv, D)
    return caches[0], caches[1], table
