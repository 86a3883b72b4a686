"""The operators around a paged key/value cache, as measurable cases.

Three operators a program needs beside packed attention when its sequences have positions and are served: the
position rotation of packed queries and keys with its gradient ("rotary"), the append of new keys and values to
a paged cache with that rotation on the way ("append"), and the attention of new tokens over the cache
("decode").  `own` false runs their plain forms in elementary torch operations, true the package's calls.

A case is a dict of plain values.  Lengths are a function of the case alone (its "lens" number seeds them); the seed
given to `prepare` makes the values, N(0, 1) as everywhere in this package's tests and benchmark, and the
order of the pages in the cache.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_BASE = 10000.0

# what a drawn case of an operator stays under: about what the dearest listed one moves (the whole caches for an append, as they are compared)
_MOST_BYTES = {"rotary": 5.0e9, "append": 1.5e9, "decode": 9.0e9}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _rotary(n, lo, hi, H, H_kv, D, R, dtype, grad, lens, interleaved=False, fused=False):
    """Rotation of the queries and keys of n packed sequences, lengths log-uniform in [lo, hi]."""
    return dict(op="rotary", n=n, lo=lo, hi=hi, H=H, H_kv=H_kv, D=D, R=R, dtype=dtype, grad=grad, lens=lens,
                interleaved=interleaved, fused=fused)


def _append(n, new_lo, new_hi, lo, hi, H, H_kv, D, R, page, dtype, lens, interleaved=False):
    """new_lo to new_hi new tokens for each of n sequences that hold lo to hi tokens already (hi = 0: prompts of new sequences).
    R = 0: keys that are rotated already; q, k and v are parts of one projection's output."""
    return dict(op="append", n=n, new_lo=new_lo, new_hi=new_hi, lo=lo, hi=hi, H=H, H_kv=H_kv, D=D, R=R, page=page, dtype=dtype, lens=lens,
                interleaved=interleaved)


def _decode(n, T, lo, hi, H, H_kv, D, page, dtype, lens):
    """T new tokens of each of n sequences over their caches of lo to hi tokens, the new ones among them."""
    return dict(op="decode", n=n, T=T, lo=lo, hi=hi, H=H, H_kv=H_kv, D=D, page=page, dtype=dtype, lens=lens)


def listed():
    cases = {
        # four short packed sequences in the default dtype of torch: the smallest training call, where latency counts
        "rotary_small_fp32": _rotary(4, 17, 255, 8, 8, 64, 64, "fp32", True, 0),
        # prefill of a serving batch, q and k as parts of one projection's output, half of each head rotated, pairs side by side
        "rotary_prefill_fp16": _rotary(16, 128, 8192, 32, 8, 128, 64, "fp16", False, 3, interleaved=True, fused=True),
        # a training step over one GPU's share of the 1 M-token batch, forward and gradients
        "rotary_train_long": _rotary(65, 128, 8192, 32, 8, 128, 128, "bf16", True, 0),
        # one step of a small serving batch: a token for each of 8 requests
        "append_step_small": _append(8, 1, 1, 512, 4096, 8, 8, 128, 128, 16, "bf16", 1),
        # one step of a large serving batch, grouped-query heads
        "append_step": _append(256, 1, 1, 16, 8192, 32, 8, 128, 128, 64, "bf16", 2),
        # the prompts of new requests, from one token to thousands, into pages of 16
        "append_prompts_fp16": _append(24, 1, 8192, 0, 0, 32, 8, 128, 128, 16, "fp16", 3),
        # one step of a small serving batch: 8 requests over caches of up to 4096 keys
        "decode_small": _decode(8, 1, 512, 4096, 8, 8, 128, 16, "bf16", 1),
        # a mid-size serving batch of unequal caches, grouped-query heads
        "decode_gqa": _decode(64, 1, 1024, 16384, 32, 8, 128, 64, "bf16", 2),
        # long caches at full key heads, where the cache's bytes are all that counts
        "decode_long": _decode(128, 1, 8192, 32768, 8, 8, 128, 16, "bf16", 0),
        # a single request with a very long cache: the split over its length has to fill the card
        "decode_one_fp16": _decode(1, 1, 102400, 102400, 8, 2, 64, 32, "fp16", 4),
        # four proposed tokens for each request are looked over at once
        "decode_four": _decode(32, 4, 7, 8192, 32, 8, 128, 16, "bf16", 5),
        # fp32 caches in pages of an odd size
        "decode_fp32": _decode(16, 1, 1, 4096, 16, 4, 64, 17, "fp32", 6),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the ranges above, cut down to what the dearest listed case of its operator costs."""
    lens = rng.randrange(1 << 20)
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    D = rng.choice((16, 32, 64, 64, 128, 128, 128, 256))
    H_kv = rng.choice((1, 2, 4, 5, 8, 8))
    H = H_kv * rng.choice((1, 1, 2, 3, 4, 4, 7, 8))
    page = rng.choice((1, 5, 8, 16, 16, 17, 32, 64, 64, 100, 128, 256))
    R = rng.choice((D, D, D, D // 2, 2 * rng.randint(1, D // 2)))
    interleaved = rng.random() < 0.3
    which = rng.randrange(8)
    if which < 2:
        hi = _logint(rng, 4, 16384)
        c = _rotary(_logint(rng, 1, 160), _logint(rng, 1, hi), hi, H, H_kv, D, R, dtype, rng.random() < 0.6, lens, interleaved, rng.random() < 0.4)
    elif which < 4:
        if rng.random() < 0.5:  # a step
            hi = _logint(rng, 16, 32768)
            c = _append(_logint(rng, 1, 512), 1, rng.choice((1, 1, 1, 4)), _logint(rng, 1, hi), hi, H, H_kv, D, R, page, dtype, lens, interleaved)
        else:  # prompts
            new = _logint(rng, 1, 8192)
            c = _append(_logint(rng, 1, 48), _logint(rng, 1, new), new, 0, 0, H, H_kv, D, rng.choice((R, 0)), page, dtype, lens, interleaved)
    else:
        hi = _logint(rng, 16, 32768)
        n = _logint(rng, 1, 256)
        if rng.random() < 0.2:  # few sequences, long ones
            n, hi = rng.randint(1, 4), _logint(rng, 32768, 131072)
        c = _decode(n, rng.choice((1, 1, 1, 1, 2, 4, 7)), _logint(rng, 1, hi), hi, H, H_kv, D, page, dtype, lens)
    while c["n"] > 1 and _dear(c) > _MOST_BYTES[c["op"]]:
        c["n"] = max(1, c["n"] * 3 // 4)
    while _dear(c) > _MOST_BYTES[c["op"]]:
        c["hi"] = max(1, c["hi"] * 3 // 4)
        c["lo"] = min(c["lo"], c["hi"])
    return c


def _dear(c):
    """Bytes of a case, or of its caches (for a decode half of them padded to the longest, as the plain form holds them)."""
    b, row = work(c)["bytes"], 2 * c["H_kv"] * c["D"] * _BYTES[c["dtype"]]
    if c["op"] == "decode":
        return max(b, c["n"] * c["hi"] * row // 2)
    return b if c["op"] == "rotary" else max(b, sum(_lengths(c)[1]) * row)


# ------------------------------------------------------------------------------------------------
# lengths and work
# ------------------------------------------------------------------------------------------------
def _lengths(c):
    """(new tokens, tokens in all) of the case's sequences."""
    r = random.Random(c["lens"])
    if c["op"] == "rotary":
        new = [_logint(r, c["lo"], c["hi"]) for _ in range(c["n"])]
        return new, new
    if c["op"] == "append":
        new = [_logint(r, c["new_lo"], c["new_hi"]) for _ in range(c["n"])]
        return new, [t + (_logint(r, c["lo"], c["hi"]) if c["hi"] else 0) for t in new]
    held = [_logint(r, c["lo"], c["hi"]) for _ in range(c["n"])]
    return [c["T"]] * c["n"], held


def work(case):
    new, held = _lengths(case)
    T, es, H, H_kv, D = sum(new), _BYTES[case["dtype"]], case["H"], case["H_kv"], case["D"]
    if case["op"] == "rotary":
        passes = 2 if case["grad"] else 1
        n = passes * (2 * T * (H + H_kv) * D * es + max(new) * case["R"] * 4) + 4 * (case["n"] + 1)
        return {"bytes": n, "flops": passes * 3 * T * (H + H_kv) * case["R"]}
    if case["op"] == "append":
        places = len(set().union(*(range(b - a, b) for a, b in zip(new, held))))
        heads = H * (case["R"] > 0) + 2 * H_kv
        n = 2 * T * heads * D * es + places * case["R"] * 4 + 4 * (2 * case["n"] + 1)
        n += 4 * sum(-(-b // case["page"]) - (b - a) // case["page"] for a, b in zip(new, held))
        return {"bytes": n, "flops": 3 * T * (H + H_kv) * case["R"]}
    keys = sum(held)
    pages = sum(-(-b // case["page"]) for b in held)
    return {"bytes": 2 * keys * H_kv * D * es + 2 * T * H * D * es + 4 * (pages + case["n"]), "flops": 4 * case["T"] * H * D * keys}


# ------------------------------------------------------------------------------------------------
# inputs and the pass
# ------------------------------------------------------------------------------------------------
def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _table(rows, R):
    """(cos, sin) of the angles pos * base^(-2 i / R), fp32 [rows, R / 2], the angles in 64 bits."""
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * _BASE ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    return angle.cos().float(), angle.sin().float()


def _cache(case, held, gen, randn):
    """(k_cache, v_cache, page_table): pages in no order, a few that nobody holds among them."""
    page = case["page"]
    need = [-(-b // page) for b in held]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    starts = torch.tensor([0] + need[:-1], dtype=torch.int64).cumsum(0).cuda()
    col = torch.arange(max(need), device="cuda")
    at = starts[:, None] + col[None, :]
    table = torch.where(col[None, :] < torch.tensor(need, device="cuda")[:, None], order[at.clamp_max(pool - 1)], 0)
    shape = (pool, page, case["H_kv"], case["D"])
    return randn(*shape), randn(*shape), table.to(torch.int32).contiguous()


def prepare(case, seed):
    new, held = _lengths(case)
    T, H, H_kv, D = sum(new), case["H"], case["H_kv"], case["D"]
    dtype = _DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    s = {"case": case}
    if case["op"] == "rotary":
        s["cu"] = _cu(new)
        s["cos"], s["sin"] = _table(max(new), case["R"])
        if case["fused"]:
            qkv = randn(T, H + 2 * H_kv, D)
            s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + H_kv]
        else:
            s["q"], s["k"] = randn(T, H, D), randn(T, H_kv, D)
        if case["grad"]:
            s["q"], s["k"] = s["q"].requires_grad_(True), s["k"].requires_grad_(True)
            s["dq"], s["dk"] = randn(T, H, D), randn(T, H_kv, D)
        return s
    s["held"] = torch.tensor(held, dtype=torch.int32).cuda()
    s["k_cache"], s["v_cache"], s["table"] = _cache(case, held, gen, randn)
    if case["op"] == "append":
        qkv = randn(T, H + 2 * H_kv, D)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + H_kv], qkv[:, H + H_kv:]
        s["cu"] = None if max(new) == 1 else _cu(new)  # None: one new token for each sequence
        if case["R"]:
            s["cos"], s["sin"] = _table(max(held), case["R"])
        return s
    s["q"] = randn(case["n"], H, D) if case["T"] == 1 else randn(case["n"], case["T"], H, D)
    return s


def run(s):
    case = s["case"]
    if own:
        import varlenabsorbflashattn_b200 as vb
        vb.set_validate_cu_seqlens(False)  # a loop that builds its lengths and page tables itself
        if case["op"] == "rotary":
            if not case["grad"]:
                return vb.packed_rotary(s["q"], s["k"], s["cos"], s["sin"], cu_seqlens=s["cu"], interleaved=case["interleaved"])
            q, k = vb.packed_rotary(s["q"], s["k"], s["cos"], s["sin"], cu_seqlens=s["cu"], interleaved=case["interleaved"])
            return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))]
        if case["op"] == "append":
            if not case["R"]:
                vb.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], page_table=s["table"], cache_seqlens=s["held"], cu_seqlens=s["cu"])
                return [s["k_cache"], s["v_cache"]]
            q = vb.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], page_table=s["table"], cache_seqlens=s["held"], cu_seqlens=s["cu"],
                                   q=s["q"], cos=s["cos"], sin=s["sin"], interleaved=case["interleaved"])
            return [s["k_cache"], s["v_cache"], q]
        return vb.paged_decode_attn_with_lse(s["q"], s["k_cache"], s["v_cache"], page_table=s["table"], cache_seqlens=s["held"])
    with torch.no_grad():
        if case["op"] == "rotary":
            return _plain_rotary(s)
        if case["op"] == "append":
            return _plain_append(s)
        return _plain_decode(s)


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _rotated(x, c, s, interleaved):
    """x [T, heads, D] with its first dims rotated by the angles whose cosines and sines are c, s [T, R / 2]."""
    R = 2 * c.shape[1]
    f = x.float()
    c, s = c[:, None], s[:, None]
    out = f.clone()
    a, b = (f[..., 0:R:2], f[..., 1:R:2]) if interleaved else (f[..., :R // 2], f[..., R // 2:R])
    u, w = a * c - b * s, b * c + a * s
    if interleaved:
        out[..., 0:R:2], out[..., 1:R:2] = u, w
    else:
        out[..., :R // 2], out[..., R // 2:R] = u, w
    return out.to(x.dtype)


def _segment_of(cu, T):
    return torch.searchsorted(cu, torch.arange(T, device=cu.device, dtype=cu.dtype), right=True) - 1


def _plain_rotary(s):
    case, cu, T = s["case"], s["cu"], s["q"].shape[0]
    pos = torch.arange(T, device="cuda") - cu[_segment_of(cu, T)]
    c, n = s["cos"][pos], s["sin"][pos]
    out = [_rotated(s["q"], c, n, case["interleaved"]), _rotated(s["k"], c, n, case["interleaved"])]
    if case["grad"]:  # the gradient of a rotation is the rotation back
        out += [_rotated(s["dq"], c, -n, case["interleaved"]), _rotated(s["dk"], c, -n, case["interleaved"])]
    return out if case["grad"] else tuple(out)


def _plain_append(s):
    case, T = s["case"], s["k"].shape[0]
    if s["cu"] is None:
        seq = torch.arange(T, device="cuda")
        pos = s["held"].long() - 1
    else:
        seq = _segment_of(s["cu"], T)
        pos = (torch.arange(T, device="cuda") - s["cu"][seq + 1] + s["held"][seq]).long()
    k, out = s["k"], [s["k_cache"], s["v_cache"]]
    if case["R"]:
        c, n = s["cos"][pos], s["sin"][pos]
        k = _rotated(k, c, n, case["interleaved"])
        out.append(_rotated(s["q"], c, n, case["interleaved"]))
    page, slot = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    s["k_cache"][page, slot] = k
    s["v_cache"][page, slot] = s["v"]
    return out


def _plain_decode(s):
    case = s["case"]
    n, T, H, H_kv, D, page = case["n"], case["T"], case["H"], case["H_kv"], case["D"], case["page"]
    L = s["table"].shape[1] * page
    q = s["q"].float().view(n, T, H_kv, H // H_kv, D).permute(0, 2, 1, 3, 4).reshape(n, H_kv, T * (H // H_kv), D)
    k = s["k_cache"][s["table"].long()].view(n, L, H_kv, D).permute(0, 2, 3, 1).float()
    x = torch.matmul(q, k).mul_(D ** -0.5).view(n, H_kv, T, H // H_kv, L)
    del k
    last = s["held"][:, None] - T + torch.arange(T, device="cuda")[None, :]
    seen = torch.arange(L, device="cuda")[None, None, :] <= last[:, :, None]
    x.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True).clamp_min(-1e30)
    p = x.sub_(m).exp_()
    z = p.sum(-1, keepdim=True)
    p = p.div_(z.clamp_min(1e-30))
    v = s["v_cache"][s["table"].long()].view(n, L, H_kv, D).permute(0, 2, 1, 3).float()
    o = torch.matmul(p.view(n, H_kv, T * (H // H_kv), L), v).view(n, H_kv, T, H // H_kv, D).permute(0, 2, 1, 3, 4)
    o = o.reshape(s["q"].shape).to(s["q"].dtype)
    lse = torch.where(z > 0, m + z.log(), -math.inf).squeeze(-1).permute(0, 2, 1, 3).reshape(s["q"].shape[:-1])
    return o, lse


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _turn(x, c, s, interleaved):
    """The rotation as a product of complex numbers."""
    R = 2 * c.shape[1]
    w = torch.complex(c.double(), s.double())[:, None]
    d = x.detach().double()
    head = d[..., :R].unflatten(-1, (-1, 2)) if interleaved else d[..., :R].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * w)
    z = z if interleaved else z.transpose(-1, -2)
    return torch.cat([z.flatten(-2), d[..., R:]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    new, held = _lengths(case)
    il = case.get("interleaved", False)
    if case["op"] == "decode":
        T, H, H_kv, D = case["T"], case["H"], case["H_kv"], case["D"]
        g = H // H_kv
        q = s["q"].view(case["n"], T, H, D)
        o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device="cuda")
        for i, L in enumerate(held):
            pages = s["table"][i, :-(-L // case["page"])].long()
            k, v = (x[pages].flatten(0, 1)[:L].double() for x in (s["k_cache"], s["v_cache"]))
            a = torch.einsum("thgd,jhd->thgj", q[i].double().view(T, H_kv, g, D), k) / math.sqrt(D)
            for t in range(T):  # token t does not see the ones after it
                a[t, ..., max(0, L - T + t + 1):] = -math.inf
            lse[i] = torch.logsumexp(a, -1).view(T, H)
            o[i] = torch.einsum("thgj,jhd->thgd", torch.softmax(a, -1).nan_to_num(0.0), v).reshape(T, H, D)
        return o.view(s["q"].shape), lse.view(s["q"].shape[:-1])
    pos = torch.cat([torch.arange(b - a, b) for a, b in zip(new, held)]).cuda()
    if case["op"] == "rotary":
        c, n = s["cos"][pos], s["sin"][pos]
        out = [_turn(s["q"], c, n, il), _turn(s["k"], c, n, il)]
        return out + [_turn(s["dq"], c, -n, il), _turn(s["dk"], c, -n, il)] if case["grad"] else tuple(out)
    seq = torch.repeat_interleave(torch.arange(case["n"]), torch.tensor(new)).cuda()
    at = s["table"][seq, pos // case["page"]].long() * case["page"] + pos % case["page"]
    k_new = _turn(s["k"], s["cos"][pos], s["sin"][pos], il) if case["R"] else s["k"].double()
    caches = [x.double().flatten(0, 1) for x in (s["k_cache"], s["v_cache"])]
    caches[0].index_copy_(0, at, k_new)
    caches[1].index_copy_(0, at, s["v"].double())
    out = [x.view(s["k_cache"].shape) for x in caches]
    return out + [_turn(s["q"], s["cos"][pos], s["sin"][pos], il)] if case["R"] else out
