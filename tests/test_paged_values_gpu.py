"""Paged decode where the values are what is hard: fp16 weights far below the largest one, held to a bound without a floor that grows with
the number of keys, and infinite values that a row sees."""
import pytest
import torch

import varlenabsorbflashattn_b200 as vb
from varlenabsorbflashattn_b200 import _lib, paged
from paged_ref import assert_within, decode, paged_cache, store_error

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# (D, H, H_kv, T) of every 16-bit tile: up to 8 rows, to 16, to 32, to 64, and several tiles
TILES = [(64, 4, 2, 1), (128, 8, 1, 1), (64, 16, 1, 1), (128, 12, 1, 1), (128, 4, 1, 7), (32, 8, 1, 8), (128, 16, 1, 4), (128, 20, 1, 5), (256, 8, 1, 1),
         (256, 16, 1, 1), (256, 10, 1, 2), (16, 3, 1, 1)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F32):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _decode_fp16(q, kc, vc, table, lens, scale, floor):
    """(o, lse, bounds) of fp16 inputs.  The fp32 part is the formula's shared one.  P goes into the second product as two fp16 pieces of half a
    step of 2^-11 each, so a weight is off by 2^-22 of itself (counted twice); the second piece has nothing below 2^-24, which is `floor`, in
    all.  A step of a warp (64 keys at most) is packed 2^15 times as large as its weights beside the row's running maximum, and where
    the step's own largest one is below 2^-8 lifted further, to 2^14 or more: half of 2^-24 is 2^-40 of the running maximum in the
    first case, 2^-39 of the step's largest in the second, and so 2^-32 of the step's largest weight in both."""
    ro, rl, e32, el = decode(q.float(), kc, vc, table, lens, scale=scale)
    pv = decode(q.float(), kc, vc.abs(), table, lens, scale=scale)[0]
    off = e32 + 2 * 2.0 ** -22 * pv + floor
    return ro, rl, off + store_error(ro.abs() + off, F16), el


@pytest.mark.parametrize("sms", [1, 148])
@pytest.mark.parametrize("D,H,H_kv,T", TILES)
def test_fp16_weights_far_below_the_largest(monkeypatch, D, H, H_kv, T, sms):
    """A first key far above the others whose own value is zero: what the others weigh is the whole answer.  On one SM a unit lies in one
    piece, so that the same warp has the first key and many of the others."""
    gen, lens = _gen(D + T), [4000, 2100, 1500, 700, 90]
    monkeypatch.setattr(_lib, "sm_count", lambda device: sms)
    monkeypatch.setattr(paged, "_plans", {})
    kc, vc, table = paged_cache(lens, H_kv, D, 16, F16, gen, fill=0.0)
    kc[...] = 0
    vc[...] = (1 + torch.rand(vc.shape, generator=gen, device="cuda")) * 16384
    q = torch.zeros(len(lens), T, H, D, dtype=F16, device="cuda")
    q[..., 0] = 1 + 0.25 * (torch.arange(T * H, device="cuda").view(T, H) % 3)  # the rows of a tile differ
    for i, peak in enumerate((12.0, 17.375, 14.0, 24.5, 17.0)):                # times 1 to 1.5
        kc[table[i, 0].long(), 0, :, 0] = peak
        vc[table[i, 0].long(), 0] = 0
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens), scale=1.0)
    # the steps without the first key have equal weights: 2^-39 of each, in the 2^-22; the step with it has up to 64 keys
    ro, rl, eo, el = _decode_fp16(q, kc, vc, table, lens, 1.0, 64 * 2.0 ** -40 * vc.max().item())
    assert_within(lse, rl, el, "lse")
    assert_within(o, ro, eo, "o")


@pytest.mark.parametrize("D,H,H_kv,T", TILES)
def test_fp16_scores_of_large_spread(D, H, H_kv, T):
    """Scores over some fifty nats, the maximum moving up and blocks far below it, values of either sign and every size."""
    gen, lens = _gen(D + H), [2000, 513, 77]
    kc, vc, table = paged_cache(lens, H_kv, D, 16, F16, gen, fill=0.0)
    vc *= 1000
    q = _randn(gen, len(lens), T, H, D, dtype=F16)
    scale = 8 / D ** 0.5
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens), scale=scale)
    # the steps' largest weights add up to no more than all weights, 1
    ro, rl, eo, el = _decode_fp16(q, kc, vc, table, lens, scale, 64 * 2.0 ** -32 * vc.abs().max().item())
    assert_within(lse, rl, el, "lse")
    assert_within(o, ro, eo, "o")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,H,H_kv,T", TILES)
def test_infinite_values_that_a_row_sees(dtype, D, H, H_kv, T):
    """An infinite value is an infinite result of the rows that see it, whatever its weight is, and two of opposite signs are NaN; the other
    dims, and the rows that do not see it, are as the formula has them."""
    gen, lens, inf = _gen(D), [1, 300, 20, 90, 5000, T], float("inf")
    kc, vc, table = paged_cache(lens, H_kv, D, 16, dtype, gen)
    q = _randn(gen, len(lens), T, H, D, dtype=dtype)

    def put(seq, key, dim, value):
        vc[table[seq, key // 16].long(), key % 16, :, dim] = value

    put(0, 0, 0, inf)                                   # the only weight, 1
    for key, dim, value in ((7, 3, inf), (250, 3, inf), (100, 5, -inf), (31, 6, inf), (40, 6, -inf), (299, 8, inf), (0, 9, -inf)):
        put(1, key, dim, value)
    for dim in range(D):
        put(2, 19, dim, -inf)                           # of several tokens only the last one sees it
    kc[table[3, :6].long()] = 0                         # a weight of 2^-29 beside the first key's
    q[3] = 0
    kc[table[3, 0].long(), 0, :, 0], q[3, ..., 0], vc[table[3, 0].long(), 0] = 20 * D ** 0.5 / 4, 4, 0
    put(3, 50, 1, inf)
    for key in range(4321, 4400):
        put(4, key, D - 1, inf)
    put(5, T - 1, 2, inf)
    ro, rl, eo, el = decode(q, kc, vc, table, lens)
    assert torch.isinf(ro).any() and ro.isnan().any()
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert_within(lse, rl, el, "lse")
    assert_within(o, ro, eo, "o")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,H,H_kv,T", [(64, 4, 2, 1), (128, 4, 1, 4), (256, 8, 1, 1), (32, 16, 1, 4)])
def test_values_that_are_nan_or_of_every_kind(dtype, D, H, H_kv, T):
    """NaN in one place, in a whole head dim, everywhere; infinite values in every key; each beside dims that are finite."""
    gen, lens, inf, nan = _gen(D + 1), [700, 700, 700, 700], float("inf"), float("nan")
    kc, vc, table = paged_cache(lens, H_kv, D, 16, dtype, gen)
    q = _randn(gen, len(lens), T, H, D, dtype=dtype)
    pages = [table[i, :44].long() for i in range(4)]
    vc[pages[0][20], 3, :, 5] = nan
    vc[pages[0][40], 1, :, 5] = inf
    vc[pages[0][40], 2, :, 4] = -inf
    vc[pages[1], :, :, 7] = nan
    vc[pages[1], :, :, 9] = inf
    vc[pages[2], :, :, D // 2:] = -inf
    vc[pages[2][0], 0, :, D - 1] = inf
    vc[pages[3]] = nan
    ro, rl, eo, el = decode(q, kc, vc, table, lens)
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert o[3].isnan().all() and o[0, ..., 5].isnan().all() and (o[0, ..., 4] == -inf).all() and (o[1, ..., 9] == inf).all()
    assert_within(lse, rl, el, "lse")
    assert_within(o, ro, eo, "o")
