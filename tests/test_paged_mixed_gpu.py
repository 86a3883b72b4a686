"""Rotation, paged append and paged decode on the GPU: arguments of other types, kinds and sizes than the usual ones."""
import pytest
import torch
from torch.autograd import forward_ad

import varlenabsorbflashattn_b200 as vb
from varlenabsorbflashattn_b200 import _lib
from paged_ref import assert_within, decode, paged_cache, positions_of, rotate, rotation_error

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def unchecked():
    vb.set_validate_cu_seqlens(False)
    yield
    vb.set_validate_cu_seqlens(True)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=F32):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _status():
    st = _lib.status_word(torch.device("cuda", 0))
    got = st.tolist()
    st.zero_()
    return got[:2]


def test_unchecked_indices_beyond_32_bits(unchecked):
    """2^32 + 3 is not page 3, nor 2^32 + 8 a length of 8: out of range like any other, reported, nothing written."""
    gen, wide = _gen(1), 2**32
    kc, vc, table = paged_cache([8, 8, 8], 2, 64, 4, BF16, gen, fill=0.0)
    q, k, v = (_randn(gen, 3, 2, 64, dtype=BF16) for _ in range(3))
    cos, sin = vb.rotary_table(8, 64, device="cuda")
    lens = torch.tensor([8, 8, 8], device="cuda")
    before = kc.clone(), vc.clone()
    call = lambda lens, table: vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=lens, q=q, cos=cos, sin=sin)  # noqa: E731
    _status()
    assert call(lens, table.long() + wide).isnan().all() and _status() == [4, 911]
    assert call(lens, table.long() - wide).isnan().all() and _status() == [4, 911]
    assert call(lens + wide, table).isnan().all() and _status() == [4, 911]
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    got, _ = vb.packed_rotary(q, None, cos, sin, positions=torch.tensor([1, wide, 2 - wide]))
    assert got[1:].isnan().all() and not got[0].isnan().any() and _status() == [4, 910]

    want = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=lens)
    for lens_, table_ in ((lens + torch.tensor([0, wide, 0], device="cuda"), table), (lens, table.long() + torch.tensor([[0], [wide], [0]], device="cuda"))):
        assert _status() == [0, 0]
        got = vb.paged_decode_attn(q, kc, vc, page_table=table_, cache_seqlens=lens_)
        assert _status() == [4, 912] and torch.equal(got[[0, 2]], want[[0, 2]])


def test_forward_mode_is_refused():
    gen = _gen(2)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, F32, gen, fill=0.0)
    before = kc.clone(), vc.clone()
    q, t = _randn(gen, 2, 2, 64), _randn(gen, 2, 2, 64)
    cos, sin = vb.rotary_table(8, 64, device="cuda")
    where = dict(page_table=table, cache_seqlens=_ints([8, 8]))
    for _ in range(2):  # a layout that has been called before, and one that has not
        with forward_ad.dual_level():
            x = forward_ad.make_dual(q, t)
            for call in (lambda: vb.packed_rotary(x, None, cos, sin, cu_seqlens=_cu([2])), lambda: vb.paged_kv_append(q, x, kc, vc, **where),
                         lambda: vb.paged_decode_attn(x, kc, vc, **where)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
        vb.packed_rotary(q, None, cos, sin, cu_seqlens=_cu([2]))
        vb.paged_kv_append(q, q, kc, vc, **where)
        vb.paged_decode_attn(q, kc, vc, **where)
        before = kc.clone(), vc.clone()
    rotated = lambda x: vb.packed_rotary(x, None, cos, sin, cu_seqlens=_cu([2]))[0]  # noqa: E731
    with pytest.raises(RuntimeError):
        torch.func.jvp(rotated, (q,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(rotated)(q[None])


def test_keys_rotated_beside_queries_with_a_gradient_have_none():
    """With frozen keys the rotated ones go into the cache while queries are trained, and dK is nobody's."""
    gen = _gen(3)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, F32, gen, fill=0.0)
    q, k = _randn(gen, 2, 4, 64).requires_grad_(), _randn(gen, 2, 2, 64)
    cos, sin = vb.rotary_table(8, 64, device="cuda")
    a, b = vb.packed_rotary(q, k, cos, sin, positions=_ints([7, 7]))
    assert a.requires_grad and not b.requires_grad
    vb.paged_kv_append(b, k, kc, vc, page_table=table, cache_seqlens=_ints([8, 8]))
    a, b = vb.packed_rotary(q.detach(), k.requires_grad_(), cos, sin, positions=_ints([7, 7]))
    assert b.requires_grad and not a.requires_grad
    g, = torch.autograd.grad(b, k, torch.ones_like(b), create_graph=True)  # the gradient's own graph
    assert g.shape == k.shape


def test_errors_of_a_server_under_inference_mode(monkeypatch, unchecked):
    """The first call of a program may be one of a serving loop: its status word is read and cleared anywhere."""
    from varlenabsorbflashattn_b200 import paged
    monkeypatch.setattr(_lib, "_status", {})
    monkeypatch.setattr(paged, "_plans", {})
    gen, dev = _gen(4), torch.device("cuda", 0)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, BF16, gen, fill=0.0)
    q = _randn(gen, 2, 2, 64, dtype=BF16)
    with torch.inference_mode():
        vb.paged_decode_attn(q, kc, vc, page_table=table + 99, cache_seqlens=_ints([8, 8]))
    with pytest.raises(RuntimeError, match="outside its array"):
        _lib.check_status(dev)
    _lib.check_status(dev)


@pytest.mark.parametrize("kept", ["k", "v"])
def test_autograd_is_told_of_either_cache(kept):
    """One cache made under inference mode, the other one kept for a gradient."""
    gen = _gen(5)
    caches, table = {}, _ints([[0, 1], [2, 3]])
    with torch.inference_mode():
        caches["v" if kept == "k" else "k"] = _randn(gen, 4, 4, 2, 64)
    caches[kept] = _randn(gen, 4, 4, 2, 64)
    k, w = _randn(gen, 2, 2, 64), torch.ones((), device="cuda", requires_grad=True)
    y = (w * caches[kept]).sum()
    vb.paged_kv_append(k, k, caches["k"], caches["v"], page_table=table, cache_seqlens=_ints([8, 8]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("dtype,H,H_kv,D,R", [(F32, 32, 8, 128, 128), (F32, 80, 8, 128, 64), (BF16, 88, 88, 128, 128), (F16, 60, 30, 256, 2), (F32, 40, 8, 256, 256)])
def test_long_batches_of_wide_tokens(dtype, H, H_kv, D, R):
    """Token rows of more than half a tile of shared memory (one token a tile), up to those that do not fit four times (48 KB)."""
    gen = _gen(H)
    T = (11 << 20) // ((H + H_kv) * D * dtype.itemsize) + 3
    lens = [1, 0, 100, T - 101]
    qkv = _randn(gen, T, H + 2 * H_kv, D, dtype=dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + H_kv], qkv[:, H + H_kv:]
    cos, sin = vb.rotary_table(max(lens), R, device="cuda")
    pos = positions_of(lens).cuda()
    out = vb.packed_rotary(q, k, cos, sin, cu_seqlens=_cu(lens))
    for name, x, y in zip("qk", (q, k), out):
        ref, mag = rotate(x, cos, sin, pos, False)
        assert_within(y, ref, rotation_error(ref, mag, dtype), name)
    kc, vc, table = paged_cache(lens, H_kv, D, 16, dtype, gen, fill=7.0)
    want = kc.clone(), vc.clone()
    at = table[torch.repeat_interleave(torch.arange(4), torch.tensor(lens)).cuda(), pos // 16].long(), pos % 16
    want[0][at], want[1][at] = out[1], v
    got = vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints(lens), cu_seqlens=_cu(lens), q=q, cos=cos, sin=sin)
    assert torch.equal(got, out[0]) and torch.equal(kc, want[0]) and torch.equal(vc, want[1])


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 16), (F32, 32)])
@pytest.mark.parametrize("T", [1, 4000])
def test_append_to_caches_at_any_address(dtype, D, T):
    """Caches with an odd offset and an odd pitch of pages, slots and heads: only the elements of the new tokens change."""
    gen, H_kv, page = _gen(T), 8, 24
    pages = -(-T // page) + 2
    whole = [torch.full((pages, page + 1, H_kv + 1, D + 3), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    kc, vc = (x[:, 1:, 1:, 3:] for x in whole)
    assert kc.data_ptr() % 16 and kc.stride(2) % 2
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)[None]
    k, v = (_randn(gen, T, H_kv, D, dtype=dtype) for _ in range(2))
    pos = torch.arange(T, device="cuda")
    want = [x.clone() for x in whole]
    for w, x in zip(want, (k, v)):
        w[:, 1:, 1:, 3:][table[0, pos // page].long(), pos % page] = x
    vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints([T]), cu_seqlens=_cu([T]))
    assert all(torch.equal(a, b) for a, b in zip(whole, want))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_lse_of_equal_weights(dtype):
    """scale 0: o is the mean of the values, lse the logarithm of their number."""
    gen, lens, H, H_kv, D = _gen(6), [40, 3, 200, 0, 5000], 6, 3, 64
    kc, vc, table = paged_cache(lens, H_kv, D, 8, dtype, gen)
    q = _randn(gen, len(lens), 2, H, D, dtype=dtype)
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens), scale=0.0)
    ro, rl, eo, el = decode(q, kc, vc, table, lens, scale=0.0)
    assert_within(o, ro, eo, "o")
    assert_within(lse, rl, el, "lse")
    assert (lse[3] == -float("inf")).all() and abs(lse[4, 1, 0].item() - torch.tensor(5000.0).log().item()) < 1e-5
