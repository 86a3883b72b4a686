"""Rotation, paged append and paged decode without a GPU: arguments of other types and kinds than the usual ones."""
import os
import re

import pytest
import torch
from torch.autograd import forward_ad

import varlenabsorbflashattn_b200 as vb
from varlenabsorbflashattn_b200 import _lib, build, paged


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
def test_integers_beyond_32_bits_stay_out_of_range(dtype):
    top = 2**31 - 1
    values = [0, 7, top, top + 1, 2**32 - 1] + ([2**32 + 3, 2**62] if dtype != torch.uint32 else []) + ([-1, -2**31 - 1, -2**32 - 5] if dtype == torch.int64 else [])
    got = paged._ints(torch.tensor(values, dtype=dtype), torch.device("cpu"), "page_table")
    assert got.dtype == torch.int32 and got.tolist() == [max(-2**31, min(top, v)) for v in values]


def test_integers_of_32_bits_and_less_stay_as_they_are():
    x = torch.tensor([5, -3], dtype=torch.int32)
    assert paged._ints(x, x.device, "x") is x
    for dtype in (torch.int8, torch.int16):
        assert paged._ints(x.to(dtype), x.device, "x").tolist() == [5, -3]


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused_by_every_call(grad_mode):
    """No result without its tangent: neither requires_grad nor grad mode has a part in it."""
    x, c = torch.zeros(3, 2, 16), torch.zeros(4, 8)
    cache, table, lens = torch.zeros(2, 4, 2, 16), torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    where = dict(page_table=table, cache_seqlens=lens)
    cu = torch.tensor([0, 3])
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: vb.packed_rotary(dual(x), None, c, c, cu_seqlens=cu), lambda: vb.packed_rotary(x, dual(x), c, c, cu_seqlens=cu),
                     lambda: vb.packed_rotary(x, x, c, dual(c), cu_seqlens=cu), lambda: vb.paged_kv_append(dual(x), x, cache, cache, **where),
                     lambda: vb.paged_kv_append(x, dual(x), cache, cache, **where),
                     lambda: vb.paged_kv_append(x, x, cache, cache, q=dual(x), cos=c, sin=c, **where),
                     lambda: vb.paged_decode_attn(dual(x), cache, cache, **where), lambda: vb.paged_decode_attn(x, cache, dual(cache), **where),
                     lambda: vb.paged_decode_attn_with_lse(x, dual(cache), cache, **where)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(AssertionError, match="CUDA"):  # a call without a tangent goes on to the other checks
            vb.packed_rotary(x, None, c, c, cu_seqlens=cu)


@pytest.mark.parametrize("wants_q,wants_k", [(True, False), (False, True), (True, True)])
def test_only_what_has_a_gradient_comes_back_with_one(monkeypatch, wants_q, wants_k):
    monkeypatch.setattr(paged, "_rotate", lambda plan, q, k, *rest: tuple(None if x is None else x.clone() for x in (q, k)))
    monkeypatch.setattr(paged, "_rotary_plan", lambda *a: None)
    monkeypatch.setattr(paged, "_plans", {})
    q, k = (torch.randn(3, 2, 16).requires_grad_(wants) for wants in (wants_q, wants_k))
    c, cu = torch.zeros(4, 8), torch.tensor([0, 3], dtype=torch.int32)
    a, b = paged._PackedRotary.apply(q, k, c, c, None, cu, None, False, False)
    assert (a.requires_grad, b.requires_grad) == (wants_q, wants_k)
    (a.sum() + b.sum()).backward()
    assert (q.grad is not None, k.grad is not None) == (wants_q, wants_k)
    x = torch.randn(3, 2, 16, requires_grad=True)  # and without the other input at all
    a, b = paged._PackedRotary.apply(x, None, c, c, None, cu, None, False, False)
    a.sum().backward()
    assert b is None and torch.equal(x.grad, torch.ones_like(x))


def test_threads_that_make_the_status_word_at_once_get_the_same_one(monkeypatch):
    monkeypatch.setattr(_lib, "_status", {})
    dev, zeros, others = torch.device("cpu", 0), torch.zeros, []

    def slow_zeros(*a, **kw):  # another thread comes in between
        monkeypatch.setattr(torch, "zeros", zeros)
        others.append(_lib.status_word(dev))
        return zeros(*a, **kw)

    monkeypatch.setattr(torch, "zeros", slow_zeros)
    mine = _lib.status_word(dev)
    assert others and mine is others[0] and _lib.status_word(dev) is mine


def test_warps_whose_lanes_meet_again_give_up_together():
    """A wait that runs out is each lane's own verdict.  Where lanes shuffle, vote or wait for one another after it, it has to be one for all, or
    those that stay wait without a limit for those that left.  (Read from the source: no wait is made to run out.)"""
    with open(os.path.join(build.CSRC, "paged_rotary_rows.cu")) as f:
        source = re.sub(r"//[^\n]*", "", f.read())
    kernel = source[source.index("rows_kernel"):source.index("launch_one")]
    roles = re.split(r"\n  (?:if|\} else if|\} else) ?(?:\(warp [^\n]*\))? ?\{\n", kernel)[1:]
    assert len(roles) >= 3, "load, store and rotation warps"
    meets = [r for r in roles if re.search(r"_sync\(|__syncwarp", r.split("\n  }\n")[0])]
    assert len(meets) >= 2
    for role in meets:
        role = role.split("\n  }\n")[0]
        assert "mbar_wait_warp(" in role and not re.search(r"mbar_wait\(", role), role


def test_status_word_made_under_inference_mode_can_be_cleared(monkeypatch):
    monkeypatch.setattr(_lib, "_status", {})
    with torch.inference_mode():
        word = _lib.status_word(torch.device("cpu", 0))
    word.zero_()
    assert not word.is_inference() and _lib.status_word(torch.device("cpu", 0)) is word


FAKE = 1 << 20  # an address that no check follows


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


_ROTARY = dict(q=FAKE, q_out=FAKE, k=FAKE, k_out=FAKE, cos=FAKE, sin=FAKE, cu_seqlens=FAKE, positions=FAKE, n_seg=1, total=4, num_heads=2,
               num_kv_heads=1, head_dim=64, rotary_dim=64, table_rows=8, dtype=1, status=FAKE)
_APPEND = dict(q=FAKE, q_out=FAKE, k=FAKE, v=FAKE, k_cache=FAKE, v_cache=FAKE, cos=FAKE, sin=FAKE, rotary_dim=64, table_rows=8, cu_seqlens=FAKE,
               cache_seqlens=FAKE, page_table=FAKE, n_seq=2, total=2, num_heads=2, num_kv_heads=2, head_dim=64, num_pages=4, page_size=16,
               max_pages=2, dtype=1, status=FAKE)
_DECODE = dict(q=FAKE, k_cache=FAKE, v_cache=FAKE, o=FAKE, lse=FAKE, cache_seqlens=FAKE, page_table=FAKE, n_seq=2, q_len=1, num_heads=8, num_kv_heads=2,
               head_dim=64, num_pages=4, page_size=16, max_pages=8, dtype=1, scale=1.0, sm_count=148, workspace=FAKE, workspace_bytes=1 << 30, status=FAKE)


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_addresses_inside_an_element_are_refused(lib, dtype):
    """What a kernel would read or write across an element's border ends a process on the GPU: refused on the host."""
    half = 2 if dtype == 0 else 1
    for entry, struct, good, tensors, words in (
            (lib.vafa_rotary, _lib.RotaryArgs, _ROTARY, "q k q_out k_out", "positions cu_seqlens status"),
            (lib.vafa_paged_append, _lib.PagedAppendArgs, _APPEND, "q k v q_out k_cache v_cache", "cu_seqlens cache_seqlens page_table status"),
            (lib.vafa_paged_decode, _lib.PagedAttnArgs, _DECODE, "", "lse cache_seqlens page_table status")):
        for name, off in [(n, half) for n in tensors.split()] + [(n, 2) for n in words.split()]:
            assert entry(struct(**{**good, "dtype": dtype, name: FAKE + off}), None) == -1, name
            assert "aligned" in _lib.last_error(), (name, _lib.last_error())


def test_more_heads_or_sequences_than_are_counted_are_refused(lib):
    many = 1 << 30
    assert lib.vafa_rotary(_lib.RotaryArgs(**{**_ROTARY, "num_heads": many, "num_kv_heads": many}), None) == -2 and "heads" in _lib.last_error()
    assert lib.vafa_paged_append(_lib.PagedAppendArgs(**{**_APPEND, "num_kv_heads": many}), None) == -2 and "heads" in _lib.last_error()
    for n in (many + 1, 2**31 - 1):
        big = _lib.PagedAttnArgs(**{**_DECODE, "n_seq": n})
        assert lib.vafa_paged_decode_workspace_bytes(big) == 0
        assert lib.vafa_paged_decode(big, None) == -2 and "n_seq" in _lib.last_error()
