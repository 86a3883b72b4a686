"""packed_rotary, paged_kv_append, paged_decode_attn on the GPU against their formulas in 64 bits, at the sizes, masks, layouts
and lengths where they can go wrong, and run together as a serving program runs them."""
import math

import pytest
import torch

import varlenabsorbflashattn_b200 as vb
from varlenabsorbflashattn_b200 import _lib, paged
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


# ---- rotation ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,H_kv,D,R", [(8, 8, 64, 64), (4, 1, 128, 128), (6, 2, 128, 64), (5, 5, 16, 16), (3, 1, 32, 26), (7, 1, 256, 256),
                                        (2, 2, 64, 2), (40, 8, 128, 92), (1, 1, 16, 4)])
def test_rotary(dtype, H, H_kv, D, R, interleaved):
    gen = _gen(D + R)
    lens = [1, 0, 37, 2, 130]
    q, k = _randn(gen, sum(lens), H, D, dtype=dtype), _randn(gen, sum(lens), H_kv, D, dtype=dtype)
    cos, sin = vb.rotary_table(130, R, device="cuda")
    got = vb.packed_rotary(q, k, cos, sin, cu_seqlens=_cu(lens), interleaved=interleaved)
    pos = positions_of(lens).cuda()
    for name, x, y in zip("qk", (q, k), got):
        ref, mag = rotate(x, cos, sin, pos, interleaved)
        assert y.dtype == dtype and y.is_contiguous()
        assert_within(y, ref, rotation_error(ref, mag, dtype), name)
    again = vb.packed_rotary(q, k, cos, sin, positions=pos, interleaved=interleaved)
    lengths = vb.packed_rotary(q.unsqueeze(0), None, cos, sin, seqinfo=torch.tensor(lens), interleaved=interleaved)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
    assert lengths[1] is None and torch.equal(lengths[0], got[0].unsqueeze(0))


@pytest.mark.parametrize("dtype,D,R", [(BF16, 128, 128), (F16, 64, 32), (F32, 64, 64), (BF16, 32, 6)])
def test_rotary_of_views(dtype, D, R):
    """Parts of one projection's output, an odd row pitch, an odd offset, a transposed view, a table that begins anywhere."""
    gen, T, H, H_kv = _gen(1), 61, 6, 3
    cos, sin = (x[1:] for x in vb.rotary_table(T + 1, R, device="cuda"))
    cos, sin = (torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape) for x in (cos, sin))
    qkv = _randn(gen, T, H + 2 * H_kv, D, dtype=dtype)
    odd = _randn(gen, T, H * D + 3, dtype=dtype)
    flat = _randn(gen, T * H * D + 1, dtype=dtype)
    for q in (qkv[:, :H], odd[:, :H * D].unflatten(1, (H, D)), flat[1:].view(T, H, D), _randn(gen, H, T, D, dtype=dtype).transpose(0, 1),
              _randn(gen, T, H, 2 * D, dtype=dtype)[..., ::2]):
        k = qkv[:, H:H + H_kv]
        a, b = vb.packed_rotary(q, k, cos, sin, cu_seqlens=_cu([T]))
        for x, y in ((q, a), (k, b)):
            ref, mag = rotate(x, cos, sin, torch.arange(T, device="cuda"), False)
            assert_within(y, ref, rotation_error(ref, mag, dtype), "view")


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    gen, lens = _gen(2), [5, 0, 1, 30]
    T, R = sum(lens), 12
    q, k = _randn(gen, T, 3, 16).requires_grad_(), _randn(gen, T, 1, 16).requires_grad_()
    dq, dk = _randn(gen, T, 3, 16), _randn(gen, T, 1, 16)
    cos, sin = vb.rotary_table(30, R, device="cuda")
    rot = lambda a, b: vb.packed_rotary(a, b, cos, sin, cu_seqlens=_cu(lens), interleaved=interleaved)  # noqa: E731
    out = rot(q, k)
    gq, gk = torch.autograd.grad(out, (q, k), (dq, dk), create_graph=True)
    pos = positions_of(lens).cuda()
    for d, g in ((dq, gq), (dk, gk)):
        ref, mag = rotate(d, cos, sin, pos, interleaved, back=True)
        assert_within(g.detach(), ref, rotation_error(ref, mag, F32), "gradient")
    # against differences: the map is linear, so a step of any size gives the slope; the difference of two outputs of
    # size |y| is off by a few half steps of fp32 at |y| for each of its elements
    with torch.no_grad():
        step = _randn(gen, T, 3, 16)
        slope = ((rot(q + step, k)[0].double() - rot(q - step, k)[0].double()) / 2 * dq.double()).sum().item()
    want = (gq.detach().double() * step.double()).sum().item()
    size = ((q.detach().abs() + step.abs()).double() * dq.double().abs()).sum().item()
    assert abs(slope - want) <= 12 * 2.0 ** -24 * size * 2
    # and the gradient's own gradient is the rotation again
    u = _randn(gen, T, 3, 16)
    dq2 = dq.clone().requires_grad_()
    g1, = torch.autograd.grad(rot(q, k)[0], q, dq2, create_graph=True)
    gg, = torch.autograd.grad(g1, dq2, u)
    ref, mag = rotate(u, cos, sin, pos, interleaved)
    assert_within(gg, ref, rotation_error(ref, mag, F32), "second gradient")


def test_rotary_gradient_of_one_input_and_of_expanded_outputs():
    gen = _gen(3)
    q, k = _randn(gen, 9, 2, 32, dtype=BF16).requires_grad_(), _randn(gen, 9, 2, 32, dtype=BF16)
    cos, sin = vb.rotary_table(9, 32, device="cuda")
    a, b = vb.packed_rotary(q, k, cos, sin, cu_seqlens=_cu([4, 5]))
    assert a.requires_grad
    (a.sum() + b.sum()).backward()  # the gradient that arrives has no strides
    ref, mag = rotate(torch.ones_like(q), cos, sin, positions_of([4, 5]).cuda(), False, back=True)
    assert_within(q.grad, ref, rotation_error(ref, mag, BF16), "dq")
    q.grad = None
    a, b = vb.packed_rotary(q, k.requires_grad_(), cos, sin, cu_seqlens=_cu([4, 5]))
    b.sum().backward()
    assert q.grad is None
    assert_within(k.grad, ref, rotation_error(ref, mag, BF16), "dk")


def test_rotary_refusals():
    gen = _gen(4)
    q, k = _randn(gen, 6, 2, 64), _randn(gen, 6, 1, 64)
    cos, sin = vb.rotary_table(4, 64, device="cuda")
    rot = vb.packed_rotary
    with pytest.raises(ValueError, match="leave the table"):
        rot(q, k, cos, sin, cu_seqlens=_cu([1, 5]))
    with pytest.raises(ValueError, match="leave the table"):
        rot(q, k, cos, sin, positions=torch.tensor([0, 1, 2, 3, -1, 0]))
    with pytest.raises(ValueError, match="leave the table"):
        rot(q, k, cos, sin, positions=torch.tensor([0, 1, 2, 3, 2**32, 0]))  # 0 in 32 bits
    with pytest.raises(ValueError, match="one of"):
        rot(q, k, cos, sin)
    with pytest.raises(ValueError, match="one of"):
        rot(q, k, cos, sin, cu_seqlens=_cu([3, 3]), seqinfo=torch.tensor([3, 3]))
    with pytest.raises(ValueError, match="total tokens"):
        rot(q, k, cos, sin, cu_seqlens=_cu([3, 2]))
    with pytest.raises(ValueError, match="at least 2"):
        rot(q, k, cos, sin, cu_seqlens=_cu([]))
    with pytest.raises(AssertionError, match="fp32"):
        rot(q, k, cos.half(), sin.half(), cu_seqlens=_cu([3, 3]))
    with pytest.raises(AssertionError, match="device"):
        rot(q, k, cos.cpu(), sin.cpu(), cu_seqlens=_cu([3, 3]))
    with pytest.raises(AssertionError, match="dtype"):
        rot(q, k.half(), cos, sin, cu_seqlens=_cu([3, 3]))
    with pytest.raises(AssertionError, match="K shape"):
        rot(q, k[:5], cos, sin, cu_seqlens=_cu([3, 3]))
    with pytest.raises(AssertionError, match="rotary_dim"):
        rot(q[..., :32].contiguous(), None, cos, sin, cu_seqlens=_cu([3, 3]))
    with pytest.raises(AssertionError, match="positions has"):
        rot(q, k, cos, sin, positions=torch.zeros(5, dtype=torch.int64))


def test_rotary_unchecked_positions_and_rows_behind(unchecked):
    q = _randn(_gen(5), 6, 2, 64)
    cos, sin = vb.rotary_table(4, 64, device="cuda")
    _status()
    got, _ = vb.packed_rotary(q, None, cos, sin, cu_seqlens=_cu([2, 2]))
    assert (got[4:] == 0).all() and torch.isfinite(got).all() and _status() == [0, 0]
    got, _ = vb.packed_rotary(q, None, cos, sin, positions=torch.tensor([0, 4, 2**31 - 1, -1, 3, 0]))
    assert got[1:4].isnan().all() and not got[[0, 4, 5]].isnan().any() and _status() == [4, 910]
    assert vb.packed_rotary(q[:0], None, cos, sin, cu_seqlens=_cu([0]))[0].shape == (0, 2, 64)


def test_rotary_step_captured_and_replayed(unchecked):
    """Forward and gradients in a graph (torch wants no eager graph of the same leaves to live meanwhile)."""
    gen, lens = _gen(6), [40, 3]
    q, k = _randn(gen, 43, 4, 64, dtype=BF16).requires_grad_(), _randn(gen, 43, 2, 64, dtype=BF16).requires_grad_()
    dq, dk, cu = _randn(gen, 43, 4, 64, dtype=BF16), _randn(gen, 43, 2, 64, dtype=BF16), _cu(lens)
    cos, sin = vb.rotary_table(40, 64, device="cuda")

    def step():
        out = vb.packed_rotary(q, k, cos, sin, cu_seqlens=cu)
        return (*(x.detach() for x in out), *torch.autograd.grad(out, (q, k), (dq, dk)))

    want = [x.clone() for x in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- append --------------------------------------------------------------------------------------------------
def _append_ref(k, v, kc, vc, table, pos, seq, page):
    kc, vc = kc.clone(), vc.clone()
    ids, slot = table[seq, pos // page].long(), pos % page
    kc[ids, slot], vc[ids, slot] = k, v
    return kc, vc


@pytest.mark.parametrize("layout", ["nhd", "hnd", "halves"])
@pytest.mark.parametrize("dtype,H,H_kv,D,R,page,interleaved", [
    (BF16, 8, 8, 128, 128, 16, False), (F16, 8, 2, 64, 64, 5, True), (F32, 6, 3, 32, 16, 64, False), (BF16, 7, 1, 256, 100, 1, True),
    (F16, 4, 4, 16, 16, 17, False), (BF16, 5, 5, 64, 0, 16, False)])
def test_append(dtype, H, H_kv, D, R, page, interleaved, layout):
    gen = _gen(7)
    new, held = [3, 0, 1, 40, 7], [20, 9, 1, 40, 39]
    kc, vc, table = paged_cache(held, H_kv, D, page, dtype, gen, layout=layout, fill=7.0)
    T = sum(new)
    qkv = _randn(gen, T, H + 2 * H_kv, D, dtype=dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + H_kv], qkv[:, H + H_kv:]
    pos, seq = positions_of(new, held).cuda(), torch.repeat_interleave(torch.arange(5), torch.tensor(new)).cuda()
    before = kc.clone(), vc.clone()
    if R:
        cos, sin = vb.rotary_table(40, R, device="cuda")
        got = vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints(held), cu_seqlens=_cu(new), q=q, cos=cos, sin=sin,
                                 interleaved=interleaved)
        ref, mag = rotate(q, cos, sin, pos, interleaved)
        assert_within(got, ref, rotation_error(ref, mag, dtype), "q")
        rk = vb.packed_rotary(k, None, cos, sin, positions=pos, interleaved=interleaved)[0]  # checked above; the same arithmetic
    else:
        assert vb.paged_kv_append(k, v, kc, vc, page_table=table.long(), cache_seqlens=torch.tensor(held), seqinfo=torch.tensor(new)) is None
        rk = k
    want = _append_ref(rk, v, *before, table, pos, seq, page)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])  # every slot, the untouched ones too


@pytest.mark.parametrize("n", [1, 5, 300])
def test_append_of_one_token_each(n):
    gen, dtype = _gen(8), BF16
    held = [1 + 37 * i % 90 for i in range(n)]
    kc, vc, table = paged_cache(held, 4, 64, 16, dtype, gen, fill=0.0)
    q, k, v = (_randn(gen, n, h, 64, dtype=dtype) for h in (8, 4, 4))
    cos, sin = vb.rotary_table(90, 64, device="cuda")
    before, pos = (kc.clone(), vc.clone()), torch.tensor(held).cuda() - 1
    got = vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints(held), q=q, cos=cos, sin=sin)
    want_q, want_k = vb.packed_rotary(q, k, cos, sin, positions=pos)
    want = _append_ref(want_k, v, *before, table, pos, torch.arange(n, device="cuda"), 16)
    assert torch.equal(got, want_q) and torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_append_passes_over_padding_and_what_is_out_of_range(unchecked):
    gen = _gen(9)
    kc, vc, table = paged_cache([8, 8, 8, 8], 2, 64, 4, BF16, gen, fill=0.0)
    before = kc.clone(), vc.clone()
    q, k, v = (_randn(gen, 4, h, 64, dtype=BF16) for h in (2, 2, 2))
    cos, sin = vb.rotary_table(8, 64, device="cuda")
    _status()
    call = lambda lens, tab=table, **kw: vb.paged_kv_append(k, v, kc, vc, page_table=tab, cache_seqlens=_ints(lens), q=q, cos=cos, sin=sin, **kw)  # noqa: E731
    got = call([0, 0, 0, 0])
    assert (got == 0).all() and _status() == [0, 0]
    got = call([-1, 13, 2**31 - 1, 0])  # too short, too long for the table, padding
    assert got[:3].isnan().all() and (got[3] == 0).all() and _status() == [4, 911]
    bad = table.clone()
    bad[:, 0] = torch.tensor([-1, kc.shape[0], 2**31 - 1, -2**31])
    assert call([1, 1, 1, 1], bad).isnan().all() and _status() == [4, 911]
    assert call([9, 9, 9, 9]).isnan().all() and _status() == [4, 911]  # in the cache's range, not in the table of angles
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    # rows behind the last sequence, as in a batch padded for a graph
    got = call([5, 6, 0, 0], cu_seqlens=_cu([1, 1, 0, 0]))
    assert (got[2:] == 0).all() and _status() == [0, 0]
    want = _append_ref(vb.packed_rotary(k[:2], None, cos, sin, positions=_ints([4, 5]))[0], v[:2], *before, table, _ints([4, 5]).long(),
                       torch.arange(2, device="cuda"), 4)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_append_is_an_operation_in_place():
    """Autograd notices that a cache it has kept for a gradient was written to."""
    gen = _gen(22)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, F32, gen, fill=0.0)
    k, w = _randn(gen, 2, 2, 64), torch.ones((), device="cuda", requires_grad=True)
    y = (w * kc).sum()
    vb.paged_kv_append(k, k, kc, vc, page_table=table, cache_seqlens=_ints([8, 8]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        kc, vc = kc.clone(), vc.clone()
        vb.paged_kv_append(k, k, kc, vc, page_table=table, cache_seqlens=_ints([5, 6]))
        vb.paged_decode_attn(k, kc, vc, page_table=table, cache_seqlens=_ints([5, 6]))


def test_append_refusals():
    gen = _gen(10)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, BF16, gen, fill=0.0)
    before = kc.clone()
    k, v, q = (_randn(gen, 2, 2, 64, dtype=BF16) for _ in range(3))
    lens, (cos, sin) = _ints([8, 8]), vb.rotary_table(8, 64, device="cuda")
    call = lambda *a, page_table=table, cache_seqlens=lens, **kw: vb.paged_kv_append(*a, page_table=page_table, cache_seqlens=cache_seqlens, **kw)  # noqa: E731
    for match, error, f in [
            ("same slot", ValueError, lambda: call(k, v, kc, vc, page_table=table[:1].expand(2, -1))),
            ("among its tokens", ValueError, lambda: call(k, v, kc, vc, cache_seqlens=_ints([1, 8]), cu_seqlens=_cu([2, 0]))),
            ("leaves the table", ValueError, lambda: call(k, v, kc, vc, cos=cos[:7], sin=sin[:7])),
            ("cache_seqlens", ValueError, lambda: call(k, v, kc, vc, cache_seqlens=_ints([8, 13]))),
            ("outside", ValueError, lambda: call(k, v, kc, vc, page_table=table + 50)),
            ("outside", ValueError, lambda: call(k, v, kc, vc, page_table=table.long() - 2**32)),
            ("go together", ValueError, lambda: call(k, v, kc, vc, cos=cos)),
            ("without them", ValueError, lambda: call(k, v, kc, vc, q=q)),
            ("need cu_seqlens", AssertionError, lambda: call(k[:1], v[:1], kc, vc)),
            ("V shape", AssertionError, lambda: call(k, v[:, :1], kc, vc)),
            ("heads", AssertionError, lambda: call(k[:, :1], v[:, :1], kc, vc)),
            ("head_dim", AssertionError, lambda: call(k[..., :32].contiguous(), v[..., :32].contiguous(), kc, vc)),
            ("dtype", AssertionError, lambda: call(k, v, kc.half(), vc)),
            ("v_cache shape", AssertionError, lambda: call(k, v, kc, vc[1:])),
            ("same memory", AssertionError, lambda: call(k, v, kc, kc)),
            ("expanded", AssertionError, lambda: call(k, v, kc[:1].expand(4, -1, -1, -1), vc[:4])),
            ("last dim", AssertionError, lambda: call(k, v, kc.transpose(2, 3).contiguous().transpose(2, 3), vc)),
            ("sequences", AssertionError, lambda: call(k, v, kc, vc, page_table=table[:1])),
            ("integers", ValueError, lambda: call(k, v, kc, vc, page_table=table.float())),
            ("no gradient", RuntimeError, lambda: call(k.clone().requires_grad_(), v, kc, vc))]:
        with pytest.raises(error, match=match):
            f()
    assert torch.equal(kc, before)
    assert call(k[:0], v[:0], kc, vc, page_table=table[:0], cache_seqlens=lens[:0], q=q[:0], cos=cos, sin=sin).shape == (0, 2, 64)


# ---- attention -----------------------------------------------------------------------------------------------
def _check_decode(q, kc, vc, table, lens, what="", **kw):
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens), **kw)
    q4 = q if q.dim() == 4 else q.unsqueeze(1)
    ro, rl, eo, el = decode(q4, kc, vc, table, lens, **kw)
    assert o.dtype == q.dtype and o.is_contiguous()
    assert_within(o.view(q4.shape), ro, eo, f"o {what}")
    assert_within(lse.view(q4.shape[:-1]), rl, el, f"lse {what}")
    return o, lse


LENS = [1, 0, 16, 17, 63, 64, 65, 129, 500, 2]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,H_kv,T,page", [(2, 2, 1, 16), (8, 1, 1, 5), (14, 1, 1, 64), (6, 2, 4, 1), (8, 1, 7, 17), (5, 5, 2, 100), (20, 2, 9, 32), (23, 1, 1, 16),
                                           (20, 1, 2, 48), (4, 1, 4, 16)])
def test_decode(dtype, D, H, H_kv, T, page):
    """Row tiles of 8 to 64 rows and several of them, pages that end inside a block, sequences shorter than the new tokens; what
    no token holds is NaN."""
    gen = _gen(D + H)
    kc, vc, table = paged_cache(LENS, H_kv, D, page, dtype, gen)
    q = _randn(gen, len(LENS), T, H, D, dtype=dtype)
    _check_decode(q, kc, vc, table, LENS)
    if T == 1:
        _check_decode(q[:, 0], kc, vc, table, LENS)


@pytest.mark.parametrize("dtype,D,H,H_kv,T", [(BF16, 128, 8, 8, 1), (F16, 64, 8, 2, 1), (F32, 64, 4, 1, 1), (BF16, 256, 4, 1, 3), (F32, 256, 2, 1, 2)])
@pytest.mark.parametrize("lens", [[20000], [5, 9000, 0, 1], [4096] * 3, [1] * 600, [(i * 131) % 700 for i in range(333)]])
def test_decode_of_long_caches_and_of_many_sequences(dtype, D, H, H_kv, T, lens):
    """Units over many pieces and pieces over many units; more sequences than a block has threads."""
    gen = _gen(len(lens))
    kc, vc, table = paged_cache(lens, H_kv, D, 16, dtype, gen)
    q = _randn(gen, len(lens), T, H, D, dtype=dtype)
    o, lse = _check_decode(q, kc, vc, table, lens)
    again = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert torch.equal(again, o), "the same call gives the same bits"


@pytest.mark.parametrize("sms", [1, 2, 7, 61])
def test_decode_cut_otherwise(monkeypatch, sms):
    gen, lens = _gen(11), [3, 1000, 64, 0, 257]
    kc, vc, table = paged_cache(lens, 2, 64, 16, BF16, gen)
    q = _randn(gen, len(lens), 2, 6, 64, dtype=BF16)
    monkeypatch.setattr(_lib, "sm_count", lambda device: sms)
    monkeypatch.setattr(paged, "_plans", {})
    _check_decode(q, kc, vc, table, lens, what=f"{sms} SMs")


@pytest.mark.parametrize("layout", ["nhd", "hnd", "halves"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_layouts_views_and_scale(dtype, layout):
    gen, lens, H, H_kv, D = _gen(12), [40, 3, 200], 6, 3, 64
    kc, vc, table = paged_cache(lens, H_kv, D, 8, dtype, gen, layout=layout)
    wide = torch.zeros(3, table.shape[1] + 5, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    qkv = _randn(gen, 3, H + 4, D, dtype=dtype)
    want, _ = _check_decode(qkv[:, :H].contiguous(), kc, vc, table, lens)
    flat = torch.cat([qkv.new_zeros(1), qkv[:, :H].reshape(-1)])[1:].view(3, H, D)  # a base that is no multiple of 16 bytes
    for q, t in ((qkv[:, :H], wide[:, :table.shape[1]]), (flat, table.long()), (qkv[:, :H].transpose(1, 2).contiguous().transpose(1, 2), wide)):
        assert torch.equal(vb.paged_decode_attn(q, kc, vc, page_table=t, cache_seqlens=torch.tensor(lens)), want)
    _check_decode(qkv[:, :H], kc, vc, table, lens, scale=0.03)
    _check_decode(qkv[:, :H], kc, vc, table, lens, scale=-0.2)
    o, lse = vb.paged_decode_attn_with_lse(qkv[:, :H], kc, vc, page_table=table, cache_seqlens=_ints(lens), scale=0.0)
    ro, rl, eo, el = decode(qkv[:, None, :H], kc, vc, table, lens, scale=0.0)
    assert_within(o.unsqueeze(1), ro, eo, "o, equal weights")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_decode_what_a_row_does_not_see_does_not_reach_it(dtype, bad):
    """Of four new tokens the last one's K and V are NaN or infinite: the rows before it do not see it."""
    gen, T, D = _gen(13), 4, 64
    lens = [4, 16, 17, 20, 64, 67, 130]
    kc, vc, table = paged_cache(lens, 2, D, 16, dtype, gen)
    q = _randn(gen, len(lens), T, 6, D, dtype=dtype)
    # (their sums may go another way where V is not finite, so they are held to the formula like any other row, not to the bits
    # of a call whose V is finite)
    want, _, off, _ = decode(q, kc, vc, table, lens)
    for which in (vc, kc):
        for i, n in enumerate(lens):
            which[table[i, (n - 1) // 16].long(), (n - 1) % 16] = bad
        got = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
        assert_within(got[:, :T - 1], want[:, :T - 1], off[:, :T - 1], "rows that do not see it")
        assert not torch.isfinite(got[:, T - 1]).all(-1).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_of_bad_and_extreme_scores(dtype):
    gen, lens, D = _gen(14), [100, 300, 70], 64
    kc, vc, table = paged_cache(lens, 1, D, 16, dtype, gen)
    q = _randn(gen, 3, 2, D, dtype=dtype)
    kc[table[0, 2].long(), 3] = float("nan")            # one bad key of sequence 0
    kc[table[1, 0].long(), :, :, 0] = 30000.0           # a few keys far above the others
    q[2] = 0
    kc[table[2, :5].long()] = -float("inf")             # 0 * inf: every score of sequence 2 is NaN
    o = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert o[0].isnan().all() and o[2].isnan().all() and torch.isfinite(o[1]).all()
    kc[table[0, 2].long(), 3] = 0
    q[2] = 1                                            # every score -inf: 0 / 0, as in the formula
    o, lse = vb.paged_decode_attn_with_lse(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert o[2].isnan().all() and (lse[2] == -math.inf).all()
    kc[table[2, 0].long(), 5] = 0.5                     # but one key: all the weight is its own
    o = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert torch.equal(o[2], vc[table[2, 0].long(), 5].expand(2, D))


def test_decode_offsets_past_32_bits():
    """Pages whose elements lie behind the first 2^31 of a cache, for the append and the attention."""
    gen, H_kv, D, page = _gen(15), 8, 128, 64
    pool = 2**31 // (page * H_kv * D) + 9
    kc, vc = (torch.empty(pool, page, H_kv, D, dtype=BF16, device="cuda") for _ in range(2))
    lens = [150, 64]
    table = _ints([[pool - 1, 1, pool - 3], [pool - 4, 0, 0]])
    for t in (pool - 1, 1, pool - 3, pool - 4):
        kc[t], vc[t] = _randn(gen, page, H_kv, D, dtype=BF16), _randn(gen, page, H_kv, D, dtype=BF16)
    k, v, q = (_randn(gen, 2, h, D, dtype=BF16) for h in (H_kv, H_kv, 16))
    vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert torch.equal(kc[pool - 3, 149 % 64], k[0]) and torch.equal(vc[pool - 4, 63], v[1])
    _check_decode(q, kc, vc, table, lens)


def test_sequences_that_share_a_prefix():
    """Pages that are only read may be anybody's: a common prefix, a sequence twice, more of the cache than its lengths reach."""
    gen, page = _gen(23), 16
    kc, vc, table = paged_cache([64, 64, 64], 2, 64, page, BF16, gen)
    table[1, :3] = table[0, :3]
    table[2] = table[0]
    lens = [50, 61, 50]
    q, k, v = (_randn(gen, 3, h, 64, dtype=BF16) for h in (6, 2, 2))
    q[2] = q[0]
    vb.paged_kv_append(k[:2], v[:2], kc, vc, page_table=table[:2], cache_seqlens=_ints(lens[:2]))
    with pytest.raises(ValueError, match="same slot"):
        vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    _check_decode(q, kc, vc, table, lens)


def test_decode_unchecked_pages_and_lengths(unchecked):
    """What is out of range is not followed: no fault, the status word tells, and the other sequences are right."""
    gen, lens = _gen(16), [40, 100, 33]
    kc, vc, table = paged_cache(lens, 2, 64, 16, BF16, gen)
    q = _randn(gen, 3, 4, 64, dtype=BF16)
    _status()
    want = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints(lens))
    assert _status() == [0, 0]
    for page in (-1, kc.shape[0], 2**31 - 1, -2**31):
        bad = table.clone()
        bad[1, 2] = page
        got = vb.paged_decode_attn(q, kc, vc, page_table=bad, cache_seqlens=_ints(lens))
        assert _status() == [4, 912] and torch.equal(got[[0, 2]], want[[0, 2]])
    got = vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints([40, -5, 33]))
    assert torch.equal(got[[0, 2]], want[[0, 2]]) and (got[1] == 0).all() and _status() == [4, 912]


def test_errors_found_on_the_device_can_be_raised(unchecked):
    gen = _gen(24)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, BF16, gen, fill=0.0)
    q, lens, bad = _randn(gen, 2, 2, 64, dtype=BF16), _ints([8, 8]), table + 99
    cos, sin = vb.rotary_table(3, 64, device="cuda")
    _status()
    _lib.set_check_status(True)
    try:
        for f in (lambda: vb.paged_decode_attn(q, kc, vc, page_table=bad, cache_seqlens=lens),
                  lambda: vb.paged_kv_append(q, q, kc, vc, page_table=bad, cache_seqlens=lens),
                  lambda: vb.packed_rotary(q, None, cos, sin, positions=_ints([2, 3]))):
            with pytest.raises(RuntimeError, match="outside its array"):
                f()
        vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=lens)
    finally:
        _lib.set_check_status(False)


def test_decode_refusals():
    gen = _gen(17)
    kc, vc, table = paged_cache([8, 8], 2, 64, 4, BF16, gen)
    q, lens = _randn(gen, 2, 4, 64, dtype=BF16), _ints([8, 8])
    call = lambda q=q, kc=kc, vc=vc, page_table=table, cache_seqlens=lens: vb.paged_decode_attn(q, kc, vc, page_table=page_table, cache_seqlens=cache_seqlens)  # noqa: E731
    for match, error, f in [
            ("cache_seqlens", ValueError, lambda: call(cache_seqlens=_ints([8, 13]))),
            ("cache_seqlens", ValueError, lambda: call(cache_seqlens=_ints([8, -1]))),
            ("cache_seqlens", ValueError, lambda: call(cache_seqlens=torch.tensor([8, 2**32 + 8]))),
            ("outside", ValueError, lambda: call(page_table=table.long() + 2**32)),
            ("outside", ValueError, lambda: call(page_table=table + 50)),
            ("1-D", ValueError, lambda: call(cache_seqlens=lens[None])),
            ("2-D", ValueError, lambda: call(page_table=table[0])),
            ("divide", AssertionError, lambda: call(q=q[:, :3])),
            ("sequences", AssertionError, lambda: call(q=q[:1])),
            ("dtype", AssertionError, lambda: call(q=q.float())),
            ("16 bytes", ValueError, lambda: call(kc=torch.zeros(kc.numel() + 1, dtype=BF16, device="cuda")[1:].view(kc.shape))),
            ("16 bytes", ValueError, lambda: call(vc=torch.zeros(*vc.shape[:3], 68, dtype=BF16, device="cuda")[..., :64])),
            ("empty cache", AssertionError, lambda: call(kc=kc[:0], vc=vc[:0])),
            ("no gradient", RuntimeError, lambda: call(q=q.clone().requires_grad_()))]:
        with pytest.raises(error, match=match):
            f()
    with torch.no_grad():
        call(q=q.clone().requires_grad_())
    assert call(q=q[:0], page_table=table[:0], cache_seqlens=lens[:0]).shape == (0, 4, 64)


def test_check_refused_while_captured():
    gen = _gen(18)
    kc, vc, table = paged_cache([8], 2, 64, 4, BF16, gen)
    q, lens = _randn(gen, 1, 4, 64, dtype=BF16), _ints([8])
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="captured"):
            vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=lens)
        q.add_(0)


# ---- together ------------------------------------------------------------------------------------------------
def _full(q, k, v, cos, sin, lens):
    """Causal attention over whole sequences, rotated, in 64 bits, from the unrotated 16-bit inputs."""
    pos = positions_of(lens).cuda()
    q, k = rotate(q, cos, sin, pos, False)[0], rotate(k, cos, sin, pos, False)[0]
    g, out, at = q.shape[1] // k.shape[1], [], 0
    for n in lens:
        qq, kk, vv = q[at:at + n], k[at:at + n].repeat_interleave(g, 1), v[at:at + n].double().repeat_interleave(g, 1)
        s = torch.einsum("ihd,jhd->hij", qq, kk) * q.shape[2] ** -0.5
        s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
        out.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), vv))
        at += n
    return torch.cat(out)


@pytest.mark.parametrize("captured", [False, True])
def test_prompt_then_tokens(captured):
    """Prompts through packed_varlen_attn into the cache, then a token at a time (in one graph, its lengths on the device), then
    three proposed tokens at once: what full attention over the whole sequences gives.  One sequence of the batch is padding."""
    gen, dtype, H, H_kv, D, page = _gen(19), BF16, 8, 2, 64, 16
    prompt, steps = [5, 33, 1], 20
    total = [n + steps + 3 for n in prompt]
    q, k, v = (_randn(gen, sum(total), h, D, dtype=dtype) for h in (H, H_kv, H_kv))
    cos, sin = vb.rotary_table(max(total), D, device="cuda")
    want = _full(q, k, v, cos, sin, total)
    starts = [0, total[0], total[0] + total[1]]
    rows = lambda a, b: torch.cat([torch.arange(s + x, s + y) for s, x, y in zip(starts, a, b)]).cuda()  # noqa: E731
    kc, vc = (torch.full((20, page, H_kv, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.randperm(20, generator=gen, device="cuda").to(torch.int32)[:16].view(4, 4).contiguous()
    lens = _ints(prompt + [0])

    def close(got, at):
        # rotated q, k and P are rounded to 16 bits on the way (2^-8 each of O(1) scores): a few 2^-8 of O(1) outputs
        assert (got.double() - want[at]).abs().max() <= 6 * 2.0 ** -8

    at = rows([0] * 3, prompt)
    cu = _cu(prompt)
    qr, kr = vb.packed_rotary(q[at], k[at], cos, sin, cu_seqlens=cu)
    close(vb.packed_varlen_attn(qr, kr, v[at], cu_seqlens_q=cu, cu_seqlens_k=cu, causal=True), at)
    vb.paged_kv_append(kr, v[at], kc, vc, page_table=table[:3], cache_seqlens=lens[:3], cu_seqlens=cu)

    xq, xk, xv = (torch.zeros(4, h, D, dtype=dtype, device="cuda") for h in (H, H_kv, H_kv))
    live = _ints([1, 1, 1, 0])

    def step():
        lens.add_(live)
        a = vb.paged_kv_append(xk, xv, kc, vc, page_table=table, cache_seqlens=lens, q=xq, cos=cos, sin=sin)
        return vb.paged_decode_attn(a, kc, vc, page_table=table, cache_seqlens=lens)

    graph = None
    if captured:
        vb.set_validate_cu_seqlens(False)
        keep = [x.clone() for x in (kc, vc, lens)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for x, y in zip((kc, vc, lens), keep):
            x.copy_(y)
    try:
        for i in range(steps):
            at = rows([n + i for n in prompt], [n + i + 1 for n in prompt])
            for x, y in ((xq, q), (xk, k), (xv, v)):
                x[:3] = y[at]
            if captured:
                graph.replay()
            else:
                out = step()
            close(out[:3], at)
            assert (out[3] == 0).all()
        # three proposed tokens of each sequence at once
        at = rows([n + steps for n in prompt], total)
        lens[:3] += 3
        qr = vb.paged_kv_append(k[at], v[at], kc, vc, page_table=table[:3], cache_seqlens=lens[:3], cu_seqlens=_cu([3, 3, 3]), q=q[at], cos=cos, sin=sin)
        close(vb.paged_decode_attn(qr.view(3, 3, H, D), kc, vc, page_table=table[:3], cache_seqlens=lens[:3]).view(9, H, D), at)
    finally:
        vb.set_validate_cu_seqlens(True)


def test_two_streams_and_two_graphs_at_once(unchecked):
    """Calls on two streams and two graphs replayed beside one another share nothing."""
    gen, cases = _gen(20), []
    for lens, H_kv in (([3000, 17, 900], 2), ([1, 5000], 4)):
        kc, vc, table = paged_cache(lens, H_kv, 128, 16, BF16, gen)
        q = _randn(gen, len(lens), 8, 128, dtype=BF16)
        cases.append((q, kc, vc, dict(page_table=table, cache_seqlens=_ints(lens))))
    want = [vb.paged_decode_attn(q, kc, vc, **kw) for q, kc, vc, kw in cases]
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], []
    torch.cuda.synchronize()
    for q, kc, vc, kw in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(vb.paged_decode_attn(q, kc, vc, **kw))
        graphs.append(g)
    for _ in range(20):
        got = []
        for s, g, (q, kc, vc, kw) in zip(streams, graphs, cases):
            with torch.cuda.stream(s):
                g.replay()
                got.append(vb.paged_decode_attn(q, kc, vc, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got + outs, want + want))


def test_the_kernels_of_this_library_ran():
    before = {n: v[2] for n, v in _lib.profile_read().items()}
    gen = _gen(21)
    kc, vc, table = paged_cache([5000], 2, 64, 16, BF16, gen)
    q = _randn(gen, 1, 2, 64, dtype=BF16)
    cos, sin = vb.rotary_table(5000, 64, device="cuda")
    vb.packed_rotary(q, None, cos, sin, cu_seqlens=_cu([1]))
    vb.paged_kv_append(q, q, kc, vc, page_table=table, cache_seqlens=_ints([5000]))
    vb.paged_decode_attn(q, kc, vc, page_table=table, cache_seqlens=_ints([5000]))
    after = {n: v[2] for n, v in _lib.profile_read().items()}
    for name in ("rotary_kernel", "rotary_kernel<append>", "paged_decode_kernel", "paged_combine_kernel"):
        assert after.get(name, 0) == before.get(name, 0) + 1, name


# ---- long batches: rows through shared memory ---------------------------------------------------------------
@pytest.mark.parametrize("dtype,H,H_kv,D,R,interleaved,view", [
    (BF16, 32, 8, 128, 128, False, False), (F16, 32, 8, 128, 64, True, True), (F32, 8, 2, 64, 58, False, False), (BF16, 8, 8, 64, 64, False, True),
    (F16, 7, 1, 256, 100, True, False), (F32, 4, 4, 128, 128, True, True), (BF16, 20, 5, 32, 30, False, False)])
def test_rotary_and_append_of_long_batches(dtype, H, H_kv, D, R, interleaved, view):
    """Batches over the size from which token rows go through shared memory, their last tile part full."""
    gen = _gen(H + D)
    T = (11 << 20) // ((H + H_kv) * D * dtype.itemsize) + 3
    lens = [1, 0, 700, 5, 33]
    lens.append(T - sum(lens))
    qkv = _randn(gen, T, H + 2 * H_kv, D, dtype=dtype)
    q, k, v = qkv[:, :H], qkv[:, H:H + H_kv], qkv[:, H + H_kv:]
    if not view:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    cos, sin = vb.rotary_table(max(lens), R, device="cuda")
    pos = positions_of(lens).cuda()
    before = sum(x[2] for n, x in _lib.profile_read().items() if n == "rotary_kernel<rows>")
    out = vb.packed_rotary(q, k, cos, sin, cu_seqlens=_cu(lens), interleaved=interleaved)
    for name, x, y in zip("qk", (q, k), out):
        ref, mag = rotate(x, cos, sin, pos, interleaved)
        assert_within(y, ref, rotation_error(ref, mag, dtype), name)
    assert torch.equal(vb.packed_rotary(q, None, cos, sin, positions=pos, interleaved=interleaved)[0], out[0])
    for page, layout in ((16, "nhd"), (7, "hnd")):
        kc, vc, table = paged_cache(lens, H_kv, D, page, dtype, gen, layout=layout, fill=7.0)
        want = _append_ref(out[1], v, kc, vc, table, pos, torch.repeat_interleave(torch.arange(6), torch.tensor(lens)).cuda(), page)
        got = vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=_ints(lens), cu_seqlens=_cu(lens), q=q, cos=cos, sin=sin,
                                 interleaved=interleaved)
        assert torch.equal(got, out[0]) and torch.equal(kc, want[0]) and torch.equal(vc, want[1])
        vb.paged_kv_append(out[1], v, kc, vc, page_table=table, cache_seqlens=_ints(lens), cu_seqlens=_cu(lens))
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    assert sum(x[2] for n, x in _lib.profile_read().items() if n == "rotary_kernel<rows>") >= before + 3


def test_long_batches_with_rows_behind_padding_and_bad_places(unchecked):
    gen, H, D = _gen(31), 8, 128
    T = 6000
    q, k, v = (_randn(gen, T, H, D, dtype=BF16) for _ in range(3))
    cos, sin = vb.rotary_table(3000, D, device="cuda")
    lens = [1500, 100, 2500]  # 1900 rows behind
    _status()
    a, b = vb.packed_rotary(q, k, cos, sin, cu_seqlens=_cu(lens))
    assert (a[4100:] == 0).all() and (b[4100:] == 0).all() and _status() == [0, 0]
    pos = positions_of(lens).cuda()
    short = vb.packed_rotary(q[:4100], k[:4100], cos, sin, positions=pos)
    assert torch.equal(a[:4100], short[0]) and torch.equal(b[:4100], short[1])
    kc, vc, table = paged_cache([1500, 100, 2500], H, D, 16, BF16, gen, fill=0.0)
    before, bad = (kc.clone(), vc.clone()), table.clone()
    bad[0, 40] = kc.shape[0]
    got = vb.paged_kv_append(k, v, kc, vc, page_table=bad, cache_seqlens=_ints([1500, 0, 2500]), cu_seqlens=_cu(lens), q=q, cos=cos, sin=sin)
    assert _status() == [4, 911]
    assert got[640:656].isnan().all() and (got[1500:1600] == 0).all() and (got[4100:] == 0).all()
    keep = torch.ones(4100, dtype=torch.bool, device="cuda")
    keep[640:656] = keep[1500:1600] = False
    assert torch.equal(got[:4100][keep], a[:4100][keep])
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(lens)).cuda()
    want = _append_ref(b[:4100][keep], v[:4100][keep], *before, table, pos[keep], seq[keep], 16)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_threads_on_streams_of_their_own(unchecked):
    """Two threads append and attend on streams of their own, layouts that no call has checked yet among them."""
    import threading
    cases = []
    for seed, (n, H, H_kv, page) in enumerate([(5, 9, 3, 24), (130, 8, 1, 8)]):
        gen, lens = _gen(40 + seed), [1 + (37 * i) % 300 for i in range(n)]
        kc, vc, table = paged_cache(lens, H_kv, 64, page, BF16, gen, fill=0.0)
        q, k, v = (_randn(gen, n, h, 64, dtype=BF16) for h in (H, H_kv, H_kv))
        cases.append((q, k, v, kc, vc, table, lens, vb.rotary_table(301, 64, device="cuda")))
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            q, k, v, kc, vc, table, lens, (cos, sin) = cases[i]
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                held = _ints(lens)
                for _ in range(30):
                    a = vb.paged_kv_append(k, v, kc, vc, page_table=table, cache_seqlens=held, q=q, cos=cos, sin=sin)
                    o = vb.paged_decode_attn_with_lse(a, kc, vc, page_table=table, cache_seqlens=held)
                stream.synchronize()
            got[i] = a, *o
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for (q, k, v, kc, vc, table, lens, _), (a, o, lse) in zip(cases, got):
        ro, rl, eo, el = decode(a.unsqueeze(1), kc, vc, table, lens)
        assert_within(o.unsqueeze(1), ro, eo, "o")
        assert_within(lse.unsqueeze(1), rl, el, "lse")
