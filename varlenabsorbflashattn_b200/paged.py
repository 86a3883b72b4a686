"""Positions and serving: rotation of packed queries and keys, a paged key/value cache, attention of new tokens over it.

The reference has no counterpart.  The calls stand around `packed_varlen_attn`: a training step or a prompt runs

    q, k = packed_rotary(q, k, cos, sin, cu_seqlens=cu)
    o = packed_varlen_attn(q, k, v, cu_seqlens_q=cu, cu_seqlens_k=cu, causal=True)
    paged_kv_append(k, v, k_cache, v_cache, page_table=table, cache_seqlens=lens, cu_seqlens=cu)     # serving

and every token after it

    lens += 1
    q = paged_kv_append(k, v, k_cache, v_cache, page_table=table, cache_seqlens=lens, q=q, cos=cos, sin=sin)
    o = paged_decode_attn(q, k_cache, v_cache, page_table=table, cache_seqlens=lens)

A cache is a pair of tensors [num_pages, page_size, H_kv, D], any strides as long as the last dim is contiguous (halves
of one tensor, or a transposed view of [num_pages, H_kv, page_size, D]).  Token j of sequence s lies in slot
j % page_size of page page_table[s, j // page_size].  `cache_seqlens` counts the tokens of a sequence with the new ones
among them, in both calls; a sequence of length 0 is padding, which is neither written nor attended over.

The first call on a device is made outside a CUDA graph's capture (it makes the device's status word); after it all calls can be captured
once validation is off, with lengths and tables that change in place between replays.

As in `packed_varlen_attn` all arithmetic happens in libvafa_b200.so.  With validation on (`set_validate_cu_seqlens`,
the default) lengths, page ids and positions are checked on the host, which waits for the device; a serving loop
switches it off.  Unchecked, an index that leaves its array is not followed on the device either: nothing outside the tensors is read or
written, and the status word reports it (`_lib.check_status`).  Lengths, tables, positions and prefix sums are taken from any integer type and device;
int32 on the device of the rest, in tensors of three dims (four for a decode of several tokens), is the fast way: other ones are converted in each call.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib
from . import varlen as _varlen
from .varlen import _SUPPORTED_HEAD_DIMS, _check_cu, _lengths_to_cu

__all__ = ["rotary_table", "packed_rotary", "paged_kv_append", "paged_decode_attn", "paged_decode_attn_with_lse"]


def _need(ok: bool, message) -> None:
    """The assertion of the other operators, which -O does not take out: the kernels go by what it says."""
    if not ok:
        raise AssertionError(message())


# ------------------------------------------------------------------------------------------------
# arguments
# ------------------------------------------------------------------------------------------------
def _counts(x: torch.Tensor, name: str) -> torch.Tensor:
    """The library counts in 32 bits: a size beyond them (an expanded tensor has it for nothing) must not arrive as a smaller one."""
    if max(x.shape, default=0) > 2**31 - 1:
        raise ValueError(f"{name}: shape {tuple(x.shape)} exceeds int32 range")
    return x


def _rows(x: torch.Tensor, name: str) -> Tuple[torch.Tensor, bool]:
    """[T, H, D] of a packed tensor, at its own strides as long as the last dim is contiguous."""
    _counts(x, name)
    was4 = x.dim() == 4
    if was4:
        if x.shape[0] != 1:
            raise ValueError(f"{name}: 4-D input must have batch=1 (packed varlen), got shape {tuple(x.shape)}")
        x = x[0]
    elif x.dim() != 3:
        raise ValueError(f"{name}: expected 3-D [T,H,D] or 4-D [1,T,H,D], got {x.dim()}-D")
    return (x if x.stride(2) == 1 else x.contiguous()), was4


def _check_heads(x: torch.Tensor, name: str) -> None:
    _need(x.is_cuda, lambda: f"{name}: CUDA tensors are required (there is no CPU path)")
    _need(x.dtype in _lib.DTYPE_CODE, lambda: f"{name} must be fp32, bf16 or fp16, got {x.dtype}")
    _need(x.shape[-1] in _SUPPORTED_HEAD_DIMS, lambda: f"head_dim {x.shape[-1]} not supported (try 64/128/256)")


def _like(x: torch.Tensor, ref: torch.Tensor, name: str) -> None:
    _need(x.device == ref.device, lambda: f"{name}: on {x.device}, the others on {ref.device}")
    _need(x.dtype == ref.dtype, lambda: f"{name}: dtype {x.dtype}, the others have {ref.dtype}")


_WIDE = (torch.int64, torch.uint64, torch.uint32)


def _ints(t: torch.Tensor, device: torch.device, name: str, dims: int = 1) -> torch.Tensor:
    """int32 on the device, the last dim contiguous; values beyond 32 bits as the nearest ones, which the kernels refuse as they do those."""
    if t.dim() != dims:
        raise ValueError(f"{name}: must be {dims}-D, got shape {tuple(t.shape)}")
    _counts(t, name)
    if t.dtype is not torch.int32 or t.device != device:
        if t.is_floating_point() or t.dtype == torch.bool:
            raise ValueError(f"{name}: must hold integers, got {t.dtype}")
        if t.dtype in _WIDE:  # what 32 bits do not hold must not arrive as something that they do
            t = t.to(torch.int64).clamp(-2**31, 2**31 - 1)
        t = t.to(device=device, dtype=torch.int32)
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _check_angles(cos: torch.Tensor, sin: torch.Tensor, ref: torch.Tensor) -> int:
    _need(cos.dim() == 2 and cos.shape == sin.shape, lambda: f"cos/sin must be [positions, rotary_dim/2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    _need(cos.dtype == sin.dtype == torch.float32, lambda: f"cos/sin must be fp32, got {cos.dtype} and {sin.dtype}")
    _need(cos.device == ref.device and sin.device == ref.device, lambda: "cos/sin must be on the device of q and k")
    _need(cos.is_contiguous() and sin.is_contiguous(), lambda: "cos/sin must be contiguous")
    _counts(cos, "cos/sin")
    _need(2 <= 2 * cos.shape[1] <= ref.shape[-1], lambda: f"rotary_dim {2 * cos.shape[1]} must be 2 to head_dim {ref.shape[-1]}")
    return 2 * cos.shape[1]


def _no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or detach its inputs")


def _no_tangent(what: str, *tensors) -> None:
    """Forward mode asks neither for requires_grad nor for grad mode: a tangent would be dropped in silence."""
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")


def _host(t: torch.Tensor) -> torch.Tensor:
    """A copy to look over on the host (waits for the device)."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("lengths, page ids and positions cannot be checked on the host while the stream is captured: "
                           "switch the check off (set_validate_cu_seqlens)")
    return t.detach().to("cpu", torch.int64)


def _check_cache(k_cache, v_cache, page_table, cache_seqlens, ref) -> None:
    for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _need(c.dim() == 4, lambda: f"{name}: expected [num_pages, page_size, H_kv, D], got shape {tuple(c.shape)}")
        _like(_counts(c, name), ref, name)
        _need(c.stride(3) == 1, lambda: f"{name}: the last dim must be contiguous")
    _need(k_cache.shape == v_cache.shape, lambda: f"v_cache shape {tuple(v_cache.shape)}, k_cache {tuple(k_cache.shape)}")
    _need(k_cache.shape[3] == ref.shape[-1], lambda: f"caches have head_dim {k_cache.shape[3]}, the new tokens {ref.shape[-1]}")
    _need(k_cache.numel() > 0, lambda: f"empty cache {tuple(k_cache.shape)}")
    _need(page_table.shape[0] == cache_seqlens.shape[0],
          lambda: f"page_table has {page_table.shape[0]} sequences, cache_seqlens {cache_seqlens.shape[0]}")
    _need(page_table.shape[1] > 0 and page_table.shape[1] * k_cache.shape[1] < 2**31 - 65536,
          lambda: f"page_table width {page_table.shape[1]} x page_size {k_cache.shape[1]} out of range")


def _check_pages(lens: torch.Tensor, table: torch.Tensor, num_pages: int, page_size: int) -> None:
    """Host copies: every length fits its row of the table, every page that it reaches is one of the cache's."""
    if lens.numel() == 0:
        return
    if int(lens.min()) < 0 or int(lens.max()) > table.shape[1] * page_size:
        raise ValueError(f"cache_seqlens must be 0 to {table.shape[1] * page_size} (page_table width x page_size), "
                         f"got {int(lens.min())} to {int(lens.max())}")
    used = torch.arange(table.shape[1])[None, :] < ((lens + page_size - 1) // page_size)[:, None]
    if bool((used & ((table < 0) | (table >= num_pages))).any()):
        raise ValueError(f"page_table names pages outside 0 to {num_pages - 1}")


# ------------------------------------------------------------------------------------------------
# plans
# ------------------------------------------------------------------------------------------------
class _Plan:
    """What the checks of a call make of its tensors' shapes, strides, types and devices: the argument struct but for the addresses.

    A serving loop makes the same calls thousands of times and a check of each argument costs as much as the kernels of a
    small step (35 us of a 40 us call), so calls of the same layout are checked once.  Nothing of the tensors' contents or addresses is in a plan."""
    __slots__ = ("layout", "struct", "device", "index", "status", "call", "workspace", "out", "keep")

    def __init__(self, struct, device, call, **more):
        self.layout, self.struct = bytes(struct), type(struct)
        self.device, self.index = device, device.index
        self.keep = _lib.status_word(device)  # (held, so that its address stays)
        self.status = self.keep.data_ptr()
        self.call = getattr(_lib.load(), call)
        self.workspace, self.out = more.get("workspace", 0), more.get("out")

    def args(self):
        a = self.struct.from_buffer_copy(self.layout)
        a.status = self.status
        return a

    def run(self, a, what: str) -> None:
        here = torch._C._cuda_getDevice() == self.index
        if here:
            rc = self.call(a, torch._C._cuda_getCurrentRawStream(self.index))
        else:
            with torch.cuda.device(self.device):
                rc = self.call(a, torch._C._cuda_getCurrentRawStream(self.index))
        if rc:
            _lib.check(rc, what)
        if _lib._check_after_each_op:
            with _lib.on_device(self.device):
                _lib.check_status(self.device)


_PACKED = torch.contiguous_format
_plans: dict = {}
_MOST_PLANS = 4096


def _keep(key, plan: _Plan) -> _Plan:
    if len(_plans) >= _MOST_PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _layout(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


# ------------------------------------------------------------------------------------------------
# rotation
# ------------------------------------------------------------------------------------------------
def rotary_table(positions: int, rotary_dim: int, *, base: float = 10000.0, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [positions, rotary_dim / 2], of the angles p * base^(-2 i / rotary_dim), computed in 64 bits.

    Made once and kept by the program.  The operators take any table of this shape, so other frequencies
    (interpolated, per-band scaled) are the caller's to fill in."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if positions < 0:
        raise ValueError(f"positions must not be negative, got {positions}")
    w = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * w
    return angle.cos().float(), angle.sin().float()


def _rotary_plan(q, k, cos, positions, cu, interleaved: bool, inverse: bool) -> _Plan:
    ref = q if q is not None else k
    T, D = ref.shape[0], ref.shape[2]
    H, H_kv = (0 if x is None else x.shape[1] for x in (q, k))
    qs, ks = ((0, 0) if x is None else x.stride()[:2] for x in (q, k))
    a = _lib.RotaryArgs(*[None] * 8, *qs, *ks, 0 if cu is None else cu.numel() - 1, T, H, H_kv, D, 2 * cos.shape[1], cos.shape[0],
                        _lib.DTYPE_CODE[ref.dtype], interleaved, inverse)
    return _Plan(a, ref.device, "vafa_rotary", out=T)


def _rotate(plan: _Plan, q, k, cos, sin, positions, cu):
    qo = None if q is None else torch.empty_like(q, memory_format=_PACKED)
    ko = None if k is None else torch.empty_like(k, memory_format=_PACKED)
    if plan.out == 0:
        return qo, ko
    a = plan.args()
    if q is not None:
        a.q, a.q_out = q.data_ptr(), qo.data_ptr()
    if k is not None:
        a.k, a.k_out = k.data_ptr(), ko.data_ptr()
    a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
    if cu is not None:
        a.cu_seqlens = cu.data_ptr()
    else:
        a.positions = positions.data_ptr()
    plan.run(a, "vafa_rotary")
    return qo, ko


class _PackedRotary(torch.autograd.Function):
    """y = R x per token and pair; the gradient is R^T dy, the rotation back, which has a gradient in turn."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, cu, plan, interleaved, inverse):
        ctx.save_for_backward(cos, sin, positions if cu is None else cu)
        ctx.flags = cu is None, interleaved, inverse
        ctx.set_materialize_grads(False)
        out = _rotate(plan, q, k, cos, sin, positions, cu)
        # (what is rotated beside an input with a gradient has none itself)
        ctx.mark_non_differentiable(*(y for y, needed in zip(out, ctx.needs_input_grad) if y is not None and not needed))
        return out

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, where = ctx.saved_tensors
        by_position, interleaved, inverse = ctx.flags
        positions, cu = (where, None) if by_position else (None, where)
        dq = _gradient(dq) if ctx.needs_input_grad[0] else None
        dk = _gradient(dk) if ctx.needs_input_grad[1] else None
        if dq is None and dk is None:
            return (None,) * 9
        key = ("rotary", _layout(dq), _layout(dk), cos.shape, where.shape, by_position, interleaved, not inverse)
        plan = _plans.get(key) or _keep(key, _rotary_plan(dq, dk, cos, positions, cu, interleaved, not inverse))
        if torch.is_grad_enabled():
            dq, dk = _PackedRotary.apply(dq, dk, cos, sin, positions, cu, plan, interleaved, not inverse)
        else:
            dq, dk = _rotate(plan, dq, dk, cos, sin, positions, cu)
        return dq, dk, None, None, None, None, None, None, None


def _gradient(d):
    return d if d is None or d.stride(2) == 1 else d.contiguous()


def packed_rotary(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    cu_seqlens: Optional[torch.Tensor] = None,
    seqinfo: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotate packed queries and keys by their positions, in one launch; differentiable in q and k (in reverse mode).

    q: [T, H, D] or [1, T, H, D], k: [T, H_kv, D] or [1, T, H_kv, D], or None (fp32, bf16 or fp16; D as in
    `packed_varlen_attn`).  Tokens and heads may be strided, as in views of one projection's output.
    cos, sin: fp32 [positions, rotary_dim / 2] (`rotary_table`).  The first rotary_dim <= D dims of a head
    rotate, in pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) with `interleaved`; the others pass through.
    A token's position is its place in its segment of cu_seqlens ([n_seg + 1]; or seqinfo: [n_seg] lengths), or
    positions[t] where those are given ([T], any integer type).

    Returns (q, k) rotated, contiguous, with the ranks of the inputs.  Rows behind the last segment, which
    only unchecked calls can have, come out as zeros; a position outside the table gives NaN there.
    A step with its gradients can be captured into a CUDA graph once validation is off; as with every operator, torch wants no
    eager autograd graph of the same leaves to be alive meanwhile (its AccumulateGrad nodes belong to the eager stream).
    """
    _no_tangent("packed_rotary", q, k, cos, sin)
    if seqinfo is not None and cu_seqlens is None and positions is None:
        cu_seqlens, seqinfo = _lengths_to_cu(seqinfo), None
    key = ("packed_rotary", _layout(q), _layout(k), _layout(cos), _layout(sin), _layout(cu_seqlens), _layout(positions), seqinfo is None, interleaved)
    plan = _plans.get(key)
    given = cu_seqlens if positions is None else positions  # (before it is taken to 32 bits)
    q4 = k4 = False
    if plan is None:
        q, q4 = _rows(q, "q")
        k, k4 = (None, False) if k is None else _rows(k, "k")
        _check_heads(q, "q")
        if k is not None:
            _like(k, q, "k")
            _need(k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2], lambda: f"K shape mismatch: {tuple(k.shape)} vs q {tuple(q.shape)}")
        _check_angles(cos, sin, q)
        if (cu_seqlens is not None) + (seqinfo is not None) + (positions is not None) != 1:
            raise ValueError("must provide one of cu_seqlens, seqinfo and positions")
        if positions is None:
            cu_seqlens = _ints(cu_seqlens, q.device, "cu_seqlens")
            if cu_seqlens.numel() < 2:
                raise ValueError("cu_seqlens: must have at least 2 elements (n_seg+1 with n_seg>=1)")
        else:
            positions = _ints(positions, q.device, "positions")
            _need(positions.shape[0] == q.shape[0], lambda: f"positions has {positions.shape[0]} entries for {q.shape[0]} tokens")
        plan = _rotary_plan(q, k, cos, positions, cu_seqlens, bool(interleaved), False)
        # (a plan is for tensors as they came: none that was converted, copied or has a fourth dim)
        if key[1:7] == (_layout(q), _layout(k), _layout(cos), _layout(sin), _layout(cu_seqlens), _layout(positions)):
            _keep(key, plan)
    T = q.shape[0]
    if _varlen._validate and T > 0:
        host = _host(given)
        if positions is None:
            _check_cu(host, T, "cu_seqlens")
            low, high = 0, int((host[1:] - host[:-1]).max()) - 1
        else:
            low, high = int(host.min()), int(host.max())
        if low < 0 or high >= cos.shape[0]:
            raise ValueError(f"positions {low} to {high} leave the table of {cos.shape[0]}")
    if torch.is_grad_enabled() and (q.requires_grad or cos.requires_grad or sin.requires_grad or (k is not None and k.requires_grad)):
        _need(not (cos.requires_grad or sin.requires_grad), lambda: "cos/sin have no gradient here")
        qo, ko = _PackedRotary.apply(q, k, cos, sin, positions, cu_seqlens, plan, bool(interleaved), False)
    else:
        qo, ko = _rotate(plan, q, k, cos, sin, positions, cu_seqlens)
    return (qo.unsqueeze(0) if q4 else qo), (ko.unsqueeze(0) if k4 else ko)


# ------------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------------
def _check_append(lens, table, cu, T, num_pages, page_size, angles) -> None:
    """Host copies of an append's lengths and pages: what it would write is in the cache, and nothing twice."""
    _check_pages(lens, table, num_pages, page_size)
    if cu is None:
        new = torch.ones_like(lens)
    else:
        _check_cu(cu, T, "cu_seqlens")
        new = cu[1:] - cu[:-1]
    new = torch.where(lens == 0, torch.zeros_like(new), new)  # padding
    if bool((new > lens).any()):
        raise ValueError("cache_seqlens must count the new tokens of a sequence among its tokens")
    seq = torch.repeat_interleave(torch.arange(lens.numel()), new)
    pos = torch.arange(seq.numel()) - (new.cumsum(0) - new)[seq] + (lens - new)[seq]
    if angles is not None and pos.numel() and int(pos.max()) >= angles:
        raise ValueError(f"position {int(pos.max())} leaves the table of {angles}")
    slot = table[seq, pos // page_size] * page_size + pos % page_size
    if slot.unique().numel() != slot.numel():
        raise ValueError("page_table gives two new tokens the same slot")


def paged_kv_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    page_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    seqinfo: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    cos: Optional[torch.Tensor] = None,
    sin: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> Optional[torch.Tensor]:
    """Write new keys and values into a paged cache, in place, rotating keys (and queries) on the way.

    k, v: [T, H_kv, D] or [1, T, H_kv, D], the new tokens of all sequences; tokens and heads may be strided.
    k_cache, v_cache: [num_pages, page_size, H_kv, D] (see the module).  page_table: [n_seq, max_pages].
    cache_seqlens: [n_seq], tokens of each sequence with the new ones among them: new token i of the n_s of sequence
    s goes to position cache_seqlens[s] - n_s + i.  cu_seqlens ([n_seq + 1]; or seqinfo: [n_seq]) cuts the new tokens
    by sequence; without it there is one for each (T = n_seq).  Sequences of length 0 are padding: their tokens
    are passed over, as are rows behind the last sequence, and so are tokens of unchecked calls whose position or page is out of range.
    cos, sin: rotate the keys by their positions as `packed_rotary` does; q ([T, H, D]) is rotated beside them.
    Without cos and sin keys are written as they are (rotated already).

    Sequences may share pages that are only read (a common prefix); what is written must be theirs alone.
    Returns the rotated q (contiguous; zeros for padding), or None without q.  Has no gradient.
    """
    _no_tangent("paged_kv_append", k, v, q, k_cache, v_cache, cos, sin)
    if seqinfo is not None and cu_seqlens is None:
        cu_seqlens = _lengths_to_cu(seqinfo)
    tensors = (k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens, q, cos, sin)
    key = ("paged_kv_append", *map(_layout, tensors), interleaved)
    plan = _plans.get(key)
    given = cache_seqlens, page_table, cu_seqlens  # (before they are taken to 32 bits)
    q4 = False
    if plan is None:
        k, _ = _rows(k, "k")
        v, _ = _rows(v, "v")
        _check_heads(k, "k")
        _like(v, k, "v")
        _need(v.shape == k.shape, lambda: f"V shape mismatch: {tuple(v.shape)} vs K {tuple(k.shape)}")
        T, H_kv, D = k.shape
        dev = k.device
        cache_seqlens = _ints(cache_seqlens, dev, "cache_seqlens")
        page_table = _ints(page_table, dev, "page_table", 2)
        _check_cache(k_cache, v_cache, page_table, cache_seqlens, k)
        num_pages, page_size = k_cache.shape[:2]
        _need(k_cache.shape[2] == H_kv, lambda: f"caches have {k_cache.shape[2]} heads, k {H_kv}")
        for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            _need(all(st > 0 or n == 1 for st, n in zip(c.stride(), c.shape)), lambda: f"{name}: an expanded tensor cannot be written to")
        n_seq = cache_seqlens.shape[0]
        if cu_seqlens is not None:
            cu_seqlens = _ints(cu_seqlens, dev, "cu_seqlens")
            _need(cu_seqlens.shape[0] == n_seq + 1, lambda: f"cu_seqlens has {cu_seqlens.shape[0] - 1} sequences, cache_seqlens {n_seq}")
        else:
            _need(T == n_seq, lambda: f"{T} new tokens for {n_seq} sequences need cu_seqlens or seqinfo")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin go together")
        R = rows = 0
        if cos is not None:
            R, rows = _check_angles(cos, sin, k), cos.shape[0]
        if q is not None:
            if cos is None:
                raise ValueError("q is rotated by cos and sin: without them it has nothing to do here")
            q, q4 = _rows(q, "q")
            _like(q, k, "q")
            _need(q.shape[0] == T and q.shape[2] == D, lambda: f"q shape mismatch: {tuple(q.shape)} vs K {tuple(k.shape)}")
            _need(q.shape[1] > 0, lambda: "q has no heads")
        a = _lib.PagedAppendArgs(
            *[None] * 11, *((0, 0) if q is None else q.stride()[:2]), *k.stride()[:2], *v.stride()[:2], *k_cache.stride()[:3],
            *v_cache.stride()[:3], page_table.stride(0), n_seq, T, 0 if q is None else q.shape[1], H_kv, D, R, rows, num_pages, page_size,
            page_table.shape[1], _lib.DTYPE_CODE[k.dtype], bool(interleaved))
        plan = _Plan(a, dev, "vafa_paged_append", out=(T, n_seq))
        if key[1:11] == tuple(map(_layout, (k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens, q, cos, sin))):
            _keep(key, plan)
    if torch.is_grad_enabled():
        _no_gradient("paged_kv_append", k, v, q, k_cache, v_cache, cos, sin)
    kc, vc = k_cache.data_ptr(), v_cache.data_ptr()
    _need(kc != vc, lambda: "k_cache and v_cache are the same memory")
    T, n_seq = plan.out
    qo = None if q is None else torch.empty_like(q, memory_format=_PACKED)
    if T > 0 and n_seq > 0:
        if _varlen._validate:
            _check_append(*(None if x is None else _host(x) for x in given), T, k_cache.shape[0], k_cache.shape[1],
                          None if cos is None else cos.shape[0])
        a = plan.args()
        a.k, a.v, a.k_cache, a.v_cache = k.data_ptr(), v.data_ptr(), kc, vc
        a.cache_seqlens, a.page_table = cache_seqlens.data_ptr(), page_table.data_ptr()
        if cu_seqlens is not None:
            a.cu_seqlens = cu_seqlens.data_ptr()
        if cos is not None:
            a.cos, a.sin = cos.data_ptr(), sin.data_ptr()
        if q is not None:
            a.q, a.q_out = q.data_ptr(), qo.data_ptr()
        plan.run(a, "vafa_paged_append")
        # autograd is told, as by every operation in place (tensors of inference mode have no version)
        told = [c for c in (k_cache, v_cache) if not c.is_inference()]
        if told:
            torch.autograd.graph.increment_version(told)
    elif qo is not None:
        qo.zero_()
    return qo.unsqueeze(0) if q4 else qo


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def _decode(q, k_cache, v_cache, page_table, cache_seqlens, scale, with_lse):
    _no_tangent("paged_decode_attn", q, k_cache, v_cache)
    tensors = (q, k_cache, v_cache, page_table, cache_seqlens)
    key = ("paged_decode_attn", *map(_layout, tensors), scale)
    plan = _plans.get(key)
    given = cache_seqlens, page_table  # (before they are taken to 32 bits)
    if plan is None:
        if q.dim() not in (3, 4):
            raise ValueError(f"q: expected [n_seq,H,D] or [n_seq,T,H,D], got {q.dim()}-D")
        _check_heads(_counts(q, "q"), "q")
        dev = q.device
        cache_seqlens = _ints(cache_seqlens, dev, "cache_seqlens")
        page_table = _ints(page_table, dev, "page_table", 2)
        _check_cache(k_cache, v_cache, page_table, cache_seqlens, q)
        n_seq, H, D = q.shape[0], q.shape[-2], q.shape[-1]
        T = q.shape[1] if q.dim() == 4 else 1
        num_pages, page_size, H_kv = k_cache.shape[:3]
        _need(n_seq == cache_seqlens.shape[0], lambda: f"q has {n_seq} sequences, cache_seqlens {cache_seqlens.shape[0]}")
        _need(H % H_kv == 0, lambda: f"{H_kv} cache heads do not divide {H} query heads")
        es = q.element_size()
        for c, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            if any(n > 1 and st * es % 16 for st, n in zip(c.stride()[:3], c.shape)):
                raise ValueError(f"{name}: base and strides must be multiples of 16 bytes")
        if q.stride(-1) != 1 or any(n > 1 and st * es % 16 for st, n in zip(q.stride()[:-1], q.shape)):
            q = q.clone(memory_format=torch.contiguous_format)
        st = q.stride()
        a = _lib.PagedAttnArgs(
            *[None] * 7, st[0], st[1] if q.dim() == 4 else 0, st[-2], *k_cache.stride()[:3], *v_cache.stride()[:3], page_table.stride(0),
            n_seq, T, H, H_kv, D, num_pages, page_size, page_table.shape[1], _lib.DTYPE_CODE[q.dtype],
            1.0 / math.sqrt(D) if scale is None else scale, _lib.sm_count(dev))
        plan = _Plan(a, dev, "vafa_paged_decode", workspace=_lib.load().vafa_paged_decode_workspace_bytes(a) if q.numel() else 0,
                     out=(tuple(q.shape[:-1]), q.numel()))
        if key[1:6] == tuple(map(_layout, (q, k_cache, v_cache, page_table, cache_seqlens))):
            _keep(key, plan)
    if torch.is_grad_enabled():
        _no_gradient("paged_decode_attn", q, k_cache, v_cache)
    kc, vc, qp = k_cache.data_ptr(), v_cache.data_ptr(), q.data_ptr()
    if (kc | vc) & 15:
        raise ValueError("k_cache, v_cache: base and strides must be multiples of 16 bytes")
    if qp & 15:
        return _decode(q.clone(), k_cache, v_cache, *reversed(given), scale, with_lse)
    o = torch.empty_like(q, memory_format=_PACKED)
    lse = torch.empty(plan.out[0], dtype=torch.float32, device=plan.device) if with_lse else None
    if plan.out[1] == 0:
        return o, lse
    if _varlen._validate:
        _check_pages(*map(_host, given), k_cache.shape[0], k_cache.shape[1])
    a = plan.args()
    a.q, a.k_cache, a.v_cache, a.o = qp, kc, vc, o.data_ptr()
    a.cache_seqlens, a.page_table = cache_seqlens.data_ptr(), page_table.data_ptr()
    if lse is not None:
        a.lse = lse.data_ptr()
    ws = torch.empty(plan.workspace, dtype=torch.uint8, device=plan.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), plan.workspace
    plan.run(a, "vafa_paged_decode")
    return o, lse


def paged_decode_attn(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    *,
    page_table: torch.Tensor,
    cache_seqlens: torch.Tensor,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Attention of the newest tokens of each sequence over its paged keys and values.

    q: [n_seq, H, D], one new token for each sequence, or [n_seq, T, H, D], T of them (fp32, bf16 or fp16; D
    as in `packed_varlen_attn`).  k_cache, v_cache: [num_pages, page_size, H_kv, D], H_kv dividing H, bases and strides
    multiples of 16 bytes.  page_table: [n_seq, max_pages].  cache_seqlens: [n_seq], the new tokens among them: token t of sequence s sees the keys
    j <= cache_seqlens[s] - T + t.  scale defaults to 1/sqrt(D).

    Returns o with the layout of q.  A row that sees no key (a sequence of length 0, or shorter than T) yields
    zeros.  The keys of all sequences are cut into equal pieces over the SMs whatever their lengths, and the parts
    joined in a fixed order: the same call gives the same bits, another batch around a sequence may round
    differently.  Meant for few new tokens; a prompt's own attention is `packed_varlen_attn`.  Has no gradient.
    """
    return _decode(q, k_cache, v_cache, page_table, cache_seqlens, None if scale is None else float(scale), False)[0]


def paged_decode_attn_with_lse(q, k_cache, v_cache, *, page_table, cache_seqlens, scale=None):
    """As paged_decode_attn, and also returns the natural-log LSE (fp32, q's shape without D; -inf for rows that see no key),
    with which parts of an attention can be joined."""
    return _decode(q, k_cache, v_cache, page_table, cache_seqlens, None if scale is None else float(scale), True)
