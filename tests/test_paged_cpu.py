"""Rotation, paged append and paged decode without a GPU: what the C ABI refuses, the struct layouts, the checks of host
copies, the table of angles."""
import ctypes as C
import math

import pytest
import torch

import varlenabsorbflashattn_b200 as vb
from varlenabsorbflashattn_b200 import _lib, build, paged


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


FAKE = 1 << 20  # an address that no check follows


def test_struct_sizes_match_header():
    assert C.sizeof(_lib.RotaryArgs) == 8 * 8 + 4 * 8 + 10 * 4 + 8
    assert C.sizeof(_lib.PagedAppendArgs) == 11 * 8 + 13 * 8 + 12 * 4 + 8
    assert C.sizeof(_lib.PagedAttnArgs) == 7 * 8 + 10 * 8 + 9 * 4 + 4 + 4 + 4 + 3 * 8


def _rotary(**kw):
    a = dict(q=FAKE, q_out=FAKE, cos=FAKE, sin=FAKE, cu_seqlens=FAKE, n_seg=1, total=4, num_heads=2, head_dim=64, rotary_dim=64,
             table_rows=8, dtype=1)
    a.update(kw)
    return _lib.RotaryArgs(**a)


@pytest.mark.parametrize("bad,code,word", [
    (dict(dtype=7), -1, "dtype"), (dict(head_dim=48), -2, "head_dim"), (dict(rotary_dim=63), -1, "rotary_dim"),
    (dict(rotary_dim=66), -1, "rotary_dim"), (dict(rotary_dim=0), -1, "rotary_dim"), (dict(cos=None), -1, "cos"),
    (dict(cu_seqlens=None), -1, "positions"), (dict(n_seg=0), -1, "positions"), (dict(q_out=None), -1, "null"), (dict(total=-1), -1, "sizes"),
    (dict(num_kv_heads=1), -1, "null"), (dict(cos=FAKE + 2), -1, "aligned")])
def test_rotary_refusals(lib, bad, code, word):
    assert lib.vafa_rotary(_rotary(**bad), None) == code
    assert word in _lib.last_error()


def _append(**kw):
    a = dict(k=FAKE, v=FAKE, k_cache=FAKE, v_cache=FAKE, cache_seqlens=FAKE, page_table=FAKE, n_seq=2, total=2, num_kv_heads=2, head_dim=64,
             num_pages=4, page_size=16, max_pages=2, dtype=1)
    a.update(kw)
    return _lib.PagedAppendArgs(**a)


@pytest.mark.parametrize("bad,code,word", [
    (dict(dtype=-1), -1, "dtype"), (dict(head_dim=80), -2, "head_dim"), (dict(cos=FAKE), -1, "cos"), (dict(q=FAKE, num_heads=2), -1, "q without"),
    (dict(cos=FAKE, sin=FAKE, rotary_dim=3), -1, "rotary_dim"), (dict(page_size=0), -1, "page_size"), (dict(num_pages=0), -1, "num_pages"),
    (dict(page_table=None), -1, "page_table"), (dict(k_cache=None), -1, "cache"), (dict(total=3), -1, "n_seq"), (dict(num_kv_heads=0), -1, "sizes"),
    (dict(max_pages=1 << 20, page_size=1 << 12), -1, "int32"), (dict(v=None), -1, "null")])
def test_append_refusals(lib, bad, code, word):
    assert lib.vafa_paged_append(_append(**bad), None) == code
    assert word in _lib.last_error()


def _attn(**kw):
    a = dict(q=FAKE, k_cache=FAKE, v_cache=FAKE, o=FAKE, cache_seqlens=FAKE, page_table=FAKE, n_seq=2, q_len=1, num_heads=8, num_kv_heads=2,
             head_dim=64, num_pages=4, page_size=16, max_pages=8, dtype=1, scale=1.0, sm_count=148, workspace=FAKE, workspace_bytes=1 << 30)
    a.update(kw)
    return _lib.PagedAttnArgs(**a)


@pytest.mark.parametrize("bad,code,word", [
    (dict(dtype=3), -1, "dtype"), (dict(head_dim=512), -2, "head_dim"), (dict(num_kv_heads=3), -1, "divide"), (dict(q_len=0), -1, "q_len"),
    (dict(n_seq=0), -1, "n_seq"), (dict(q=None), -1, "null"), (dict(workspace=None), -3, "workspace"), (dict(workspace_bytes=16), -3, "workspace"),
    (dict(workspace=FAKE + 16), -3, "aligned"), (dict(k_cache=FAKE + 8), -1, "16-byte"), (dict(k_slot_stride=4), -1, "16-byte"),
    (dict(q_len=1 << 18), -2, "q_len"), (dict(max_pages=1 << 20, page_size=1 << 12), -1, "int32")])
def test_decode_refusals(lib, bad, code, word):
    assert lib.vafa_paged_decode(_attn(**bad), None) == code
    assert word in _lib.last_error()


def test_decode_workspace_is_a_function_of_sizes_and_sms(lib):
    size = lambda **kw: lib.vafa_paged_decode_workspace_bytes(_attn(**kw))  # noqa: E731
    assert size() > 0 and size(dtype=9) == 0
    assert size(n_seq=512) >= size()
    assert size(n_seq=512, max_pages=4096) == size(n_seq=512, max_pages=8192), "bounded by the SMs, not by the batch"
    assert size(n_seq=512, max_pages=4096, sm_count=74) < size(n_seq=512, max_pages=4096)


def test_null_args(lib):
    assert lib.vafa_rotary(None, None) == lib.vafa_paged_append(None, None) == lib.vafa_paged_decode(None, None) == -1


def test_cpu_tensors_refused():
    x, c = torch.zeros(3, 2, 16), torch.zeros(4, 8)
    cache, table, lens = torch.zeros(2, 4, 2, 16), torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        vb.packed_rotary(x, None, c, c, cu_seqlens=torch.tensor([0, 3]))
    with pytest.raises(AssertionError, match="CUDA"):
        vb.paged_kv_append(x, x, cache, cache, page_table=table, cache_seqlens=lens)
    with pytest.raises(AssertionError, match="CUDA"):
        vb.paged_decode_attn(x, cache, cache, page_table=table, cache_seqlens=lens)
    with pytest.raises(ValueError, match="3-D"):
        vb.packed_rotary(x[0], None, c, c, cu_seqlens=torch.tensor([0, 3]))
    with pytest.raises(ValueError, match="n_seq,H,D"):
        vb.paged_decode_attn(x[0], cache, cache, page_table=table, cache_seqlens=lens)


def test_integer_arguments():
    dev = torch.device("cpu")
    assert paged._ints(torch.tensor([1, 2]), dev, "x").dtype == torch.int32
    for bad in (torch.tensor([1.0]), torch.tensor([True]), torch.zeros(1, 1, dtype=torch.int32)):
        with pytest.raises(ValueError):
            paged._ints(bad, dev, "x")


def test_sizes_beyond_32_bits():
    # 2^32 + 1 rows would arrive in the library as one
    many = 2**32 + 1
    for x in (torch.zeros(1, 1, 64).expand(many, 1, 64), torch.zeros(1, 1, 64).expand(1, many, 64)):
        with pytest.raises(ValueError, match="int32 range"):
            paged._rows(x, "q")
        with pytest.raises(ValueError, match="int32 range"):
            vb.paged_decode_attn(x, x, x, page_table=torch.zeros(1, 1), cache_seqlens=torch.zeros(1))
    with pytest.raises(ValueError, match="int32 range"):
        paged._ints(torch.zeros(1, dtype=torch.int64).expand(many), torch.device("cpu"), "cache_seqlens")
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for cache in (torch.zeros(1, 16, 1, 64).expand(many, 16, 1, 64), torch.zeros(1, 16, 1, 64).expand(1, 16, many, 64)):
        with pytest.raises(ValueError, match="int32 range"):
            paged._check_cache(cache, cache, table, lens, torch.zeros(1, 1, 64))
    assert paged._counts(torch.zeros(0), "q").numel() == 0 and paged._counts(torch.zeros(()), "q").dim() == 0


def test_check_pages():
    table = torch.tensor([[0, 1, 99], [2, -7, 3]])
    paged._check_pages(torch.tensor([8, 4]), table, 4, 4)  # what lies behind the length is nobody's
    with pytest.raises(ValueError, match="outside"):
        paged._check_pages(torch.tensor([9, 4]), table, 4, 4)
    with pytest.raises(ValueError, match="outside"):
        paged._check_pages(torch.tensor([8, 5]), table, 4, 4)
    with pytest.raises(ValueError, match="cache_seqlens"):
        paged._check_pages(torch.tensor([13, 4]), table, 200, 4)
    with pytest.raises(ValueError, match="cache_seqlens"):
        paged._check_pages(torch.tensor([-1, 4]), table, 4, 4)
    paged._check_pages(torch.zeros(2, dtype=torch.int64), table, 4, 4)


def test_check_append():
    table, lens = torch.tensor([[0, 1], [2, 3]]), torch.tensor([5, 2])
    paged._check_append(lens, table, None, 2, 4, 4, 8)
    paged._check_append(lens, table, torch.tensor([0, 5, 6]), 6, 4, 4, 8)
    paged._check_append(torch.tensor([5, 0]), table, torch.tensor([0, 5, 9]), 9, 4, 4, 8)  # the second sequence is padding
    with pytest.raises(ValueError, match="same slot"):
        paged._check_append(lens, torch.tensor([[0, 1], [1, 3]]), torch.tensor([0, 2, 4]), 4, 4, 4, 8)
    paged._check_append(lens, torch.tensor([[1, 0], [1, 3]]), None, 2, 4, 4, 8)  # shared for reading only
    with pytest.raises(ValueError, match="among its tokens"):
        paged._check_append(lens, table, torch.tensor([0, 5, 8]), 8, 4, 4, 8)
    with pytest.raises(ValueError, match="table of 4"):
        paged._check_append(lens, table, None, 2, 4, 4, 4)
    paged._check_append(lens, table, None, 2, 4, 4, None)
    with pytest.raises(ValueError, match="total tokens"):
        paged._check_append(lens, table, torch.tensor([0, 5, 6]), 7, 4, 4, 8)


def test_rotary_table():
    cos, sin = vb.rotary_table(1 << 17, 6, base=500.0)
    assert cos.shape == sin.shape == (1 << 17, 3) and cos.dtype == torch.float32
    for p in (0, 1, 1000, (1 << 17) - 1):
        for i in range(3):
            a = p * 500.0 ** (-2 * i / 6)
            # the angle in 64 bits is off by 2^-52 of up to 2^17, far below half a step of fp32 at 1
            assert abs(cos[p, i].item() - math.cos(a)) <= 2.0 ** -25 + 2.0 ** -34
            assert abs(sin[p, i].item() - math.sin(a)) <= 2.0 ** -25 + 2.0 ** -34
    for bad in ((8, 5), (8, 0), (-1, 4)):
        with pytest.raises(ValueError):
            vb.rotary_table(*bad)
