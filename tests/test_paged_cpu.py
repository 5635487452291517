"""Refusals of the paged-cache operators, made on the host before any CUDA call."""
import ctypes

import pytest
import torch

import cuda_fused_attention_b200 as fa
from cuda_fused_attention_b200 import _lib
from paged_reference import FaPagedPlan


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def _plan(**changes):
    plan = FaPagedPlan()
    values = dict(num_seqs=2, total_tokens=4, max_new=4, num_pages=8, table_width=4, table_stride=4, heads=8, kv_heads=2,
                  head_dim=128, page_size=16, causal=1, query_start=0x1000, kv_lens=0x1000, positions=0x1000,
                  slots=0x1000, block_table=0x1000, free_cursor=0x1000, schedule=0x1000)
    for name, value in {**values, **changes}.items():
        setattr(plan, name, value)
    return plan


BAD_PLANS = [
    (dict(head_dim=96), 1002), (dict(page_size=8), 1002), (dict(page_size=48), 1002), (dict(page_size=512), 1002),
    (dict(heads=7), 1001), (dict(heads=0), 1001), (dict(kv_heads=0), 1001), (dict(heads=129, kv_heads=1), 1002),
    (dict(num_seqs=-1), 1001), (dict(total_tokens=-1), 1001), (dict(max_new=-1), 1001), (dict(num_pages=-1), 1001),
    (dict(table_width=-1), 1001), (dict(table_stride=3), 1001), (dict(num_pages=2 ** 27), 1001),
    (dict(table_width=2 ** 27, table_stride=2 ** 27), 1001), (dict(query_start=None), 1001), (dict(kv_lens=None), 1001),
    (dict(positions=None), 1001), (dict(slots=None), 1001), (dict(block_table=None), 1001),
    (dict(free_cursor=None), 1001), (dict(schedule=None), 1001)]


@pytest.mark.parametrize("changes,status", BAD_PLANS, ids=lambda v: str(v))
def test_c_plan_refusals(lib, changes, status):
    plan = ctypes.byref(_plan(**changes))
    assert lib.fa_sm100_paged_plan(plan, 0x1000, 0x1000, 0x1000, 4, None, None) == status
    strides = (ctypes.c_longlong * 10)(*[128] * 10)
    assert lib.fa_sm100_paged_fwd(plan, 0x1000, 0x1000, 0x1000, 0x1000, strides, 0x1000, 1 << 40, None) == status


def test_c_refusals(lib):
    plan = ctypes.byref(_plan())
    good = (ctypes.c_longlong * 10)(*[128] * 10)
    odd = (ctypes.c_longlong * 10)(*[128] * 9, 132)
    back = (ctypes.c_longlong * 10)(*[128] * 9, -128)
    assert lib.fa_sm100_paged_plan(None, 0x1000, 0x1000, 0x1000, 4, None, None) == 1001
    assert lib.fa_sm100_paged_plan(plan, None, 0x1000, 0x1000, 4, None, None) == 1001
    assert lib.fa_sm100_paged_plan(plan, 0x1000, None, 0x1000, 4, None, None) == 1001
    assert lib.fa_sm100_paged_plan(plan, 0x1000, 0x1000, None, 4, None, None) == 1001
    assert lib.fa_sm100_paged_plan(plan, 0x1000, 0x1000, 0x1000, -1, None, None) == 1001
    fwd = lib.fa_sm100_paged_fwd
    assert fwd(None, 0x1000, 0x1000, 0x1000, 0x1000, good, None, 0, None) == 1001
    for i in range(4):
        assert fwd(plan, *[None if j == i else 0x1000 for j in range(4)], good, None, 0, None) == 1001
        assert fwd(plan, *[0x1008 if j == i else 0x1000 for j in range(4)], good, None, 0, None) == 1003
    assert fwd(plan, 0x1000, 0x1000, 0x1000, 0x1000, None, None, 0, None) == 1001
    assert fwd(plan, 0x1000, 0x1000, 0x1000, 0x1000, odd, None, 0, None) == 1003
    assert fwd(plan, 0x1000, 0x1000, 0x1000, 0x1000, back, None, 0, None) == 1001
    assert fwd(ctypes.byref(_plan(total_tokens=0)), None, None, None, None, good, None, 0, None) == 0
    assert lib.fa_sm100_paged_schedule_bytes(3) == 64 and lib.fa_sm100_paged_schedule_bytes(-1) == 0


def test_c_rotary_refusals(lib):
    three, two = (ctypes.c_longlong * 3)(*[128] * 3), (ctypes.c_longlong * 2)(8, 0)
    odd = (ctypes.c_longlong * 3)(128, 128, 68)
    sections = (ctypes.c_int * 4)(16, 24, 24, 0)

    def call(x=0x1000, xs=three, out=0x1000, batch=1, dim=128, positions=0x1000, freq=0x1000, rot=128, axes=3, sec=sections):
        return lib.fa_sm100_rotary(x, xs, out, three, batch, 2, 3, dim, positions, two, freq, rot, sec, axes, 0, 0, None)

    assert call(batch=0) == 0
    assert call(dim=80) == 1002
    for bad in (dict(x=None), dict(out=None), dict(positions=None), dict(freq=None), dict(xs=None), dict(sec=None),
                dict(batch=-1), dict(rot=130), dict(rot=24), dict(rot=0), dict(axes=0), dict(axes=5), dict(axes=2),
                dict(rot=64), dict(sec=(ctypes.c_int * 4)(-8, 48, 24, 0))):
        assert call(**bad) == 1001, bad
    assert call(x=0x1008) == 1003 and call(xs=odd) == 1003
    assert call(xs=(ctypes.c_longlong * 3)(128, -128, 128)) == 1001

    strides = (ctypes.c_longlong * 14)(*[128] * 14)

    def append(ptrs=(0x1000,) * 6, s=strides, tokens=2, heads=4, dim=128, page=16, pages=8, slots=0x1000):
        return lib.fa_sm100_rotary_append(*ptrs, s, tokens, heads, 2, dim, page, pages, 0x1000, 2, slots, 0x1000, 128,
                                          sections, 3, 0, None)

    assert append(tokens=0) == 0
    assert append(dim=32) == 1002 and append(page=24) == 1002
    for i in range(6):
        assert append(ptrs=[None if j == i else 0x1000 for j in range(6)]) == 1001
        assert append(ptrs=[0x1002 if j == i else 0x1000 for j in range(6)]) == 1003
    assert append(slots=None) == 1001 and append(s=None) == 1001 and append(tokens=-1) == 1001
    assert append(heads=0) == 1001 and append(pages=2 ** 28) == 1001 and append(pages=-1) == 1001
    assert append(s=(ctypes.c_longlong * 14)(*[128] * 13, 4)) == 1003


@pytest.mark.parametrize("args", [(8, 3, 64, 16), (0, 1, 64, 16), (8, 0, 64, 16), (129, 1, 64, 16), (8, 8, 80, 16),
                                  (8, 8, 64, 24), (8, 8, 64, 8)])
def test_shape_refusals(args):
    with pytest.raises(ValueError):
        fa.PagedShape(*args)


def test_python_refusals():
    shape = fa.PagedShape(8, 2, 64, 16)
    good = dict(cached_lens=_i32(2), new_lens=_i32(2), block_table=_i32(2, 4), free_pages=_i32(3), total_tokens=5,
                shape=shape, num_pages=9)
    for change, error in [
            (dict(cached_lens=_i32(2).long()), TypeError), (dict(cached_lens=_i32(2, 1)), ValueError),
            (dict(new_lens=_i32(3)), ValueError), (dict(new_lens=_i32(4)[::2]), ValueError),
            (dict(block_table=_i32(3, 4)), ValueError), (dict(block_table=_i32(8)), ValueError),
            (dict(block_table=_i32(4, 2).t()), ValueError), (dict(block_table=_i32(1, 4).expand(2, 4)), ValueError),
            (dict(free_pages=_i32(3).float()), TypeError), (dict(free_cursor=_i32(2)), ValueError),
            (dict(total_tokens=-1), ValueError), (dict(num_pages=-1), ValueError), (dict(max_new=-1), ValueError),
            (dict(num_pages=2 ** 28), ValueError), (dict(total_tokens=2 ** 31), ValueError), (dict(num_pages=1.5), TypeError),
            (dict(shape=(8, 2, 64)), TypeError),
            ({}, TypeError)]:        # CPU tensors: no silent CPU path
        with pytest.raises(error):
            fa.paged_plan(**{**good, **change})

    freq, positions = torch.ones(32), _i32(7)
    good = dict(x=_bf16(2, 3, 7, 64), positions=positions, inv_freq=freq)
    for change, error in [
            (dict(x=_bf16(3, 7, 64)), ValueError), (dict(x=_bf16(2, 3, 7, 32)), ValueError),
            (dict(x=torch.zeros(2, 3, 7, 64)), TypeError), (dict(x=_bf16(2, 3, 64, 64).transpose(2, 3)), ValueError),
            (dict(x=_bf16(2, 3, 7, 68)[..., :64]), ValueError), (dict(positions=_i32(8)), ValueError),
            (dict(positions=_i32(7).long()), TypeError), (dict(positions=_i32(2, 7)), ValueError),
            (dict(positions=_i32(1, 3, 7)), ValueError), (dict(positions=_i32(7, 1).t()[:, ::1].expand(1, 7)[:, :0]), ValueError),
            (dict(inv_freq=torch.ones(12)), ValueError), (dict(inv_freq=torch.ones(40)), ValueError),
            (dict(inv_freq=torch.ones(32).half()), TypeError), (dict(inv_freq=torch.ones(0)), ValueError),
            (dict(sections=(16, 15)), ValueError), (dict(sections=(16, 17)), ValueError),
            (dict(sections=(-1, 33)), ValueError), (dict(sections=()), ValueError),
            (dict(sections=(8, 8, 8, 4, 4)), ValueError), (dict(sections=3), TypeError), (dict(x=3), TypeError),
            ({}, TypeError)]:
        with pytest.raises(error):
            fa.rotary_embed(**{**good, **change})

    good = dict(q=_bf16(5, 4, 64), k=_bf16(5, 2, 64), v=_bf16(5, 2, 64), k_cache=_bf16(3, 2, 16, 64),
                v_cache=_bf16(3, 2, 16, 64), positions=_i32(5), slots=_i32(5), inv_freq=freq)
    for change, error in [
            (dict(q=_bf16(5, 4, 128)), ValueError), (dict(q=_bf16(5, 256)), ValueError), (dict(k=_bf16(4, 2, 64)), ValueError),
            (dict(v=_bf16(5, 3, 64)), ValueError), (dict(v_cache=_bf16(3, 2, 32, 64)), ValueError),
            (dict(k_cache=_bf16(3, 2, 24, 64), v_cache=_bf16(3, 2, 24, 64)), ValueError),
            (dict(k_cache=_bf16(1, 2, 16, 64).expand(3, 2, 16, 64)), ValueError), (dict(slots=_i32(4)), ValueError),
            (dict(slots=_i32(5).long()), TypeError), (dict(positions=_i32(1, 4)), ValueError),
            (dict(positions=_i32(2, 5)), ValueError), ({}, TypeError)]:
        with pytest.raises(error):
            fa.rotary_append(**{**good, **change})

    plan = fa.PagedPlan(shape, 2, 5)
    struct = _plan(total_tokens=5, num_pages=3, heads=8, kv_heads=2, head_dim=64, page_size=16)
    plan._filled((_i32(40), bytes(struct), 0, 0), _i32(2, 4), 3, True)
    good = dict(q=_bf16(5, 8, 64), k_cache=_bf16(3, 2, 16, 64), v_cache=_bf16(3, 2, 16, 64), plan=plan)
    for change, error in [
            (dict(q=_bf16(4, 8, 64)), ValueError), (dict(q=torch.zeros(5, 8, 64)), TypeError),
            (dict(k_cache=_bf16(4, 2, 16, 64)), ValueError), (dict(v_cache=_bf16(3, 2, 16, 128)), ValueError),
            (dict(v_cache=_bf16(3, 2, 16, 72)[..., 4:68]), ValueError), ({}, TypeError)]:
        with pytest.raises(error):
            fa.paged_attention(**{**good, **change})


def test_status_strings(lib):
    for code in (fa.STATUS_BAD_REQUEST, fa.STATUS_OUT_OF_PAGES, fa.STATUS_WORKSPACE):
        assert b"unknown" not in lib.fa_sm100_status_string(code)


def test_append_refuses_caches_that_share_memory(lib):
    """K and V would be written over each other."""
    q, k = _bf16(5, 4, 64), _bf16(5, 2, 64)
    rest = dict(positions=_i32(5), slots=_i32(5), inv_freq=torch.ones(32))

    def refusal(k_cache, v_cache):
        with pytest.raises((ValueError, TypeError)) as caught:
            fa.rotary_append(q, k, k, k_cache, v_cache, **rest)
        return str(caught.value)

    pages = _bf16(6, 2, 16, 64)
    rows = _bf16(6, 16, 2, 64).transpose(1, 2)
    halves, both = _bf16(6, 2, 2, 16, 64), _bf16(6, 16, 2, 2, 64).permute(0, 2, 3, 1, 4)
    wide = _bf16(6, 2, 16, 128)
    for a, b in [(pages, pages), (rows, rows), (pages[:4], pages[2:]), (pages[1:], pages[:-1]), (halves[:, 0], halves[:, 0]),
                 (both[:, 1], both[:, 1]), (halves[1:, 0], halves[:-1, 0]), (wide[..., :64], wide[..., 32:96])]:
        assert "must not share memory" in refusal(a, b) and "must not share memory" in refusal(b, a)
    for a, b in [(pages, pages.clone()), (pages[:3], pages[3:]), (halves[:, 0], halves[:, 1]), (halves[:, 1], halves[:, 0]),
                 (both[:, 0], both[:, 1]), (wide[..., :64], wide[..., 64:]), (pages[:1], pages[1:2])]:
        assert "must be a CUDA tensor" in refusal(a, b) and "must be a CUDA tensor" in refusal(b, a)

    sections = (ctypes.c_int * 1)(32)
    strides = (ctypes.c_longlong * 14)(*[64] * 14)
    assert lib.fa_sm100_rotary_append(0x1000, 0x2000, 0x2000, 0x1000, 0x3000, 0x3000, strides, 2, 4, 2, 64, 16, 8, 0x1000, 2,
                                      0x1000, 0x1000, 64, sections, 1, 0, None) == 1001


@pytest.mark.parametrize("changes", [dict(num_seqs=2 ** 30), dict(num_seqs=2 ** 31 - 1), dict(total_tokens=2 ** 30),
                                     dict(total_tokens=2 ** 31 - 1)], ids=str)
def test_c_plan_refuses_more_than_the_kernels_can_count(lib, changes):
    plan = ctypes.byref(_plan(**changes))
    strides = (ctypes.c_longlong * 10)(*[128] * 10)
    assert lib.fa_sm100_paged_plan(plan, 0x1000, 0x1000, 0x1000, 4, None, None) == 1001
    assert lib.fa_sm100_paged_fwd(plan, 0x1000, 0x1000, 0x1000, 0x1000, strides, 0x1000, 1 << 40, None) == 1001
    assert lib.fa_sm100_paged_workspace_bytes(plan) == 0


def test_plan_refuses_inputs_inside_the_table():
    """One block would read what another has written."""
    shape = fa.PagedShape(8, 2, 64, 16)
    pool = _i32(64)
    good = dict(cached_lens=_i32(2), new_lens=_i32(2), block_table=pool[16:48].view(2, 16)[:, :6], free_pages=_i32(3),
                total_tokens=5, shape=shape, num_pages=9, free_cursor=_i32(1))

    def refusal(**change):
        with pytest.raises((ValueError, TypeError)) as caught:
            fa.paged_plan(**{**good, **change})
        return str(caught.value)

    # The table's elements are 16 to 21 and 32 to 37 of the pool.
    for name, size in (("cached_lens", 2), ("new_lens", 2), ("free_pages", 9), ("free_cursor", 1)):
        for at in range(64 - size):
            inside = any(at <= e < at + size for e in (*range(16, 22), *range(32, 38)))
            text = refusal(**{name: pool[at: at + size]})
            assert (f"{name} must not share memory with block_table" in text) == inside, (name, at)
            assert inside or "must be a CUDA tensor" in text
    one = refusal(cached_lens=pool[3:4], new_lens=_i32(1), block_table=pool[:4].view(1, 4))
    assert "cached_lens must not share" in one
