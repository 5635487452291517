"""Paged-cache operators on a B200 at sizes where their kernels share out work in other ways: plans of several
blocks, tokens that share a block, rotary positions of long tensors."""
import numpy as np
import pytest
import torch

import cuda_fused_attention_b200 as fa
from paged_reference import Requests, normal, rotary

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    fa.device_status()
    yield
    torch.cuda.synchronize()


def status_ok():
    assert fa.device_status() == (fa.STATUS_OK, 0)


def _freq(pairs):
    return (10000.0 ** (-torch.arange(pairs, dtype=torch.float32, device="cuda") / pairs)).contiguous()


@pytest.mark.parametrize("dim,new", [(64, [1] * 40 + [4200]), (128, [1, 3, 2500, 1, 2200, 7] + [1] * 30)])
def test_steps_whose_plan_has_several_blocks(cuda_device, dim, new):
    """Plans of several blocks, other pages in every step, and the calls that read them, launched without a wait between:
    the same bits as with a synchronisation behind each call."""
    heads, kv_heads, page_size = 8, 2, 16
    cached = [(97 * b) % 700 for b in range(len(new))]
    r = Requests(cached, new, page_size, cuda_device, seed=7, padding=3)
    assert r.total > 4096
    shape = fa.PagedShape(heads, kv_heads, dim, page_size)
    start = r.block_table.clone()
    # Three namings of the pages: the table's and the free list's ids go through a permutation.
    namings = [torch.from_numpy(np.random.RandomState(s).permutation(r.num_pages).astype(np.int32)).cuda() for s in range(3)]
    tables = [torch.where(start >= 0, n[start.clamp(min=0).long()], start) for n in namings]
    frees = [n[r.free_pages.long()] for n in namings]
    caches = [normal(s, r.num_pages, kv_heads, page_size, dim) for s in (1, 2)]
    held = [c.clone() for c in caches]
    qkv = normal(3, r.total, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    freq, tokens, table = _freq(dim // 2), sum(new), torch.empty_like(start)

    def step(i, wait):
        table.copy_(tables[i])
        for c, h in zip(caches, held):
            c.copy_(h)
        wait()
        plan = fa.paged_plan(r.cached_lens, r.new_lens, table, frees[i], r.total, shape, r.num_pages)
        wait()
        turned = fa.rotary_append(q, k, v, *caches, plan.positions, plan.slots, freq)
        wait()
        one = fa.paged_attention(turned, *caches, plan)
        wait()
        # Again without the append in between: attention behind the plan itself.
        plan = fa.paged_plan(r.cached_lens, r.new_lens, table, frees[i], r.total, shape, r.num_pages)
        wait()
        return one[:tokens], fa.paged_attention(turned, *caches, plan)[:tokens], table.clone()

    want = [step(i, torch.cuda.synchronize) for i in range(3)]
    assert not torch.equal(want[0][2], want[1][2])
    torch.cuda.synchronize()
    for i in range(12):
        for got, expected in zip(step(i % 3, lambda: None), want[i % 3]):
            assert torch.equal(got, expected)
    status_ok()


# ---------------------------------------------------------------------------
# Rotary positions of long tensors: threads keep a token's angles and walk over heads
# ---------------------------------------------------------------------------
def _sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _long_tokens(dim):
    """Tokens of all batches from which rotary_embed shares heads out: 512 units of 16 elements of a head per SM."""
    return 512 * _sms() * 16 // dim


def _positions(axes, tokens, batch=None):
    gen = torch.Generator().manual_seed(axes * 1000 + tokens)
    shape = (axes, tokens) if batch is None else (axes, batch, tokens)
    return torch.randint(-300, 200000, shape, generator=gen).to(torch.int32).cuda()


ROTARY_FORMS = [(64, 64, (32,)), (64, 48, (5, 0, 19)), (128, 128, (16, 24, 24)), (128, 96, (1, 2, 5, 40)), (128, 16, (8,))]


@pytest.mark.parametrize("dim,rotary_dim,sections", ROTARY_FORMS)
@pytest.mark.parametrize("interleaved,inverse", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("batch,heads,off", [(1, 6, 0), (1, 1, 1), (2, 5, 0), (2, 3, -1), (3, 7, 500)])
def test_rotary_of_long_tensors(cuda_device, dim, rotary_dim, sections, interleaved, inverse, batch, heads, off):
    """On both sides of the border between the kernels; heads that do not divide evenly among the threads."""
    tokens = -(-_long_tokens(dim) // batch) + off
    x = normal(1, batch, heads, tokens, dim)
    freq = _freq(rotary_dim // 2)
    for positions in (_positions(len(sections), tokens), _positions(len(sections), tokens, batch)):
        got = fa.rotary_embed(x, positions, freq, sections, interleaved, inverse)
        for b in range(batch):
            pos = positions if positions.dim() == 2 else positions[:, b]
            want, bound = rotary(x[b].transpose(0, 1), pos, freq, sections, interleaved, inverse)
            assert ((got[b].transpose(0, 1).double() - want).abs() <= bound).all()
        # A short piece of it goes through the other kernel: the same bits.
        at = slice(tokens - 77, tokens)
        piece = fa.rotary_embed(x[:, :, at], positions[..., at], freq, sections, interleaved, inverse)
        assert torch.equal(piece, got[:, :, at])
    status_ok()


@pytest.mark.parametrize("dim,rotary_dim,sections", ROTARY_FORMS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_of_long_tensors_strides_and_in_place(cuda_device, dim, rotary_dim, sections, interleaved):
    batch, heads = 2, 3
    tokens = _long_tokens(dim) // batch + 13
    x = normal(2, batch, heads, tokens, dim)
    freq, positions = _freq(rotary_dim // 2), _positions(len(sections), tokens, batch)
    want = fa.rotary_embed(x, positions, freq, sections, interleaved)
    fused = normal(3, batch, tokens, 3, heads, dim)
    fused[:, :, 1] = x.transpose(1, 2)
    view = fused[:, :, 1].transpose(1, 2)
    assert torch.equal(fa.rotary_embed(view, positions, freq, sections, interleaved), want)
    kept = fused.clone()
    assert fa.rotary_embed(view, positions, freq, sections, interleaved, out=view) is view
    assert torch.equal(view, want)
    assert torch.equal(fused[:, :, 0], kept[:, :, 0]) and torch.equal(fused[:, :, 2], kept[:, :, 2])
    out = torch.zeros(tokens, batch, heads, dim, dtype=torch.bfloat16, device=cuda_device).permute(1, 2, 0, 3)
    assert torch.equal(fa.rotary_embed(x, positions, freq, sections, interleaved, out=out), want)
    mine = x.clone()
    assert torch.equal(fa.rotary_embed(mine, positions, freq, sections, interleaved, out=mine), want)


# ---------------------------------------------------------------------------
# Append of many tokens: two, then four of them share a block
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("per_sm,off", [(8, -1), (8, 0), (8, 1), (16, -1), (16, 0), (16, 1), (16, 3), (40, 2)])
@pytest.mark.parametrize("heads,kv_heads,dim,page_size,sections,interleaved", [
    (8, 2, 128, 16, (64,), False), (5, 5, 64, 32, (8, 12, 12), True), (7, 1, 128, 256, (3, 29), False)])
def test_append_of_many_tokens(cuda_device, per_sm, off, heads, kv_heads, dim, page_size, sections, interleaved):
    """Slots in any order, some of them negative and some outside the cache, in every place of a shared block."""
    tokens = per_sm * _sms() + off
    pages = -(-(tokens + 50) // page_size)
    rng = np.random.RandomState(tokens + dim)
    slots = rng.permutation(pages * page_size)[:tokens].astype(np.int64)
    skipped = np.zeros(tokens, bool)
    for i, value in enumerate([-1, -2 ** 31, pages * page_size, 2 ** 31 - 1]):
        at = rng.permutation(tokens)[: tokens // 25] if i < 2 else rng.permutation(tokens)[:3]
        slots[at], skipped[at] = value, True
    slots[-2:], skipped[-2:] = -1, True       # the last, part-filled block ends in padding
    qkv = normal(6, tokens, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    k_cache, v_cache = normal(7, pages, kv_heads, page_size, dim), normal(8, pages, kv_heads, page_size, dim)
    k_held, v_held = k_cache.clone(), v_cache.clone()
    freq, positions = _freq(sum(sections)), _positions(len(sections), tokens)
    out = torch.full((tokens, heads, dim), 9.0, dtype=torch.bfloat16, device=cuda_device)
    ids = torch.from_numpy(slots.astype(np.int32)).cuda()
    fa.rotary_append(q, k, v, k_cache, v_cache, positions, ids, freq, sections, interleaved, out=out)
    assert fa.device_status() == (fa.STATUS_BAD_REQUEST, 0x40000)
    done = torch.from_numpy(~skipped).cuda()
    want, bound = rotary(q, positions, freq, sections, interleaved)
    assert ((out.double() - want).abs() <= bound)[done].all() and (out[~done] == 9.0).all()
    page, row = ids[done].long() // page_size, ids[done].long() % page_size
    want, bound = rotary(k, positions, freq, sections, interleaved)
    assert ((k_cache[page, :, row].double() - want[done]).abs() <= bound[done]).all()
    assert torch.equal(v_cache[page, :, row], v[done])
    k_held[page, :, row], v_held[page, :, row] = k_cache[page, :, row], v_cache[page, :, row]
    assert torch.equal(k_cache, k_held) and torch.equal(v_cache, v_held)      # nothing else was written
    # Twenty tokens alone do not share blocks: the same bits. In place too.
    some = torch.from_numpy(np.flatnonzero(~skipped)[-20:]).cuda()
    k2, v2 = torch.zeros_like(k_cache), torch.zeros_like(v_cache)
    few = fa.rotary_append(q[some], k[some], v[some], k2, v2, positions[:, some].contiguous(), ids[some], freq, sections, interleaved)
    assert torch.equal(few, out[some])
    at = ids[some].long()
    assert torch.equal(k2[at // page_size, :, at % page_size], k_cache[at // page_size, :, at % page_size])
    packed = qkv.clone()
    fa.rotary_append(packed[:, :heads], k, v, k2, v2, positions, ids, freq, sections, interleaved, out=packed[:, :heads])
    assert torch.equal(packed[:, :heads][done], out[done]) and torch.equal(packed[~done], qkv[~done])
    assert torch.equal(packed[:, heads:], qkv[:, heads:])
    assert fa.device_status() == (fa.STATUS_BAD_REQUEST, 0x40000)
