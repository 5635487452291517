"""Paged-cache operators on a B200 at sizes where their kernels share out work in other ways: plans of several
blocks, tokens that share a block, rotary positions of long tensors."""
import numpy as np
import pytest
import torch

import cuda_fused_attention_b200 as fa
from paged_reference import Requests, normal

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
