"""Paged-cache operators on a B200 when something is wrong with a step: what is recorded, and that nothing
else is touched."""
import pytest
import torch

import cuda_fused_attention_b200 as fa
from paged_reference import normal

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE = 4, 2, 64, 16


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    fa.device_status()
    yield
    torch.cuda.synchronize()


def i32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _layer(plan, total, caches, seed):
    qkv = normal(seed, total, HEADS + 2 * KV_HEADS, DIM)
    q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], dim=1)
    freq = (10000.0 ** (-torch.arange(DIM // 2, dtype=torch.float32, device="cuda") / (DIM // 2))).contiguous()
    out = torch.zeros(total, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
    fa.rotary_append(q, k, v, *caches, plan.positions, plan.slots, freq, out=out)
    return fa.paged_attention(out, *caches, plan)


@pytest.mark.parametrize("new", [20, 100])
@pytest.mark.parametrize("free", [(5,), (5, 99)], ids=["list ends", "page outside the cache"])
def test_a_request_without_pages_leaves_others_alone(cuda_device, new, free):
    """Request 1 needs more pages than there are, and its table row holds ids of an earlier use, which are request 0's
    pages now. Neither this step nor the next one reads or writes them for request 1."""
    shape = fa.PagedShape(HEADS, KV_HEADS, DIM, PAGE)
    pages = 12
    table = torch.zeros(2, 10, dtype=torch.int32, device=cuda_device)
    table[0, :3] = i32(0, 1, 2)
    table[1] = i32(*[0, 1, 2] * 3, 0)       # stale
    held = [normal(s, pages, KV_HEADS, PAGE, DIM) for s in (1, 2)]

    def steps(caches):
        mine = table.clone()
        one = fa.paged_plan(i32(40, 0), i32(1, new), mine, i32(*free), new + 1, shape, pages)
        slots = one.slots.tolist()
        assert slots[0] == 2 * 16 + 8 and slots[1:17] == list(range(80, 96)) and set(slots[17:]) == {-1}
        assert mine[1, : -(-new // PAGE)].tolist() == [5] + [-1] * (-(-new // PAGE) - 1)
        assert torch.equal(mine[1, -(-new // PAGE):], table[1, -(-new // PAGE):]) and torch.equal(mine[0], table[0])
        want = fa.STATUS_OUT_OF_PAGES if len(free) == 1 or new > 32 else fa.STATUS_BAD_REQUEST
        assert fa.device_status()[0] == want
        first = _layer(one, new + 1, caches, 3)
        assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST     # attention met the absent page
        two = fa.paged_plan(one.kv_lens, i32(1, 1), mine, i32(*free), 2, shape, pages, free_cursor=one.free_cursor)
        assert two.slots.tolist()[1] == -1
        return first, _layer(two, 2, caches, 4)

    caches = [c.clone() for c in held]
    outs = steps(caches)
    changed = [c.clone() for c in held]
    for c, h in zip(caches, held):
        # Written: request 0's two new tokens and request 1's page.
        mask = torch.zeros(pages, PAGE, dtype=torch.bool, device=cuda_device)
        mask[2, 8:10] = mask[5] = True
        keep = ~mask[:, None, :, None].expand_as(c)
        assert torch.equal(c[keep], h[keep])
    # Request 1's rows do not depend on what request 0's pages hold.
    for c in changed:
        c[:2] = 3.0
    other = steps(changed)
    for a, b in zip(outs, other):
        assert torch.equal(a[1:], b[1:]) and not torch.equal(a[:1], b[:1])
    fa.device_status()


@pytest.mark.parametrize("seqs,placed", [(3, 1), (3, 2), (512, 511), (600, 100), (600, 512), (1300, 1024), (1300, 1299)])
def test_requests_without_rows_take_no_pages(cuda_device, seqs, placed):
    """total_tokens ends inside request `placed`: only the requests before it get pages, and the next step begins in the
    free list where theirs end."""
    width = 3
    cached, new = [(7 * b) % 20 for b in range(seqs)], [1 + (5 * b) % 23 for b in range(seqs)]
    table = torch.full((seqs, width), -5, dtype=torch.int32, device=cuda_device)
    free = torch.arange(seqs * width, dtype=torch.int32, device=cuda_device)
    total = sum(new[:placed]) + new[placed] - 1
    plan = fa.paged_plan(i32(*cached), i32(*new), table, free, total, fa.PagedShape(HEADS, KV_HEADS, DIM, PAGE), seqs * width)
    assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST
    want, taken = [[-5] * width for _ in range(seqs)], 0
    for b in range(placed):
        for i in range(-(-cached[b] // PAGE), -(-(cached[b] + new[b]) // PAGE)):
            want[b][i] = taken
            taken += 1
    assert table.tolist() == want
    assert plan.free_cursor.tolist() == [taken]
    assert plan.kv_lens.tolist() == [c + n if b < placed else 0 for b, (c, n) in enumerate(zip(cached, new))]
