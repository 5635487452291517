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


def _captured(q, caches, plan, out):
    """A graph of one attention call with the plan as it is now."""
    fa.paged_attention(q, *caches, plan, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fa.paged_attention(q, *caches, plan, out=out)
    return graph


OTHER_PLAN = 0x80000

# Heads, K/V heads, rows of the token axis, then (new lengths, causal, max_new) at capture and at replay.
OTHERS = [
    (8, 2, 340, ((300, 40), True, None), ((300, 40), False, None)),
    (8, 2, 340, ((300, 40), False, None), ((300, 40), True, None)),
    (8, 2, 16, ((1, 1), True, 1), ((8, 8), True, 8)),          # 4, then 32 rows to the narrow kernel
    (8, 2, 16, ((1, 1), True, 1), ((12, 1), True, 12)),        # no wide kernel, then work for one
    (8, 2, 16, ((4, 12), True, 16), ((8, 8), True, 8)),        # 16 narrow rows, then 32
    (8, 2, 40, ((8, 8), True, 8), ((33, 7), True, 33)),        # 32 narrow rows, no wide kernel; then 28 for one
    (24, 1, 2, ((1, 1), True, 2), ((1, 1), True, 1)),          # no narrow kernel, then work for one
]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,total,then,now", OTHERS)
def test_a_captured_call_meets_another_plan(cuda_device, dim, heads, kv_heads, total, then, now):
    """The arrays are written again for another mask or max_new while a graph holds a call made for the first: the
    replay reports it, ends, and is right again once the plan is."""
    shape = fa.PagedShape(heads, kv_heads, dim, PAGE)
    table = torch.arange(128, dtype=torch.int32, device=cuda_device).view(2, 64).contiguous()
    free = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    cached = i32(0, 500)
    # Every page is in the table, so plans hand out none: all of a request's tokens count as cached but the last new ones.
    kv = i32(900, 1000)

    def plan_of(which, plan=None):
        new, causal, max_new = which
        cached.copy_(kv - i32(*new))
        return fa.paged_plan(cached, i32(*new), table, free, total, shape, 128, causal=causal, max_new=max_new, plan=plan)

    caches = [normal(s, 128, kv_heads, PAGE, dim) for s in (1, 2)]
    q = normal(3, total, heads, dim)
    # Pages of the new tokens come from the free list; give the list what the table holds.
    entries = table.clone()
    plan = plan_of(then)
    table.copy_(entries)
    fa.device_status()
    out = torch.zeros_like(q)
    graph = _captured(q, caches, plan, out)
    want = out.clone()
    assert fa.device_status() == (fa.STATUS_OK, 0)
    plan_of(now, plan)
    table.copy_(entries)
    fa.device_status()
    graph.replay()
    status, word = fa.device_status()
    assert status == fa.STATUS_BAD_REQUEST and word == OTHER_PLAN
    plan_of(then, plan)
    table.copy_(entries)
    fa.device_status()
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    assert fa.device_status() == (fa.STATUS_OK, 0)
    graph.reset()


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("change", ["table", "kv_lens", "query_start"])
def test_a_call_whose_arrays_do_not_fit(cuda_device, new, change):
    """A table of a captured call that is shorter than what the plan was written for again, and arrays of a plan that
    somebody else wrote to."""
    shape = fa.PagedShape(HEADS, KV_HEADS, DIM, PAGE)
    pages, total = 256, 2 * new
    long_table = torch.arange(pages, dtype=torch.int32, device=cuda_device).view(2, 128).contiguous()
    table = long_table[:, :8].contiguous()
    free = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    caches = [normal(s, pages, KV_HEADS, PAGE, DIM) for s in (1, 2)]
    q = normal(3, total, HEADS, DIM)

    def plan_of(kv, block_table, plan=None):
        entries = block_table.clone()
        plan = fa.paged_plan(i32(kv - new, kv - new), i32(new, new), block_table, free, total, shape, pages, plan=plan)
        block_table.copy_(entries)
        fa.device_status()
        return plan

    plan = plan_of(128, table)
    out = torch.zeros_like(q)
    graph = _captured(q, caches, plan, out)
    want = out.clone()
    if change == "table":
        plan_of(1500, long_table, plan)
    elif change == "kv_lens":
        plan.kv_lens.add_(1000)
    else:
        plan.query_start[1:].add_(10 ** 6)
    graph.replay()
    status, word = fa.device_status()
    assert status == fa.STATUS_BAD_REQUEST and word == OTHER_PLAN
    plan_of(128, table, plan)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    assert fa.device_status() == (fa.STATUS_OK, 0)
    graph.reset()
