"""Paged-cache operators on a B200 against plain 64-bit forms: plan, rotary positions, append, attention,
and a run of them together."""
import ctypes

import numpy as np
import pytest
import torch

import cuda_fused_attention_b200 as fa
from cuda_fused_attention_b200 import _lib
from paged_reference import FaPagedPlan, Requests, attention, attention_bound, normal, rotary

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    fa.device_status()
    yield
    torch.cuda.synchronize()


def status_ok():
    assert fa.device_status() == (fa.STATUS_OK, 0)


# ---------------------------------------------------------------------------
# Plan
# ---------------------------------------------------------------------------
PLAN_LENGTHS = [
    ([0], [1]), ([15], [1]), ([16], [1]), ([17], [0]), ([0], [0]), ([], []),
    ([5, 0, 31, 16, 100], [1, 33, 0, 16, 300]),
    (list(range(0, 700)), [i % 5 for i in range(700)]),
    ([7 * i % 900 for i in range(1537)], [1 + (i * i) % 23 for i in range(1537)]),
    ([0, 3], [20000, 4097]),
]


@pytest.mark.parametrize("lengths", PLAN_LENGTHS, ids=lambda v: f"B{len(v[0])}")
@pytest.mark.parametrize("page_size,padding", [(16, 0), (32, 5), (256, 3000)])
def test_plan(cuda_device, lengths, page_size, padding):
    r = Requests(*lengths, page_size, cuda_device, seed=len(lengths[0]), padding=padding)
    plan = r.plan(fa.PagedShape(8, 2, 128, page_size))
    start, kv, positions, slots = r.expected()
    assert np.array_equal(plan.query_start.cpu().numpy(), start)
    assert np.array_equal(plan.kv_lens.cpu().numpy(), kv)
    assert np.array_equal(plan.positions.cpu().numpy(), positions)
    assert np.array_equal(plan.slots.cpu().numpy(), slots)
    assert np.array_equal(r.block_table.cpu().numpy(), r.table_after)
    assert plan.free_cursor.tolist() == [r.taken]
    assert plan.block_table is r.block_table
    again = r.plan(fa.PagedShape(8, 2, 128, page_size), plan=plan)      # the same inputs, the same buffers
    assert again is plan and np.array_equal(plan.slots.cpu().numpy(), slots)
    status_ok()


def _units(cached, new, group, causal):
    """Attention units of a request: (64-key tiles and an idle unit, 128-key tiles of token blocks, two units each or
    one for a block of at most 128 rows, and four idle units per block)."""
    if new == 0:
        return 0, 0
    if new * group <= 16:
        return 1 + -(-(cached + new) // 64), 0
    span = 2 * (128 // group)
    return 0, sum(4 + (1 if new - u <= span // 2 else 2) * -(-(cached + (min(new, u + span) if causal else new)) // 128)
                  for u in range(0, new, span))


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 16, 33, 64, 127, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_plan_schedule(cuda_device, group, causal):
    """The schedule's prefix sums, from whose closed form the attention finds its work."""
    cached = [0, 1, 63, 64, 127, 128, 129, 1000, 5003, 77, 0, 40000, 12, 300]
    new = [1, 300, 16, 17, 1, 128, 513, 2, 999, 0, 7001, 3, 1, 40]
    r = Requests(cached, new, 16, cuda_device)
    plan = r.plan(fa.PagedShape(group, 1, 64, 16), causal=causal)
    torch.cuda.synchronize()
    got = plan._buffer[: 4 * (len(new) + 1)].view(torch.int64).view(2, -1).tolist()
    units = np.array([_units(c, n, group, causal) for c, n in zip(cached, new)])
    want = np.concatenate([np.zeros((1, 2), np.int64), np.cumsum(units, 0)]).T.tolist()
    assert got == want


def test_plan_views_are_the_struct_s_pointers(cuda_device):
    """The struct that the C calls get has the C layout, and the views are where its pointers say."""
    r = Requests([5, 40, 0], [1, 3, 7], 16, cuda_device)
    plan = r.plan(fa.PagedShape(8, 2, 64, 16), max_new=9)
    c = FaPagedPlan.from_buffer_copy(plan._struct)
    assert len(plan._struct) == ctypes.sizeof(FaPagedPlan)
    width = r.block_table.shape[1]
    assert [getattr(c, n) for n, _ in FaPagedPlan._fields_[:12]] == [3, 11, 9, r.num_pages, width, width, 8, 2, 64, 16, 1, 0]
    for name, size in (("query_start", 4), ("kv_lens", 3), ("positions", 11), ("slots", 11), ("free_cursor", 1)):
        view = getattr(plan, name)
        assert view.data_ptr() == getattr(c, name) and view.shape == (size,) and view.dtype == torch.int32
    assert c.block_table == r.block_table.data_ptr() and c.schedule == plan._buffer.data_ptr()
    assert plan.free_cursor.data_ptr() + 4 == plan._buffer.data_ptr() + 4 * plan._buffer.numel()
    assert c.query_start == c.schedule + _lib.load().fa_sm100_paged_schedule_bytes(3)
    with pytest.raises(ValueError):
        r.plan(fa.PagedShape(8, 2, 128, 16), plan=plan)
    for own in ("cached_lens", "free_cursor"):      # blocks would read what others have written
        args = dict(cached_lens=r.cached_lens, free_cursor=None)
        args[own] = plan.kv_lens if own == "cached_lens" else plan.free_cursor
        with pytest.raises(ValueError, match="part of the plan"):
            fa.paged_plan(args["cached_lens"], r.new_lens, r.block_table, r.free_pages, r.total, plan.shape, r.num_pages,
                          free_cursor=args["free_cursor"], plan=plan)


def test_plan_steps_through_the_free_list(cuda_device):
    """Two steps: the second begins where the first left the cursor."""
    shape = fa.PagedShape(4, 4, 64, 16)
    table = torch.full((2, 8), -1, dtype=torch.int32, device=cuda_device)
    free = torch.tensor([9, 4, 7, 1, 3, 8, 0, 2, 6, 5], dtype=torch.int32, device=cuda_device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    one = fa.paged_plan(i32(0, 0), i32(20, 16), table, free, 36, shape, 10)
    assert one.free_cursor.tolist() == [3]
    two = fa.paged_plan(one.kv_lens, i32(12, 1), table, free, 13, shape, 10, free_cursor=one.free_cursor)
    assert two.free_cursor.tolist() == [4]
    assert table[:, :3].tolist() == [[9, 4, -1], [7, 1, -1]]
    assert two.slots.tolist() == [4 * 16 + i for i in range(4, 16)] + [16]
    status_ok()


def test_plan_records_what_is_wrong(cuda_device):
    shape = fa.PagedShape(4, 4, 64, 16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731

    def table(width=4):
        return torch.arange(2 * width, dtype=torch.int32, device=cuda_device).view(2, width)

    # A free list that runs out: the pages that exist are handed out, the others' tokens have no slot.
    plan = fa.paged_plan(i32(0, 0), i32(20, 17), table(), i32(30, 31, 32), 37, shape, 40)
    assert plan.slots.tolist() == [*range(480, 496), *range(496, 500), *range(512, 528), -1]
    assert plan.free_cursor.tolist() == [4]
    assert fa.device_status()[0] == fa.STATUS_OUT_OF_PAGES
    status_ok()
    # A page id outside the cache, in the table and in the free list.
    plan = fa.paged_plan(i32(3, 16), i32(1, 1), table() + 38, i32(40), 2, shape, 40)
    assert plan.slots.tolist() == [38 * 16 + 3, -1]
    assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST
    # Lengths: negative, past the table, more than the rows, more than max_new.
    for cached, new, total, how in [((-1, 3), (1, 1), 2, {}), ((64, 3), (1, 1), 2, {}), ((3, 3), (-2, 1), 1, {}),
                                    ((3, 3), (1, 2), 2, {}), ((3, 3), (2, 1), 3, {"max_new": 1})]:
        plan = fa.paged_plan(i32(*cached), i32(*new), table(), i32(20, 21), total, shape, 40, **how)
        assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST, (cached, new)
        bad = [c < 0 or n < 0 or c + n > 64 or how.get("max_new", 9) < n for c, n in zip(cached, new)]
        if new == (1, 2):
            bad = [False, True]     # its second token has no row
        assert (plan.kv_lens > 0).tolist() == [not x for x in bad]
    # INT_MAX lengths do not wrap.
    big = 2 ** 31 - 1
    plan = fa.paged_plan(i32(big, big), i32(big, 1), table(), i32(20, 21), 4, shape, 40)
    assert plan.kv_lens.tolist() == [0, 0] and fa.device_status()[0] == fa.STATUS_BAD_REQUEST
    status_ok()


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
def _freq(pairs, device="cuda"):
    return (10000.0 ** (-torch.arange(pairs, dtype=torch.float32, device=device) / pairs)).contiguous()


def _positions(axes, tokens, batch=None, far=0):
    gen = torch.Generator().manual_seed(axes * 1000 + tokens)
    shape = (axes, tokens) if batch is None else (axes, batch, tokens)
    return (torch.randint(0, 5000, shape, generator=gen) + far).to(torch.int32).cuda()


@pytest.mark.parametrize("dim,rotary_dim,sections", [
    (64, 64, (32,)), (64, 64, (8, 12, 12)), (128, 128, (16, 24, 24)), (128, 96, (1, 2, 5, 40)), (128, 16, (0, 8)),
    (64, 48, (5, 0, 19))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,heads,tokens", [(1, 1, 1), (2, 3, 37), (1, 40, 5), (3, 2, 1025)])
def test_rotary(cuda_device, dim, rotary_dim, sections, interleaved, batch, heads, tokens):
    x = normal(1, batch, heads, tokens, dim)
    freq = _freq(rotary_dim // 2)
    for positions in (_positions(len(sections), tokens), _positions(len(sections), tokens, batch, far=100000)):
        for inverse in (False, True):
            got = fa.rotary_embed(x, positions, freq, sections, interleaved, inverse)
            for b in range(batch):
                pos = positions if positions.dim() == 2 else positions[:, b]
                want, bound = rotary(x[b].transpose(0, 1), pos, freq, sections, interleaved, inverse)
                assert ((got[b].transpose(0, 1).double() - want).abs() <= bound).all()
    status_ok()


def test_rotary_far_positions(cuda_device):
    """Positions whose products with the frequencies need more than 32 bits, and negative ones."""
    freq = _freq(32)
    positions = torch.tensor([2 ** 31 - 1, -2 ** 31, 123456789, -1, 0, 2 ** 24 + 1], dtype=torch.int32).cuda()
    x = normal(2, 1, 2, 6, 64)
    got = fa.rotary_embed(x, positions, freq)
    want, bound = rotary(x[0].transpose(0, 1), positions[None], freq, (32,), False)
    assert ((got[0].transpose(0, 1).double() - want).abs() <= bound).all()


def test_rotary_strides_and_in_place(cuda_device):
    """[B, N, H, D] storage, a slice of a fused projection, and out = x give the same bits."""
    freq = _freq(64)
    positions = _positions(1, 65)
    x = normal(3, 2, 4, 65, 128)
    want = fa.rotary_embed(x, positions, freq)
    fused = torch.empty(2, 65, 3, 4, 128, dtype=torch.bfloat16, device=cuda_device)
    fused[:, :, 1] = x.transpose(1, 2)
    view = fused[:, :, 1].transpose(1, 2)
    assert torch.equal(fa.rotary_embed(view, positions, freq), want)
    out = torch.zeros(2, 65, 4, 128, dtype=torch.bfloat16, device=cuda_device).transpose(1, 2)
    assert fa.rotary_embed(x, positions, freq, out=out) is out and torch.equal(out, want)
    kept = fused.clone()
    fa.rotary_embed(view, positions, freq, out=view)
    assert torch.equal(view, want)
    assert torch.equal(fused[:, :, 0].view(torch.int16), kept[:, :, 0].view(torch.int16))
    assert torch.equal(fused[:, :, 2].view(torch.int16), kept[:, :, 2].view(torch.int16))


def test_rotary_gradient(cuda_device):
    """The inverse rotation is the gradient: against autograd of the 64-bit formula and against differences."""
    freq, positions = _freq(32), _positions(2, 9)
    sections = (10, 22)
    x, g = normal(4, 1, 2, 9, 64), normal(5, 1, 2, 9, 64)
    leaf = x.double().requires_grad_()
    out, _ = rotary(leaf[0].transpose(0, 1), positions, freq, sections, True)
    weight = g[0].transpose(0, 1).double()
    (out * weight).sum().backward()
    got = fa.rotary_embed(g, positions, freq, sections, True, inverse=True)
    _, bound = rotary(g[0].transpose(0, 1), positions, freq, sections, True, inverse=True)
    assert ((got[0].transpose(0, 1).double() - leaf.grad[0].transpose(0, 1)).abs() <= bound).all()
    # The map is linear, so a difference of any width is its derivative up to rounding in 64 bits.
    for e in (0, 1, 17, 63):
        step = torch.zeros_like(weight)
        step[4, 1, e] = 0.5
        base = x[0].transpose(0, 1).double()
        high, _ = rotary(base + step, positions, freq, sections, True)
        low, _ = rotary(base - step, positions, freq, sections, True)
        slope = ((high - low) * weight).sum()
        assert abs(got[0, 1, 4, e].double() - slope) <= bound[4, 1, e] + 1e-12


@pytest.mark.parametrize("shape", [(0, 2, 8, 64), (2, 0, 8, 64), (2, 2, 0, 64)])
def test_rotary_empty(cuda_device, shape):
    out = fa.rotary_embed(torch.empty(shape, dtype=torch.bfloat16, device=cuda_device), _positions(1, shape[2]), _freq(32))
    assert out.shape == shape


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv_heads,dim,page_size,sections,interleaved", [
    (8, 2, 128, 16, (64,), False), (5, 5, 64, 32, (8, 12, 12), True), (7, 1, 128, 256, (3, 29), False),
    (32, 8, 128, 64, (16, 24, 24), True)])
@pytest.mark.parametrize("cached,new", [([0], [1]), ([3, 250, 16], [40, 1, 17]), ([60] * 33, [1] * 33)])
def test_append(cuda_device, heads, kv_heads, dim, page_size, sections, interleaved, cached, new):
    r = Requests(cached, new, page_size, cuda_device, padding=3)
    plan = r.plan(fa.PagedShape(heads, kv_heads, dim, page_size))
    tokens = sum(new)
    qkv = normal(6, r.total, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
    k_cache = normal(7, r.num_pages, kv_heads, page_size, dim)
    v_cache = normal(8, r.num_pages, kv_heads, page_size, dim)
    freq = _freq(sum(sections))
    positions = plan.positions if len(sections) == 1 else _positions(len(sections), r.total)
    k_want, v_want = k_cache.clone(), v_cache.clone()
    out = torch.full((r.total, heads, dim), 9.0, dtype=torch.bfloat16, device=cuda_device)
    assert fa.rotary_append(q, k, v, k_cache, v_cache, positions, plan.slots, freq, sections, interleaved, out=out) is out
    axes = positions.view(len(sections), -1)
    want, bound = rotary(q, axes, freq, sections, interleaved)
    assert ((out.double() - want).abs() <= bound)[:tokens].all()
    assert (out[tokens:] == 9.0).all()
    slots = plan.slots[:tokens].long()
    page, row = slots // page_size, slots % page_size
    want, bound = rotary(k, axes, freq, sections, interleaved)
    assert ((k_cache[page, :, row].double() - want[:tokens]).abs() <= bound[:tokens]).all()
    assert torch.equal(v_cache[page, :, row], v[:tokens])
    k_want[page, :, row], v_want[page, :, row] = k_cache[page, :, row], v_cache[page, :, row]
    assert torch.equal(k_cache, k_want) and torch.equal(v_cache, v_want)      # nothing else was written
    # In place, and into caches of another stride order: the same bits.
    both = torch.zeros(r.num_pages, page_size, 2, kv_heads, dim, dtype=torch.bfloat16, device=cuda_device)
    k2, v2 = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    packed = q.clone()
    fa.rotary_append(packed, k, v, k2, v2, positions, plan.slots, freq, sections, interleaved, out=packed)
    assert torch.equal(packed[:tokens], out[:tokens]) and torch.equal(packed[tokens:], q[tokens:])
    assert torch.equal(k2[page, :, row], k_cache[page, :, row]) and torch.equal(v2[page, :, row], v[:tokens])
    status_ok()


def test_append_slot_outside_the_cache(cuda_device):
    q, k = normal(9, 3, 2, 64), normal(10, 3, 2, 64)
    caches = [torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device=cuda_device) for _ in range(2)]
    slots = torch.tensor([31, 32, -1], dtype=torch.int32, device=cuda_device)
    out = torch.zeros_like(q)
    fa.rotary_append(q, k, k, *caches, _positions(1, 3), slots, _freq(32), out=out)
    assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST
    assert (out[1:] == 0).all() and torch.equal(caches[1][1, :, 15], k[0]) and (caches[1][0] == 0).all()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def check_attention(r, heads, kv_heads, dim, causal=True, seed=0, q=None, caches=None, q_scale=1.0, **how):
    if caches is None:
        caches = (normal(seed + 11, r.num_pages, kv_heads, r.page_size, dim, device=r.device),
                  normal(seed + 12, r.num_pages, kv_heads, r.page_size, dim, device=r.device))
    if q is None:
        q = normal(seed + 13, r.total, heads, dim, device=r.device, scale=q_scale)
    plan = r.plan(fa.PagedShape(heads, kv_heads, dim, r.page_size), causal=causal, **how)
    out = torch.full((r.total, heads, dim), 9.0, dtype=torch.bfloat16, device=r.device)
    assert fa.paged_attention(q, *caches, plan, out=out) is out
    want, mag = attention(q, *caches, r, causal)
    tokens = sum(r.new)
    off = (out.double() - want).abs() - attention_bound(want, mag)
    assert off[:tokens].max() <= 0 if tokens else True, f"over the bound by {off[:tokens].max().item():.3e}"
    assert (out[tokens:] == 9.0).all()
    status_ok()
    return q, caches, plan, out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 2), (7, 1), (16, 1), (6, 2), (32, 1)])
@pytest.mark.parametrize("page_size", [16, 128])
def test_decode(cuda_device, dim, heads, kv_heads, page_size):
    cached = [0, 1, 14, 15, 16, 62, 63, 64, 65, 127, 128, 500, 1023, 3001]
    check_attention(Requests(cached, [1] * len(cached), page_size, cuda_device, padding=2), heads, kv_heads, dim)


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_page_sizes(cuda_device, page_size, causal):
    """One-token, few-token and chunk requests in one call, at every page size."""
    r = Requests([700, 5, 130, 0, 64, 255, 9], [1, 4, 100, 257, 0, 1, 3], page_size, cuda_device, padding=1)
    check_attention(r, 8, 2, 128, causal)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (3, 1), (14, 2), (40, 1), (128, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(cuda_device, dim, heads, kv_heads, causal):
    """Chunk lengths on both sides of the 128-row tiles, with and without cached tokens."""
    span = 128 // (heads // kv_heads)
    new = sorted({1, span - 1, span, span + 1, 2 * span - 1, 2 * span, 2 * span + 1, 3 * span + 2, 130, 301})
    new = [n for n in new if n > 0]
    cached = [(0, 1, 127, 128, 300, 63)[i % 6] for i in range(len(new))]
    check_attention(Requests(cached, new, 32, cuda_device), heads, kv_heads, dim, causal)


@pytest.mark.parametrize("new", [1, 3, 16, 200])
@pytest.mark.parametrize("q_scale", [1.0, 8.0])
def test_long_context_is_split(cuda_device, new, q_scale):
    """One request with a long cache: its keys are shared out over the GPU and merged. Large scores move a row's
    maximum along the keys, so the parts' weights differ."""
    check_attention(Requests([20011], [new], 64, cuda_device), 8, 2, 128, q_scale=q_scale)


def test_many_requests(cuda_device):
    """More requests than threads of a block, most of them short, some empty."""
    cached = [(37 * i) % 211 for i in range(1500)]
    new = [(i * 7) % 4 for i in range(1500)]
    check_attention(Requests(cached, new, 16, cuda_device), 4, 2, 64)


def test_one_new_token_in_an_empty_cache(cuda_device):
    """The softmax of a single key is one: the output is V, bit for bit."""
    r = Requests([0, 0, 0], [1, 1, 1], 16, cuda_device)
    q, (_, v), plan, out = check_attention(r, 4, 2, 64)
    slots = plan.slots.long()
    assert torch.equal(out, v[slots // 16, :, slots % 16].repeat_interleave(2, dim=1))


@pytest.mark.parametrize("new", [1, 40])
def test_large_scores(cuda_device, new):
    """Scores in the thousands, of either sign, and equal keys (all weights equal)."""
    r = Requests([400, 1000], [new, new], 16, cuda_device)
    check_attention(r, 4, 1, 128, q_scale=300.0)
    k = torch.ones(r.num_pages, 1, 16, 128, dtype=torch.bfloat16, device=cuda_device)
    check_attention(r, 4, 1, 128, q_scale=-100.0, caches=(k, normal(3, *k.shape)))


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("cached,new", [([0, 30, 100, 500], [1, 1, 1, 1]), ([0, 30, 100, 500], [70, 129, 40, 5]),
                                        ([5000], [1]), ([5000], [60])])
@pytest.mark.parametrize("page_size", [16, 256])
def test_what_lies_behind_the_last_token_is_not_used(cuda_device, poison, cached, new, page_size):
    r = Requests(cached, new, page_size, cuda_device, padding=4)
    k, v = (normal(s, r.num_pages, 2, page_size, 64) for s in (1, 2))
    seen = torch.zeros(r.num_pages, page_size, dtype=torch.bool, device=cuda_device)
    for b, (c, n) in enumerate(zip(cached, new)):
        for i in range(-(-(c + n) // page_size)):
            seen[int(r.table_after[b, i]), : c + n - i * page_size] = True
    q = normal(3, r.total, 8, 64)
    q[sum(new):] = poison
    clean = check_attention(r, 8, 2, 64, q=q, caches=(k, v))[3]
    hidden = ~seen[:, None, :, None].expand_as(k)
    dirty = check_attention_bits(r, 8, 2, 64, q, k.masked_fill(hidden, poison), v.masked_fill(hidden, poison))
    assert torch.equal(clean[: sum(new)], dirty[: sum(new)])


def check_attention_bits(r, heads, kv_heads, dim, q, k, v):
    plan = r.plan(fa.PagedShape(heads, kv_heads, dim, r.page_size))
    out = fa.paged_attention(q, k, v, plan)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("new", [1, 90])
def test_non_finite_inputs_reach_their_rows_only(cuda_device, new):
    """A NaN in one request's Q, K or V stays in that request (and that K/V head)."""
    r = Requests([100, 300, 64], [new, new, new], 16, cuda_device)
    q, (k, v), plan, clean = check_attention(r, 4, 2, 64)
    page = int(r.table_after[1, 2])
    for t in (k, v):
        dirty = t.clone()
        dirty[page, 1, 5, 7] = float("nan")
        out = fa.paged_attention(q, dirty if t is k else k, dirty if t is v else v, plan)
        assert torch.equal(out[:new], clean[:new]) and torch.equal(out[2 * new:], clean[2 * new:])
        assert torch.equal(out[new: 2 * new, :2], clean[new: 2 * new, :2])
        assert out[new: 2 * new, 2:, 7].isnan().all()
    dirty = q.clone()
    dirty[new, 3, 0] = float("nan")
    out = fa.paged_attention(dirty, k, v, plan)
    assert out[new, 3].isnan().all()
    out[new, 3] = clean[new, 3]
    assert torch.equal(out, clean)


def test_strides(cuda_device):
    """Q as a slice of a fused projection, caches as [pages, rows, heads, D] and as halves of one tensor, out with
    rows apart: the same bits as contiguous tensors."""
    r = Requests([100, 700, 3], [1, 3, 150], 32, cuda_device)
    q, (k, v), plan, want = check_attention(r, 8, 4, 128)
    fused = normal(5, r.total, 16, 128)
    fused[:, :8] = q
    both = torch.empty(r.num_pages, 32, 2, 4, 128, dtype=torch.bfloat16, device=cuda_device)
    both[:, :, 0], both[:, :, 1] = k.transpose(1, 2), v.transpose(1, 2)
    out = torch.empty(r.total, 8, 136, dtype=torch.bfloat16, device=cuda_device)[..., :128]
    fa.paged_attention(fused[:, :8], both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2), plan, out=out)
    assert torch.equal(out, want)
    halves = torch.stack([k, v], dim=1)
    assert torch.equal(fa.paged_attention(q, halves[:, 0], halves[:, 1], plan), want)
    # Only one table: its rows apart from each other.
    wide = torch.full((3, r.block_table.shape[1] + 5), -1, dtype=torch.int32, device=cuda_device)
    wide[:, : r.block_table.shape[1]] = r.block_table
    plan2 = fa.paged_plan(r.cached_lens, r.new_lens, wide[:, : r.block_table.shape[1]], r.free_pages, r.total,
                          plan.shape, r.num_pages)
    assert torch.equal(fa.paged_attention(q, k, v, plan2), want)


def test_shared_pages_and_output_over_q(cuda_device):
    """Two requests that share a prefix's pages; one tensor as K and V; O written over Q."""
    r = Requests([160, 160], [5, 40], 16, cuda_device)
    r.table_after[1, :10] = r.table_after[0, :10]
    r.block_table[1, :10] = r.block_table[0, :10]
    q, (k, v), plan, want = check_attention(r, 4, 2, 64)
    mine = q.clone()
    assert fa.paged_attention(mine, k, v, plan, out=mine) is mine and torch.equal(mine, want)
    same = check_attention(r, 4, 2, 64, q=q, caches=(k, k))
    assert same[3].isfinite().all()


@pytest.mark.parametrize("seed", range(40))
def test_mixed_batches(cuda_device, seed):
    """Random batches over all head layouts, page sizes and kinds of requests, with scores that move the rows' maxima."""
    rng = np.random.RandomState(seed)
    dim, page_size = int(rng.choice([64, 128])), int(rng.choice([16, 32, 64, 128, 256]))
    kv_heads = int(rng.choice([1, 2, 3, 8]))
    heads = kv_heads * int(rng.choice([1, 2, 3, 4, 5, 8, 16, 24]))
    seqs = int(rng.choice([1, 2, 7, 33, 64]))
    most = int(rng.choice([1, 4, 9, 40, 300]))
    cached = [int(x) for x in np.exp(rng.uniform(0, np.log(4000), seqs)).astype(int) - 1]
    new = [int(x) for x in rng.randint(0, most + 1, seqs)]
    r = Requests(cached, new, page_size, cuda_device, seed=seed, padding=int(rng.randint(0, 5)))
    how = {"max_new": most} if seed % 2 else {}
    q, caches, plan, out = check_attention(r, heads, kv_heads, dim, bool(rng.randint(0, 4)), seed, q_scale=float(rng.choice([1, 4, 12])),
                                           **how)
    if sum(new):
        again = fa.paged_attention(q, *caches, plan)
        assert torch.equal(again[: sum(new)], out[: sum(new)])


def test_same_bits_every_time(cuda_device):
    r = Requests([9000, 17, 4000], [1, 200, 6], 16, cuda_device)
    q, (k, v), plan, want = check_attention(r, 8, 2, 128)
    for _ in range(20):
        assert torch.equal(fa.paged_attention(q, k, v, plan), want)


def test_offsets_past_32_bits(cuda_device):
    """A cache of more than 2^31 elements, the pages in use at both ends."""
    pages = 2 ** 31 // (8 * 64 * 128) + 40
    r = Requests([200, 100, 3000], [1, 130, 2], 64, cuda_device)
    used = r.num_pages
    r.table_after = np.where(r.table_after >= 0, pages - 1 - r.table_after * (pages // used), -7).astype(np.int32)
    r.block_table = torch.from_numpy(r.table_after).cuda()
    caches = []
    for seed in (1, 2):
        c = torch.zeros(pages, 8, 64, 128, dtype=torch.bfloat16, device=cuda_device)
        ids = torch.from_numpy(r.table_after[r.table_after >= 0].astype(np.int64)).cuda()
        c[ids] = normal(seed, ids.numel(), 8, 64, 128)
        caches.append(c)
    assert caches[0].numel() > 2 ** 31 and int(r.table_after.max()) * 8 * 64 * 128 > 2 ** 31
    r.num_pages = pages
    # The table holds every page already: cached + new tokens of a plan that takes none.
    plan = fa.paged_plan(r.cached_lens, r.new_lens, r.block_table, free_of(r, cuda_device), r.total,
                         fa.PagedShape(16, 8, 128, 64), pages)
    q = normal(3, r.total, 16, 128)
    out = fa.paged_attention(q, *caches, plan)
    want, mag = attention(q, *caches, r)
    assert ((out.double() - want).abs() <= attention_bound(want, mag)).all()
    status_ok()


def free_of(r, device):
    """The pages that r's new tokens take, in order, so that a plan hands out what table_after holds."""
    ids = []
    for b, (c, n) in enumerate(zip(r.cached, r.new)):
        ids += r.table_after[b, -(-c // r.page_size): -(-(c + n) // r.page_size)].tolist()
    return torch.tensor(ids, dtype=torch.int32, device=device)


def test_bad_pages_are_recorded(cuda_device):
    """A page id outside the cache: recorded, nothing read, the other requests unharmed."""
    for new in (1, 60):
        r = Requests([100, 300], [new, new], 16, cuda_device)
        q, (k, v), plan, want = check_attention(r, 4, 2, 64)
        for bad in (-1, r.num_pages, 2 ** 31 - 1, -2 ** 31):
            r.block_table[1, 3] = bad
            out = fa.paged_attention(q, k, v, plan)
            assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST
            assert torch.equal(out[:new], want[:new])
        status_ok()


def test_bad_lengths_get_no_work(cuda_device):
    """A request with invalid lengths keeps its place on the token axis; its rows are not written."""
    r = Requests([100, 300, 20], [2, 3, 40], 16, cuda_device)
    q, caches, plan, want = check_attention(r, 4, 2, 64)
    r.cached_lens[1] = 10 ** 6
    plan = r.plan(plan.shape)
    assert fa.device_status()[0] == fa.STATUS_BAD_REQUEST
    out = torch.full_like(want, 9.0)
    fa.paged_attention(q, *caches, plan, out=out)
    assert torch.equal(out[:2], want[:2]) and torch.equal(out[5:], want[5:]) and (out[2:5] == 9.0).all()
    status_ok()


def test_empty_calls(cuda_device):
    for cached, new, padding in [([], [], 0), ([5, 0], [0, 0], 0), ([], [], 4), ([7], [0], 3)]:
        check_attention(Requests(cached, new, 16, cuda_device, padding=padding), 4, 2, 64)


@pytest.mark.parametrize("new", [[1, 1], [100, 40], [1, 100]])
def test_a_stalled_launch_gives_up(cuda_device, new):
    """A wait that runs out: an error status, nothing written, and the next call is right."""
    r = Requests([700, 90], new, 16, cuda_device)
    q, (k, v), plan, want = check_attention(r, 8, 2, 128)
    out = torch.full_like(want, 9.0)
    assert _lib.load().fa_sm100_paged_test_arm_stall() == 0
    fa.paged_attention(q, k, v, plan, out=out)
    status, word = fa.device_status()
    assert status == fa.STATUS_DEVICE_TIMEOUT and word & 1
    assert (out == 9.0).all()
    status_ok()
    assert torch.equal(fa.paged_attention(q, k, v, plan), want)
    status_ok()


# ---------------------------------------------------------------------------
# Streams, graphs, and the operators together
# ---------------------------------------------------------------------------
def test_streams(cuda_device):
    """Calls at the same time on two streams, with their plans made there: each its own result."""
    sets = []
    for i, (cached, new) in enumerate([([9000, 40], [1, 1]), ([3000, 100], [64, 200])]):
        r = Requests(cached, new, 16, cuda_device, seed=i)
        sets.append((r, *check_attention(r, 8, 2, 128, seed=i)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (r, q, (k, v), plan, want) in enumerate(sets):
            plan = r.plan(plan.shape, stream=streams[i])
            outs[i].append(fa.paged_attention(q, k, v, plan, stream=streams[i].cuda_stream if i else streams[i]))
    torch.cuda.synchronize()
    for got, (*_, want) in zip(outs, sets):
        assert all(torch.equal(o, want) for o in got)


def _layer(r, plan, q, k, v, caches, freq, out=None):
    turned = fa.rotary_append(q, k, v, *caches, plan.positions, plan.slots, freq)
    return fa.paged_attention(turned, *caches, plan, out=out)


def test_steps_of_a_request_equal_the_dense_forward(cuda_device):
    """A prompt in chunks, then single tokens, through plan, append and attention: the rows of one causal dense
    forward over the whole sequence, whose Q and K were rotated with rotary_embed."""
    heads, dim, page_size, length = 4, 128, 16, 333
    shape = fa.PagedShape(heads, heads, dim, page_size)
    q, k, v = (normal(s, length, heads, dim) for s in (1, 2, 3))
    freq = _freq(dim // 2)
    positions = torch.arange(length, dtype=torch.int32, device=cuda_device)
    dense = lambda t: t.transpose(0, 1)[None].contiguous()  # noqa: E731
    qr, kr = (fa.rotary_embed(dense(t), positions, freq) for t in (q, k))
    want = fa.attention_forward(qr, kr, dense(v), causal=True)[0].transpose(0, 1).double()
    pages = 30
    caches = [torch.full((pages, heads, page_size, dim), float("nan"), dtype=torch.bfloat16, device=cuda_device)
              for _ in range(2)]
    table = torch.full((1, 25), -1, dtype=torch.int32, device=cuda_device)
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    at, cached, cursor, rows = 0, torch.zeros(1, dtype=torch.int32, device=cuda_device), None, []
    for n in [100, 1, 1, 130, 16, 5, 1, 1, 64, 14]:
        new = torch.tensor([n], dtype=torch.int32, device=cuda_device)
        plan = fa.paged_plan(cached, new, table, free, n, shape, pages, free_cursor=cursor)
        rows.append(_layer(None, plan, q[at: at + n], k[at: at + n], v[at: at + n], caches, freq))
        cached, cursor, at = plan.kv_lens, plan.free_cursor, at + n
    got = torch.cat(rows).double()
    assert at == length
    keys = kr[0].transpose(0, 1)
    s = torch.einsum("ihd,jhd->hij", qr[0].transpose(0, 1).double(), keys.double()) / dim ** 0.5
    s.masked_fill_(torch.ones(length, length, device=cuda_device).triu(1).bool(), float("-inf"))
    exact = torch.einsum("hij,jhd->ihd", s.softmax(-1), v.double())
    mag = torch.einsum("hij,jhd->ihd", s.softmax(-1), v.double().abs())
    assert ((got - exact).abs() <= attention_bound(exact, mag)).all()
    assert ((want - exact).abs() <= attention_bound(exact, mag)).all()
    status_ok()


def test_captured_steps(cuda_device):
    """A decode step captured with room for padding, replayed for growing requests: each replay equals eager calls.
    A second graph of the same plan buffers, captured between, does not disturb it."""
    heads, kv_heads, dim, page_size, pages = 8, 2, 64, 16, 64
    shape = fa.PagedShape(heads, kv_heads, dim, page_size)
    seqs, total = 3, 12
    freq = _freq(dim // 2)
    cached = torch.tensor([5, 40, 200], dtype=torch.int32, device=cuda_device)
    new = torch.tensor([1, 4, 1], dtype=torch.int32, device=cuda_device)
    table = torch.full((seqs, 20), -1, dtype=torch.int32, device=cuda_device)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
    table[0, :1], table[1, :3], table[2, :13] = order[:1], order[1:4], order[4:17]
    free = order[17:].clone()
    cursor = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    caches = [normal(s, pages, kv_heads, page_size, dim) for s in (1, 2)]
    qkv = normal(3, total, heads + 2 * kv_heads, dim)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)

    def step(plan=None, out=None):
        plan = fa.paged_plan(cached, new, table, free, total, shape, pages, free_cursor=cursor, plan=plan)
        return plan, _layer(None, plan, q, k, v, caches, freq, out)

    state = [t.clone() for t in (cached, new, table, cursor, *caches)]

    def restore():
        for t, s in zip((cached, new, table, cursor, *caches), state):
            t.copy_(s)

    def advance(plan, i):
        cached.copy_(plan.kv_lens)
        cursor.copy_(plan.free_cursor)
        new.copy_(torch.tensor([(1, 1, 1), (6, 1, 0), (2, 8, 2)][i % 3], dtype=torch.int32))

    want = []
    for i in range(7):
        plan, out = step()
        want.append((out[: int(new.sum())].clone(), table.clone()))
        advance(plan, i)
    restore()
    plan, _ = step()
    out = torch.empty(total, heads, dim, dtype=torch.bfloat16, device=cuda_device)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(plan, out)
        graphs.append(graph)
    restore()
    for i in range(7):
        graphs[i % 2].replay()
        rows = int(new.sum())
        assert torch.equal(out[:rows], want[i][0]) and torch.equal(table, want[i][1])
        advance(plan, i)
    status_ok()
    for graph in graphs:
        graph.reset()


@pytest.mark.parametrize("dim, new", [(64, [1, 1, 3, 1]), (128, [1, 40, 0, 300]), (64, [70, 129, 257, 64])])
def test_launches_that_overlap(cuda_device, dim, new):
    """Kernels that start before the one in front of them is done: chains in which each call needs the one before,
    with copies between, on one stream and over a fork and a join, launched and captured; the inputs change
    before every pass. Each pass equals calls with a synchronisation behind each."""
    heads, kv_heads, page_size = 8, 2, 16
    r = Requests([700, 0, 33, 64], new, page_size, cuda_device, seed=5)
    shape = fa.PagedShape(heads, kv_heads, dim, page_size)
    freq = _freq(dim // 2)
    caches = [normal(s, r.num_pages, kv_heads, page_size, dim) for s in (1, 2)]
    start = [c.clone() for c in caches]
    sources = [normal(s, r.total, heads + 2 * kv_heads, dim) for s in (3, 4, 5)]
    source, qkv = sources[0].clone(), torch.empty_like(sources[0])
    table = r.block_table.clone()
    side = torch.cuda.Stream()

    def chain(wait):
        r.block_table.copy_(table)
        for c, s in zip(caches, start):
            c.copy_(s)
        qkv.copy_(source)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], dim=1)
        wait()
        plan = r.plan(shape)
        wait()
        outs = []
        for _ in range(3):
            out = _layer(None, plan, q, k, v, caches, freq)
            wait()
            main = torch.cuda.current_stream()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                turned = fa.rotary_embed(out.transpose(0, 1)[None], plan.positions, freq)[0].transpose(0, 1)
            wait()
            q = fa.paged_attention(out, *caches, plan)
            wait()
            main.wait_stream(side)
            q = fa.paged_attention(q + turned, *caches, plan)
            wait()
            outs += [out, turned, q]
        return outs

    want = []
    for s in sources:
        source.copy_(s)
        want.append([o.clone() for o in chain(torch.cuda.synchronize)])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain(lambda: None)
    for i in range(9):
        source.copy_(sources[i % 3])
        for o, w in zip(chain(lambda: None), want[i % 3]):
            assert torch.equal(o, w)
        graph.replay()
        for o, w in zip(captured, want[i % 3]):
            assert torch.equal(o, w)
    graph.reset()
    status_ok()
