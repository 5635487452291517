"""Paged attention under bounds that see a lost or doubled key: marked values whose sums are exact, and bounds that
follow each kernel's arithmetic (see `bounds`)."""
import math

import numpy as np
import pytest
import torch

import cuda_fused_attention_b200 as fa
from paged_reference import BF16_HALF_STEP, Requests, normal


def marked(r, kv_heads, dim, device, by=1):
    """K = 0 and V one-hot: the value of key j has its one in column (j // by) % D. All weights are one, so the output is
    (keys of a column) / (keys), from sums that 32 bits hold exactly: it is rounded by the reciprocal, the product and bf16."""
    k = torch.zeros(r.num_pages, kv_heads, r.page_size, dim, dtype=torch.bfloat16, device=device)
    v = torch.zeros_like(k)
    for b, (c, n) in enumerate(zip(r.cached, r.new)):
        key = torch.arange(c + n, device=device)
        page = torch.from_numpy(r.table_after[b].astype(np.int64)).to(device)[key // r.page_size]
        v[page, :, key % r.page_size] = torch.eye(dim, dtype=torch.bfloat16, device=device)[key // by % dim][:, None]
    return k, v


def counted(r, heads, dim, causal, by, device):
    """The output for `marked` values: [tokens, heads, D]."""
    rows = []
    for c, n in zip(r.cached, r.new):
        if n == 0:
            continue
        seen = torch.nn.functional.one_hot(torch.arange(c + n) // by % dim, dim).double().cumsum(0)
        last = torch.arange(c, c + n) if causal else torch.full((n,), c + n - 1)
        rows.append(seen[last] / (last + 1)[:, None].double())
    return torch.cat(rows)[:, None].expand(-1, heads, dim).to(device)


def counted_bound(o):
    # bf16's half step; the reciprocal and the product, and merged weights that are one: 2^-22 in all.
    return (BF16_HALF_STEP * (1 + 2.0 ** -8) + 2.0 ** -22) * o


def check_marked(r, heads, kv_heads, dim, causal=True, **how):
    for by in (1, 64):
        plan = r.plan(fa.PagedShape(heads, kv_heads, dim, r.page_size), causal=causal, **how)
        q = normal(5, r.total, heads, dim)
        out = fa.paged_attention(q, *marked(r, kv_heads, dim, "cuda", by), plan)
        want = counted(r, heads, dim, causal, by, "cuda")
        assert ((out[: sum(r.new)].double() - want).abs() <= counted_bound(want)).all()
    assert fa.device_status() == (fa.STATUS_OK, 0)


# Keys of a column: at most 2 * 64 where 64 neighbours share one, so a single lost key changes it by 2^-7, two half steps.
LOST = [([1000], [1], 64, 1), ([16383], [1], 128, 64), ([8100], [5], 64, 64), ([130], [70], 64, 1), ([16000], [200], 128, 64)]


@pytest.mark.parametrize("cached,new,dim,by", LOST)
def test_marks_see_a_lost_or_doubled_key(cached, new, dim, by):
    """Planted in the oracle: each key in turn missing from, or twice in, a row's sums is outside the bound."""
    r = Requests(cached, new, 16, "cpu")
    want = counted(r, 1, dim, True, by, "cpu")[:, 0]
    keys = torch.arange(cached[0] + 1)         # of the first new token
    count = want[0] * keys.numel()
    for step in (-1, 1):
        hit = count[keys // by % dim] + step
        off = (hit / (keys.numel() + step) - want[0][keys // by % dim]).abs()
        assert (off > counted_bound(want[0][keys // by % dim]) + BF16_HALF_STEP * want[0][keys // by % dim] / 8).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cached,new", [
    ([0], [1]), ([2047], [1]), ([16383], [1]), ([5000, 17, 8000, 0], [1, 1, 1, 1]), ([9001], [4]), ([8100, 64], [5, 8]),
    ([0], [1]), ([0], [777]), ([8000], [200]), ([3000, 100, 0, 7777], [64, 300, 129, 1]), ([14336], [512])])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (5, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_every_key_counts_once(cuda_device, cached, new, heads, kv_heads, dim, causal):
    check_marked(Requests(cached, new, 32, cuda_device, padding=1), heads, kv_heads, dim, causal, max_new=max(new))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_every_key_counts_once_in_mixed_batches(cuda_device, seed):
    rng = np.random.RandomState(seed)
    dim, page_size = int(rng.choice([64, 128])), int(rng.choice([16, 32, 64, 128, 256]))
    kv_heads = int(rng.choice([1, 2, 8]))
    seqs, most = int(rng.choice([1, 3, 20, 50])), int(rng.choice([1, 6, 40, 400]))
    cached = [int(x) for x in np.exp(rng.uniform(0, np.log(6000), seqs)).astype(int) - 1]
    new = [int(x) for x in rng.randint(0, most + 1, seqs)]
    new[0] = most
    r = Requests(cached, new, page_size, cuda_device, seed=seed)
    check_marked(r, kv_heads * int(rng.choice([1, 2, 3, 4, 7, 16])), kv_heads, dim, bool(seed % 3), **({"max_new": most} if seed % 2 else {}))


# ---------------------------------------------------------------------------
# The kernels' arithmetic
# ---------------------------------------------------------------------------
def bounds(q, k_cache, v_cache, r, causal, max_new, sms):
    """(o, bound) in 64 bits of every row. A row's o = sum_j w_j v_j / sum_j w_j, w_j = exp(s_j - m):

    scores   a matrix instruction adds 16 products to what it has; each of the 17 numbers is cut below 2^-24 of the
             largest, which is at most what it has plus the 16 products' sizes. D / 16 of them, over sqrt(D).
    weights  the exponent's product and difference 2^-22 of |s| and of the base, which lies within 16 log(2) of a score;
             exp2 2^-22. Parts are weighted twice more (groups of keys, then parts).
             Narrow kernel: a weight is two bf16 numbers, 2^-16 of it. Wide kernel: one, 2^-8 of it, for the product
             with V alone; these roundings have no common sign, and 8 times the root of their squares' sum is passed
             by chance with a probability of 2 exp(-32).
    sums     products with V as the scores, over the keys of one stretch of the work; the weights' sum in at least four
             chains; parts one after another.
    result   one rounding to bf16.
    """
    total, heads, dim = q.shape
    kv_heads = k_cache.shape[1]
    group = heads // kv_heads
    most = min(max_new, total) * group
    narrow_rows = 32 if 16 < most <= 32 else 16
    tiles = [-(-(c + n) // 64) for c, n in zip(r.cached, r.new)]
    narrow = [n * group <= narrow_rows for n in r.new]
    span = 2 * (128 // group)
    narrow_units = kv_heads * sum(t + 1 for t, n, is_narrow in zip(tiles, r.new, narrow) if n and is_narrow)
    wide_units = kv_heads * sum(-(-n // span) * (4 + 2 * -(-t // 2)) for t, n, is_narrow in zip(tiles, r.new, narrow) if not is_narrow)
    stretch = {True: 64 * max(2, -(-narrow_units // (2 * sms))), False: 128 * max(4, -(-wide_units // sms))}
    out = torch.zeros(total, heads, dim, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    row, step = 0, 2.0 ** -24
    for b, (c, n) in enumerate(zip(r.cached, r.new)):
        kv = c + n
        if n == 0:
            continue
        pages = torch.from_numpy(r.table_after[b, : -(-kv // r.page_size)].astype(np.int64)).to(q.device)
        for h in range(kv_heads):
            k = k_cache[pages, h].reshape(-1, dim)[:kv].double().view(kv, dim // 16, 16)
            v = v_cache[pages, h].reshape(-1, dim)[:kv].double()
            x = q[row: row + n, h * group: (h + 1) * group].double().reshape(n * group, dim // 16, 16)
            blocks = torch.einsum("rbe,kbe->rkb", x, k)
            sizes = torch.einsum("rbe,kbe->rkb", x.abs(), k.abs())
            sums = blocks.cumsum(-1)
            off = 17 * step * ((sums - blocks).abs() + sizes).sum(-1) / math.sqrt(dim)
            s = sums[..., -1] / math.sqrt(dim)
            del blocks, sizes, sums
            if causal:
                last = torch.arange(c, kv, device=q.device).repeat_interleave(group)
                s.masked_fill_(torch.arange(kv, device=q.device) > last[:, None], -math.inf)
            p = torch.softmax(s, -1)
            size = torch.where(s.isinf(), torch.zeros_like(s), s.abs())
            delta = off + 3 * (2.0 ** -22 + 2.0 ** -22 * (size + size.amax(-1, keepdim=True) + 12))
            if narrow[b]:
                delta += 2.0 ** -16
            o, mag = p @ v, p @ v.abs()
            keys = min(kv, stretch[narrow[b]])
            chain = (17 / 16 * keys + keys / 4 + 2 * (kv / 64) + 64) * step
            e = BF16_HALF_STEP * (1 + 2.0 ** -8) * o.abs() + (p * delta) @ v.abs() + (p * delta).sum(-1, keepdim=True) * o.abs()
            e += chain * (mag + o.abs()) + 1e-30
            if not narrow[b]:
                e += 8 * BF16_HALF_STEP * ((p * p) @ (v * v)).sqrt()
            at = slice(h * group, (h + 1) * group)
            out[row: row + n, at], bound[row: row + n, at] = o.view(n, group, dim), e.view(n, group, dim)
        row += n
    return out, bound


@pytest.mark.parametrize("q_scale", [1.0, 8.0])
@pytest.mark.parametrize("new", [1, 16])
def test_bounds_see_a_lost_tile(new, q_scale):
    """Planted in the oracle: each 64-key tile in turn missing from a long context, seen if it holds 2^-12 of a row's
    weight (with large scores some tiles hold less: their loss is smaller than the result's rounding)."""
    r = Requests([5000], [new], 64, "cpu")
    k, v = normal(11, r.num_pages, 1, 64, 128, device="cpu"), normal(12, r.num_pages, 1, 64, 128, device="cpu")
    q = normal(13, r.total, 4, 128, device="cpu", scale=q_scale)
    want, bound = bounds(q, k, v, r, True, new, 148)
    pages = torch.from_numpy(r.table_after[0, : -(-(5000 + new) // 64)].astype(np.int64))
    kd, vd = (t[pages, 0].reshape(-1, 128)[: 5000 + new].double() for t in (k, v))
    s = q.double().reshape(-1, 128) @ kd.T / math.sqrt(128)
    s.masked_fill_(torch.arange(5000 + new) > torch.arange(5000, 5000 + new).repeat_interleave(4)[:, None], -math.inf)
    p = torch.softmax(s, -1)
    for tile in range(79):
        keys = slice(64 * tile, 64 * tile + 64)
        if p[:, keys].sum(-1).max() <= 2.0 ** -12:
            assert q_scale > 1
            continue
        rest = p.clone()
        rest[:, keys] = 0
        o = rest @ vd / rest.sum(-1, keepdim=True)
        assert ((o.view(-1, 4, 128) - want).abs() > bound).any(), tile


def check_bounds(r, heads, kv_heads, dim, causal=True, seed=0, q_scale=1.0, max_new=None):
    caches = [normal(seed + s, r.num_pages, kv_heads, r.page_size, dim) for s in (11, 12)]
    q = normal(seed + 13, r.total, heads, dim, scale=q_scale)
    plan = r.plan(fa.PagedShape(heads, kv_heads, dim, r.page_size), causal=causal, max_new=max_new)
    out = fa.paged_attention(q, *caches, plan)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    want, bound = bounds(q, *caches, r, causal, r.total if max_new is None else max_new, sms)
    tokens = sum(r.new)
    over = ((out.double() - want).abs() / bound)[:tokens]
    assert over.max() <= 1, f"{over.max().item():.3f} of the bound"
    assert fa.device_status() == (fa.STATUS_OK, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("q_scale", [1.0, 8.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cached,new", [
    ([0, 1, 5, 30, 63, 64, 200], [1] * 7), ([20011], [1]), ([20011], [4]), ([3000, 17, 900], [8, 5, 7]), ([20011], [40]),
    ([700, 0, 100, 4000], [130, 300, 17, 64]), ([0], [600])])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 3), (16, 1)])
def test_attention_within_its_arithmetic(cuda_device, cached, new, heads, kv_heads, dim, q_scale):
    check_bounds(Requests(cached, new, 64, cuda_device), heads, kv_heads, dim, q_scale=q_scale, max_new=max(new))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(16))
def test_mixed_batches_within_their_arithmetic(cuda_device, seed):
    rng = np.random.RandomState(100 + seed)
    dim, page_size = int(rng.choice([64, 128])), int(rng.choice([16, 32, 64, 128, 256]))
    kv_heads = int(rng.choice([1, 2, 3]))
    seqs, most = int(rng.choice([1, 5, 20])), int(rng.choice([1, 4, 9, 40, 200]))
    cached = [int(x) for x in np.exp(rng.uniform(0, np.log(4000), seqs)).astype(int) - 1]
    new = [int(x) for x in rng.randint(1, most + 1, seqs)]
    r = Requests(cached, new, page_size, cuda_device, seed=seed)
    check_bounds(r, kv_heads * int(rng.choice([1, 2, 3, 4, 8])), kv_heads, dim, bool(seed % 4), seed, float(rng.choice([1, 4, 12])),
                 most if seed % 2 else None)
