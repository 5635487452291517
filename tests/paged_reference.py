"""Plain 64-bit forms of the paged-cache operators, and builders of their inputs, for the tests.

Tolerances count roundings: one to bf16 is off by at most 2^-8 of the value (half a step).
"""
import ctypes
import math

import numpy as np
import torch

BF16_HALF_STEP = 2.0 ** -8


class FaPagedPlan(ctypes.Structure):
    """Layout of FaPagedPlan (include/fa_sm100_paged.h)."""
    _fields_ = [(name, ctypes.c_int) for name in (
        "num_seqs", "total_tokens", "max_new", "num_pages", "table_width", "table_stride", "heads", "kv_heads",
        "head_dim", "page_size", "causal", "reserved")] + [(name, ctypes.c_void_p) for name in (
            "query_start", "kv_lens", "positions", "slots", "block_table", "free_cursor", "schedule")]


class Requests:
    """Cached and new lengths, a table of distinct shuffled pages and a free list, on a device."""

    def __init__(self, cached, new, page_size, device, seed=0, spare_pages=3, spare_columns=1, padding=0):
        self.cached, self.new = list(cached), list(new)
        self.page_size, self.padding = page_size, padding
        have = [-(-c // page_size) for c in self.cached]
        want = [-(-(c + n) // page_size) for c, n in zip(self.cached, self.new)]
        self.num_pages = sum(want) + spare_pages
        ids = np.random.RandomState(seed).permutation(self.num_pages).astype(np.int32)
        width = max(want, default=0) + spare_columns
        before = np.full((len(self.cached), width), -7, np.int32)
        after = before.copy()
        at = 0
        for b, h in enumerate(have):
            before[b, :h] = ids[at: at + h]
            at += h
        free = ids[at:]
        after[:] = before
        at = 0
        for b, (h, w) in enumerate(zip(have, want)):
            after[b, h:w] = free[at: at + w - h]
            at += w - h
        self.taken = at
        self.table_after = after
        self.total = sum(self.new) + padding
        as_tensor = lambda a: torch.tensor(a, dtype=torch.int32, device=device)  # noqa: E731
        self.cached_lens, self.new_lens = as_tensor(self.cached), as_tensor(self.new)
        self.block_table = torch.from_numpy(before).to(device)
        self.free_pages = torch.from_numpy(free.copy()).to(device)
        self.device = device

    def plan(self, shape, **how):
        import cuda_fused_attention_b200 as fa
        return fa.paged_plan(self.cached_lens, self.new_lens, self.block_table, self.free_pages, self.total, shape,
                             self.num_pages, **how)

    def expected(self):
        """(query_start, kv_lens, positions, slots) as numpy arrays."""
        start, positions, slots = [0], [], []
        for b, (c, n) in enumerate(zip(self.cached, self.new)):
            start.append(start[-1] + n)
            for i in range(n):
                pos = c + i
                positions.append(pos)
                slots.append(int(self.table_after[b, pos // self.page_size]) * self.page_size + pos % self.page_size)
        pad = self.total - start[-1]
        kv = np.array([c + n for c, n in zip(self.cached, self.new)], np.int32)
        return (np.array(start, np.int32), kv, np.array(positions + [0] * pad, np.int32),
                np.array(slots + [-1] * pad, np.int32))


def normal(seed, *shape, device="cuda", scale=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=device) * scale).to(torch.bfloat16)


def attention(q, k_cache, v_cache, requests, causal=True):
    """(o, a) in 64 bits, [total, heads, D]: the output and sum_j p_j |v_j| / sum_j p_j, which bounds what
    rounding the weights does; zero for padding rows."""
    total, heads, dim = q.shape
    group = heads // k_cache.shape[1]
    out = torch.zeros(total, heads, dim, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    row = 0
    for b, (c, n) in enumerate(zip(requests.cached, requests.new)):
        kv = c + n
        if n == 0:
            continue
        pages = torch.from_numpy(requests.table_after[b, : -(-kv // requests.page_size)].astype(np.int64)).to(q.device)
        for h in range(k_cache.shape[1]):
            k = k_cache[pages, h].reshape(-1, dim)[:kv].double()
            v = v_cache[pages, h].reshape(-1, dim)[:kv].double()
            s = q[row: row + n, h * group: (h + 1) * group].double() @ k.T / math.sqrt(dim)
            if causal:
                hidden = torch.arange(kv, device=q.device) > torch.arange(c, kv, device=q.device)[:, None]
                s.masked_fill_(hidden[:, None], -math.inf)
            p = torch.softmax(s, -1)
            out[row: row + n, h * group: (h + 1) * group] = p @ v
            mag[row: row + n, h * group: (h + 1) * group] = p @ v.abs()
        row += n
    return out, mag


def attention_bound(o, mag):
    """Each weight is rounded to bf16 once (2^-8 of it) and the result once (2^-8 of that). Scores, sums and
    exponentials are in 32 bits: D = 128 products of size about 1 add up with an error below 128 * 2^-24 * 128, in
    the exponent after scaling by 1/sqrt(D) below 2^-13; the remaining 2^-12 covers that and the sums."""
    return BF16_HALF_STEP * (mag + o.abs()) * (1 + 2.0 ** -8) + 2.0 ** -12 * mag + 1e-30


def rotary(x, positions, inv_freq, sections, interleaved, inverse=False):
    """(out, bound) in 64 bits for x [tokens, ..., D] and positions [axes, tokens]."""
    x = x.double()
    pairs = inv_freq.numel()
    angle, lo = [], 0
    for a, n in enumerate(sections):
        angle.append(positions[a].double()[:, None] * inv_freq[lo: lo + n].double())
        lo += n
    angle = torch.cat(angle, 1)
    angle = angle.view(angle.shape[0], *([1] * (x.dim() - 2)), pairs)
    c, s = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
    out, size = x.clone(), torch.zeros_like(x)
    lo_i, hi_i = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs),
                                                                                      slice(pairs, 2 * pairs))
    a, b = x[..., lo_i], x[..., hi_i]
    out[..., lo_i], out[..., hi_i] = a * c - b * s, b * c + a * s
    size[..., lo_i] = size[..., hi_i] = a.abs() + b.abs()
    # One rounding to bf16; the angle's rest, its sine and cosine, two products and a sum in 32 bits: each
    # below 2^-23 of the operands, the rest (up to pi) below 2^-22: 2^-20 in all.
    return out, BF16_HALF_STEP * out.abs() * (1 + 2.0 ** -8) + 2.0 ** -20 * size + 1e-30
