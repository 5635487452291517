"""Paged K/V cache operators: the plan of a step, rotary positions, the append to the
cache, and the attention of the new tokens over it.

A server keeps K and V of many requests in pages of a common cache. One step of it:

    plan = paged_plan(cached_lens, new_lens, block_table, free_pages, total, PagedShape(32, 8, 128, 16), num_pages,
                      max_new=most)
    for every layer:
        q = rotary_append(q, k, v, k_cache, v_cache, plan.positions, plan.slots, inv_freq)
        o = paged_attention(q, k_cache, v_cache, plan)

The plan is built once on the GPU, without a synchronisation, and serves every layer of the
step. The new tokens of all requests are packed along one axis (request after request); rows
behind the last request are padding that no call writes, so a step can be captured into a CUDA
graph at a fixed `total`. Everything goes through the C ABI of include/fa_sm100_paged.h, which
states the formulas; PyTorch only holds memory and streams. Arguments are checked and handed over
by a compiled binding (csrc/paged_binding.cpp), since a small step is bound by its calls. What is wrong with the contents of
device arrays is recorded on the device: device_status() reports it.

No counterpart in the reference, whose attention has contiguous K and V of Q's own length.
"""
import collections
import importlib.util
import os

from . import _lib
from .build import BINDING_PATH

__all__ = ["PagedShape", "PagedPlan", "paged_plan", "paged_attention", "rotary_embed", "rotary_append"]

_PAGE_SIZES = (16, 32, 64, 128, 256)
_ops = None


def _load():
    """The compiled binding, on the library that _lib loads. Raises if either is missing."""
    global _ops
    if _ops is None:
        _lib.load()
        if not os.path.exists(BINDING_PATH):
            raise RuntimeError(f"the binding {BINDING_PATH} is not built; run "
                               "`python -m cuda_fused_attention_b200.build` (or __graft_entry__.build())")
        import torch  # noqa: F401  (the binding needs its libraries)
        spec = importlib.util.spec_from_file_location(__package__ + "._paged", BINDING_PATH)
        ops = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(ops)
        ops.load(_lib.library_path())
        _ops = ops
    return _ops


class PagedShape(collections.namedtuple("PagedShape", "heads kv_heads head_dim page_size")):
    """Heads of the attention and page size of the cache; kv_heads divides heads."""
    __slots__ = ()

    def __new__(cls, heads, kv_heads, head_dim, page_size):
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"kv_heads must divide heads, got {kv_heads} and {heads}")
        if heads // kv_heads > 128:
            raise ValueError(f"at most 128 query heads per K/V head, got {heads // kv_heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if page_size not in _PAGE_SIZES:
            raise ValueError(f"page_size must be one of {_PAGE_SIZES}, got {page_size}")
        return super().__new__(cls, heads, kv_heads, head_dim, page_size)


class PagedPlan:
    """A step's plan: the arrays that paged_plan writes and the calls of the step read.

    query_start [B + 1], kv_lens [B], positions [total_tokens], slots [total_tokens] and
    free_cursor [1] are int32 views of one buffer of the plan; block_table is the caller's.
    """
    __slots__ = ("shape", "num_seqs", "total_tokens", "num_pages", "causal", "block_table", "_struct", "_workspace",
                 "_device", "_buffer", "_views")

    def __init__(self, shape, num_seqs, total_tokens):
        self.shape, self.num_seqs, self.total_tokens = shape, num_seqs, total_tokens
        self._buffer = self._views = None

    def _filled(self, made, block_table, num_pages, causal):
        self._buffer, self._struct, self._workspace, self._device = made
        self.block_table, self.num_pages, self.causal = block_table, num_pages, causal
        return self

    def _view(self, index):
        if self._views is None:
            self._views = _load().split(self._buffer, self.num_seqs, self.total_tokens)
        return self._views[index]

    query_start = property(lambda self: self._view(0))
    kv_lens = property(lambda self: self._view(1))
    positions = property(lambda self: self._view(2))
    slots = property(lambda self: self._view(3))
    free_cursor = property(lambda self: self._view(4))


def _refused(status, what):
    from . import FaError
    raise FaError(status, what)


def paged_plan(cached_lens, new_lens, block_table, free_pages, total_tokens, shape, num_pages, free_cursor=None,
               causal=True, max_new=None, plan=None, stream=None):
    """Block tables, slots, positions and schedule of a step, built on the GPU.

    cached_lens, new_lens: int32 [B], tokens that each request has in the cache and brings now.
    block_table: int32 [B, W], extended in place by the pages that the new tokens need (it shares memory
    with no input); they are free_pages[free_cursor + k], handed out in request order, and
    plan.free_cursor is where the next step begins (free_cursor: int32 [1], default 0). Where the list has
    ended the table gets -1: tokens of such a page have slot -1, are not written, and count as zeros in
    attention; device_status() reports it. total_tokens: rows of the packed token axis, at least the sum
    of new_lens. num_pages: pages of the cache. max_new: an upper bound of new_lens (default
    total_tokens). It decides which kernels paged_attention launches, so give a tight one: a decode step of
    32 requests with 4 heads per K/V head takes 52 us with max_new=1 and 56 without, 16 requests of 5 to 8
    drafted tokens 62 with max_new=8 and 72 without.
    plan: an earlier plan of the same B, total_tokens and shape whose buffers are written again
    (for CUDA graphs); its own arrays cannot be inputs then: copy kv_lens and free_cursor to the next
    step's tensors first. A captured attention call keeps the causal, max_new and table of the plan that it
    saw; replayed after the plan was written with others its output is of no use, which device_status()
    reports (STATUS_BAD_REQUEST). Returns the PagedPlan.
    """
    ops = _ops or _load()
    seqs = cached_lens.numel()
    if plan is None:
        plan = PagedPlan(shape, seqs, total_tokens)
    elif (plan.shape, plan.num_seqs, plan.total_tokens) != (shape, seqs, total_tokens):
        raise ValueError("plan was made for other sizes or another device")
    made = ops.plan(cached_lens, new_lens, block_table, free_pages, total_tokens, shape, num_pages, free_cursor, causal,
                    max_new, plan._buffer, stream)
    if made.__class__ is int:
        _refused(made, "fa_sm100_paged_plan")
    return plan._filled(made, block_table, num_pages, causal)


def rotary_embed(x, positions, inv_freq, sections=None, interleaved=False, inverse=False, out=None, stream=None):
    """Rotary positions over x [batch, heads, seq_len, head_dim] (bf16, head_dim 64 or 128).

    positions: int32 [seq_len], [axes, seq_len] or [axes, batch, seq_len]. inv_freq: float32, one
    frequency per pair (rotary_dim / 2 of them; elements from rotary_dim on are copied). sections:
    how many pairs take each axis, in order (default: all take the one axis). interleaved: pairs are
    neighbours (2p, 2p + 1) instead of (p, p + rotary_dim / 2). inverse: the opposite rotation, which
    is also the gradient: dL/dx = rotary_embed(dL/dout, ..., inverse=True). out may be x.
    """
    out = (_ops or _load()).embed(x, positions, inv_freq, sections, interleaved, inverse, out, stream)
    if out.__class__ is int:
        _refused(out, "fa_sm100_rotary")
    return out


def rotary_append(q, k, v, k_cache, v_cache, positions, slots, inv_freq, sections=None, interleaved=False, out=None,
                  stream=None):
    """Rotary positions of a step's new tokens, K and V written to the cache.

    q [tokens, heads, D], k and v [tokens, kv_heads, D]: bf16, rows of a fused projection's output
    may be passed as they are. q is rotated into out (returned; may be q itself), k into k_cache and v
    copied into v_cache at slots[token]; caches are [num_pages, kv_heads, page_size, D] in any stride
    order with contiguous rows. positions: int32 [tokens] or [axes, tokens]. A token with a negative
    slot (padding) is skipped, its row of out included. Slots must be distinct, and the caches must not
    share memory. inv_freq, sections,
    interleaved: as in rotary_embed.
    """
    out = (_ops or _load()).append(q, k, v, k_cache, v_cache, positions, slots, inv_freq, sections, interleaved, out,
                                   stream)
    if out.__class__ is int:
        _refused(out, "fa_sm100_rotary_append")
    return out


def paged_attention(q, k_cache, v_cache, plan, out=None, stream=None):
    """Attention of the plan's new tokens over the cache, scale 1/sqrt(head_dim).

    q: bf16 [plan.total_tokens, heads, head_dim], rows of a fused projection's output may be passed as
    they are. k_cache, v_cache: [plan.num_pages, kv_heads, page_size, head_dim] in any stride order with
    contiguous rows; the new tokens' K and V are in them, and V is finite. Returns out [total_tokens, heads,
    head_dim] (out may be q); padding rows are not written.

    Scores, weights and sums are in 32 bits. For the product with V a weight is rounded to bf16 in requests of
    more than 16 query rows (new tokens times heads per K/V head; 32 where max_new allows no request
    more), as in attention_forward: the result is off by 0.0024 of its size, against 0.0017 where it alone is
    rounded. Below that a weight keeps 16 bits. So the last bits of a request's rows depend on max_new, and on
    how the step's work is shared out among the GPU's multiprocessors: on the other requests of the step.
    """
    out = (_ops or _load()).attention(q, k_cache, v_cache, plan._struct, plan._workspace, plan._device, out, stream)
    if out.__class__ is int:
        _refused(out, "fa_sm100_paged_fwd")
    return out
