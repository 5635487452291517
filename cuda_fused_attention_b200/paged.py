"""Paged K/V cache operators: the plan of a step, rotary positions, the append to the
cache, and the attention of the new tokens over it.

A server keeps K and V of many requests in pages of a common cache. One step of it:

    plan = paged_plan(cached_lens, new_lens, block_table, free_pages, total, PagedShape(32, 8, 128, 16), num_pages)
    for every layer:
        q = rotary_append(q, k, v, k_cache, v_cache, plan.positions, plan.slots, inv_freq)
        o = paged_attention(q, k_cache, v_cache, plan)

The plan is built once on the GPU, without a synchronisation, and serves every layer of the
step. The new tokens of all requests are packed along one axis (request after request); rows
behind the last request are padding that no call writes, so a step can be captured into a CUDA
graph at a fixed `total`. Everything goes through the C ABI of include/fa_sm100_paged.h, which
states the formulas; PyTorch only holds memory and streams. What is wrong with the contents of
device arrays is recorded on the device: device_status() reports it.

No counterpart in the reference, whose attention has contiguous K and V of Q's own length.
"""
import contextlib
import functools
import struct
from dataclasses import dataclass

from . import _lib

__all__ = ["PagedShape", "PagedPlan", "paged_plan", "paged_attention", "rotary_embed", "rotary_append"]

_PAGE_SIZES = (16, 32, 64, 128, 256)
_INT_MAX = 2 ** 31 - 1

# Small steps are bound by what the host does, so the calls below check their arguments in few
# steps, look closer only at what those do not pass, and hand structs and strides to the C ABI
# as packed bytes (a ctypes array costs several times as much).
_PLAN = struct.Struct("12i7P")          # FaPagedPlan
_STRIDES = {n: struct.Struct(f"{n}q").pack for n in (2, 3, 10, 14)}


@dataclass(frozen=True)
class PagedShape:
    """Heads of the attention and page size of the cache; kv_heads divides heads."""
    heads: int
    kv_heads: int
    head_dim: int
    page_size: int

    def __post_init__(self):
        if self.heads < 1 or self.kv_heads < 1 or self.heads % self.kv_heads:
            raise ValueError(f"kv_heads must divide heads, got {self.kv_heads} and {self.heads}")
        if self.heads // self.kv_heads > 128:
            raise ValueError(f"at most 128 query heads per K/V head, got {self.heads // self.kv_heads}")
        if self.head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {self.head_dim}")
        if self.page_size not in _PAGE_SIZES:
            raise ValueError(f"page_size must be one of {_PAGE_SIZES}, got {self.page_size}")


class PagedPlan:
    """A step's plan: the arrays that paged_plan writes and the calls of the step read.

    query_start [B + 1], kv_lens [B], positions [total_tokens], slots [total_tokens] and
    free_cursor [1] are int32 views of one buffer of the plan; block_table is the caller's.
    """

    def __init__(self, num_seqs, total_tokens, shape, like):
        self.shape = shape
        self.num_seqs = num_seqs
        self.total_tokens = total_tokens
        self.device_index = like.get_device()
        self.block_table = None
        self.num_pages = 0
        self.causal = True
        # [schedule, as 64-bit words][query_start][kv_lens][positions][slots][free_cursor]
        self._sizes = (4 * (num_seqs + 1), num_seqs + 1, num_seqs, total_tokens, total_tokens, 1)
        self._buffer = like.new_empty(sum(self._sizes))
        self._views = None
        self.c = b""                    # FaPagedPlan
        self._workspace = 0             # bytes of workspace that paged_attention needs

    def _fill(self, block_table, width, stride, num_pages, max_new, causal):
        self.block_table, self.num_pages, self.causal = block_table, num_pages, causal
        shape, seqs, tokens = self.shape, self.num_seqs, self.total_tokens
        schedule = self._buffer.data_ptr()
        start = schedule + 16 * (seqs + 1)
        lens = start + 4 * (seqs + 1)
        positions = lens + 4 * seqs
        slots = positions + 4 * tokens
        self.c = _PLAN.pack(seqs, tokens, max_new, num_pages, width, stride, shape.heads, shape.kv_heads, shape.head_dim,
                            shape.page_size, causal, 0, start, lens, positions, slots, block_table.data_ptr(),
                            slots + 4 * tokens, schedule)

    def _view(self, index):
        if self._views is None:
            self._views = self._buffer.split_with_sizes(self._sizes)
        return self._views[index]

    query_start = property(lambda self: self._view(1))
    kv_lens = property(lambda self: self._view(2))
    positions = property(lambda self: self._view(3))
    slots = property(lambda self: self._view(4))
    free_cursor = property(lambda self: self._view(5))


def _check(status, what):
    if status:
        from . import FaError
        raise FaError(status, what)


def _device_error(**tensors):
    """Raises for tensors that are not all on one CUDA device."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name} is on {t.device}, other arguments on {device}")
    raise ValueError("arguments are on different devices")


@functools.lru_cache(maxsize=None)
def _raw_stream():
    """The function that gives a device's current stream as an integer."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw if raw is not None else lambda index: torch.cuda.current_stream(index).cuda_stream


@contextlib.contextmanager
def _elsewhere(index, stream):
    """Make device `index` current and yield the stream's handle. What is allocated inside belongs to that
    stream, so that its memory is not handed to another one while the call still uses it."""
    import torch
    with torch.cuda.device(index):
        if stream is None:
            yield _raw_stream()(index)
            return
        handle = stream if isinstance(stream, int) else int(stream.cuda_stream)
        if handle == _raw_stream()(index):
            yield handle
            return
        if not isinstance(stream, torch.cuda.Stream):
            stream = (torch.cuda.ExternalStream(handle, device=index) if handle
                      else torch.cuda.default_stream(index))
        with torch.cuda.stream(stream):
            yield handle


def _launch(call, index, stream, *args):
    """call(stream handle, *args) with device `index` current."""
    import torch
    if stream is None and torch.cuda.current_device() == index:
        return call(_raw_stream()(index), *args)
    with _elsewhere(index, stream) as handle:
        return call(handle, *args)


def _int32(name, t, dims):
    import torch
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimension(s), got {t.dim()}")


def _vector(name, t, size=None):
    _int32(name, t, 1)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if size is not None and t.numel() != size:
        raise ValueError(f"{name} must have {size} elements, got {t.numel()}")


def _rows(name, t, shape):
    """A bf16 tensor of this shape with contiguous rows on 16-byte boundaries; its strides without the last."""
    import torch
    strides = t.stride()
    if t.dtype is torch.bfloat16 and t.shape == shape and strides[-1] == 1 and not t.data_ptr() & 15:
        strides = strides[:-1]
        if len(strides) == 3:
            if not (strides[0] | strides[1] | strides[2]) & 7:
                return strides
        elif not (strides[0] | strides[1]) & 7:
            return strides
    if t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    # The stride of a dimension with one element is never used.
    strides = tuple(s if n > 1 else shape[-1] for s, n in zip(t.stride()[:-1], shape))
    for s in strides:
        if s % 8:
            raise ValueError(f"{name} has rows off 16-byte boundaries (strides {list(t.stride())})")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must start on a 16-byte boundary")
    return strides


def _written(name, t):
    """An output (or cache) whose elements share no memory."""
    if t.is_contiguous():
        return t
    span = sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1)
    reach = 1
    for s, n in span:
        if s < reach:
            raise ValueError(f"{name} has elements that share memory (strides {list(t.stride())})")
        reach = s * (n - 1) + reach
    return t


def paged_plan(cached_lens, new_lens, block_table, free_pages, total_tokens, shape, num_pages, free_cursor=None,
               causal=True, max_new=None, plan=None, stream=None):
    """Block tables, slots, positions and schedule of a step, built on the GPU.

    cached_lens, new_lens: int32 [B], tokens that each request has in the cache and brings now.
    block_table: int32 [B, W], extended in place by the pages that the new tokens need; they are
    free_pages[free_cursor + k], handed out in request order, and plan.free_cursor is where the
    next step begins (free_cursor: int32 [1], default 0). total_tokens: rows of the packed token
    axis, at least the sum of new_lens. num_pages: pages of the cache. max_new: an upper bound of
    new_lens (default total_tokens); a tight one lets calls leave out kernels that have no work.
    plan: an earlier plan of the same B, total_tokens and shape whose buffers are written again
    (for CUDA graphs). Returns the PagedPlan.
    """
    import torch
    i32 = torch.int32
    num_seqs = cached_lens.numel()
    width = block_table.shape[-1] if block_table.dim() else 0
    if not (cached_lens.dtype is i32 and new_lens.dtype is i32 and block_table.dtype is i32 and free_pages.dtype is i32
            and cached_lens.shape == new_lens.shape == (num_seqs,) and block_table.shape == (num_seqs, width)
            and free_pages.dim() == 1 and cached_lens.is_contiguous() and new_lens.is_contiguous()
            and block_table.is_contiguous() and free_pages.is_contiguous()):
        _vector("cached_lens", cached_lens)
        _vector("new_lens", new_lens, num_seqs)
        _vector("free_pages", free_pages)
        _int32("block_table", block_table, 2)
        if block_table.shape[0] != num_seqs:
            raise ValueError(f"block_table must have {num_seqs} rows, got {block_table.shape[0]}")
        if width > 1 and block_table.stride(1) != 1:
            raise ValueError("block_table must be contiguous in its last dimension")
    stride = block_table.stride(0) if num_seqs > 1 else width
    if stride < width:
        raise ValueError("block_table has rows that share memory")
    if free_cursor is not None:
        _vector("free_cursor", free_cursor, 1)
    total_tokens, num_pages = int(total_tokens), int(num_pages)
    max_new = total_tokens if max_new is None else int(max_new)
    if total_tokens < 0 or num_pages < 0 or max_new < 0:
        raise ValueError("total_tokens, num_pages and max_new must not be negative")
    if total_tokens > _INT_MAX // 2 or max_new > _INT_MAX:
        raise ValueError("total_tokens must be below 2^30")
    if num_pages * shape.page_size > _INT_MAX or width * shape.page_size > _INT_MAX:
        raise ValueError("a cache, and a table row, must hold fewer than 2^31 tokens")
    index = cached_lens.get_device()
    if index < 0 or not (index == new_lens.get_device() == block_table.get_device() == free_pages.get_device()) or (
            free_cursor is not None and free_cursor.get_device() != index):
        _device_error(cached_lens=cached_lens, new_lens=new_lens, block_table=block_table, free_pages=free_pages,
                      free_cursor=free_cursor)
    if plan is not None and (plan.num_seqs, plan.total_tokens, plan.shape, plan.device_index) != (
            num_seqs, total_tokens, shape, index):
        raise ValueError("plan was made for other sizes or another device")
    return _launch(_plan, index, stream, cached_lens, new_lens, block_table, free_pages, total_tokens, shape, num_pages,
                   free_cursor, causal, max_new, plan, width, stride)


def _plan(handle, cached_lens, new_lens, block_table, free_pages, total_tokens, shape, num_pages, free_cursor, causal,
          max_new, plan, width, stride):
    if plan is None:
        plan = PagedPlan(cached_lens.numel(), total_tokens, shape, cached_lens)
    plan._fill(block_table, width, stride, num_pages, max_new, 1 if causal else 0)
    lib = _lib.load()
    status = lib.fa_sm100_paged_plan(plan.c, cached_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(),
                                     free_pages.numel(), free_cursor.data_ptr() if free_cursor is not None else None,
                                     handle)
    if status:
        _check(status, "fa_sm100_paged_plan")
    plan._workspace = lib.fa_sm100_paged_workspace_bytes(plan.c)
    return plan


@functools.lru_cache(maxsize=64)
def _sections(sections, pairs):
    """(sections, the same packed) for a number of pairs."""
    sections = (pairs,) if sections is None else tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections must be 1 to 4 counts that add up to {pairs}, got {sections}")
    return sections, struct.pack(f"{len(sections)}i", *sections)


def _frequencies(inv_freq, head_dim, sections):
    """(rotary_dim, axes, packed sections)."""
    import torch
    pairs = inv_freq.numel()
    if inv_freq.dtype is not torch.float32:
        raise TypeError(f"inv_freq must be float32, got {inv_freq.dtype}")
    if inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous vector")
    if pairs == 0 or pairs % 8 or 2 * pairs > head_dim:
        raise ValueError(f"inv_freq must have a multiple of 8 and at most {head_dim // 2} elements, got {pairs}")
    if sections is not None and not isinstance(sections, tuple):
        sections = tuple(sections)
    counts, packed = _sections(sections, pairs)
    return 2 * pairs, len(counts), packed


def rotary_embed(x, positions, inv_freq, sections=None, interleaved=False, inverse=False, out=None, stream=None):
    """Rotary positions over x [batch, heads, seq_len, head_dim] (bf16, head_dim 64 or 128).

    positions: int32 [seq_len], [axes, seq_len] or [axes, batch, seq_len]. inv_freq: float32, one
    frequency per pair (rotary_dim / 2 of them; elements from rotary_dim on are copied). sections:
    how many pairs take each axis, in order (default: all take the one axis). interleaved: pairs are
    neighbours (2p, 2p + 1) instead of (p, p + rotary_dim / 2). inverse: the opposite rotation, which
    is also the gradient: dL/dx = rotary_embed(dL/dout, ..., inverse=True). out may be x.
    """
    import torch
    shape = x.shape
    if len(shape) != 4:
        raise ValueError("x must be [batch, heads, seq_len, head_dim]")
    batch, heads, tokens, dim = shape
    if dim != 128 and dim != 64:
        raise ValueError(f"head_dim must be 64 or 128, got {dim}")
    x_strides = _rows("x", x, shape)
    rotary_dim, axes, packed = _frequencies(inv_freq, dim, sections)
    at, step = positions.shape, positions.stride()
    if positions.dtype is not torch.int32 or not 1 <= len(at) <= 3:
        _int32("positions", positions, 2)
    if len(at) == 1:
        at, step = (1, *at), (0, *step)
    if at != ((axes, tokens) if len(at) == 2 else (axes, batch, tokens)):
        raise ValueError(f"positions must be {[axes, tokens]} or {[axes, batch, tokens]}, got {list(positions.shape)}")
    if tokens > 1 and step[-1] != 1:
        raise ValueError("positions must be contiguous in their last dimension")
    index = x.get_device()
    if index < 0 or not (index == positions.get_device() == inv_freq.get_device()) or (
            out is not None and out.get_device() != index):
        _device_error(x=x, positions=positions, inv_freq=inv_freq, out=out)
    return _launch(_embed, index, stream, x, x_strides, positions, step[0], step[1] if len(at) == 3 else 0, inv_freq,
                   rotary_dim, axes, packed, interleaved, inverse, out)


def _embed(handle, x, x_strides, positions, axis_stride, batch_stride, inv_freq, rotary_dim, axes, packed, interleaved,
           inverse, out):
    shape = x.shape
    if out is None:
        out = x.new_empty(shape)
    pack = _STRIDES[3]
    status = _lib.load().fa_sm100_rotary(
        x.data_ptr(), pack(*x_strides), out.data_ptr(), pack(*_rows("out", _written("out", out), shape)), *shape,
        positions.data_ptr(), _STRIDES[2](axis_stride, batch_stride), inv_freq.data_ptr(), rotary_dim, packed, axes,
        1 if interleaved else 0, 1 if inverse else 0, handle)
    if status:
        _check(status, "fa_sm100_rotary")
    return out


def rotary_append(q, k, v, k_cache, v_cache, positions, slots, inv_freq, sections=None, interleaved=False, out=None,
                  stream=None):
    """Rotary positions of a step's new tokens, K and V written to the cache.

    q [tokens, heads, D], k and v [tokens, kv_heads, D]: bf16, rows of a fused projection's output
    may be passed as they are. q is rotated into out (returned; may be q itself), k into k_cache and v
    copied into v_cache at slots[token]; caches are [num_pages, kv_heads, page_size, D] in any stride
    order with contiguous rows. positions: int32 [tokens] or [axes, tokens]. A token with a negative
    slot (padding) is skipped, its row of out included. Slots must be distinct. inv_freq, sections,
    interleaved: as in rotary_embed.
    """
    import torch
    cache_shape = k_cache.shape
    if len(cache_shape) != 4:
        raise ValueError("k_cache must be [num_pages, kv_heads, page_size, head_dim]")
    num_pages, kv_heads, page_size, dim = cache_shape
    rows = q.shape
    if len(rows) != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    tokens = rows[0]
    if dim != 128 and dim != 64:
        raise ValueError(f"head_dim must be 64 or 128, got {dim}")
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"page_size must be one of {_PAGE_SIZES}, got {page_size}")
    if num_pages * page_size > _INT_MAX:
        raise ValueError("a cache must hold fewer than 2^31 tokens")
    if rows[2] != dim:
        raise ValueError(f"q must have {dim} elements per head, got {rows[2]}")
    kv_rows = (tokens, kv_heads, dim)
    strides = (*_rows("k", k, kv_rows), *_rows("v", v, kv_rows),
               *_rows("k_cache", _written("k_cache", k_cache), cache_shape),
               *_rows("v_cache", _written("v_cache", v_cache), cache_shape))
    q_strides = _rows("q", q, rows)
    rotary_dim, axes, packed = _frequencies(inv_freq, dim, sections)
    at, step = positions.shape, positions.stride()
    if positions.dtype is not torch.int32 or not 1 <= len(at) <= 2:
        _int32("positions", positions, 2)
    if len(at) == 1:
        at, step = (1, *at), (0, *step)
    if at != (axes, tokens):
        raise ValueError(f"positions must be {[axes, tokens]}, got {list(positions.shape)}")
    if tokens > 1 and step[1] != 1:
        raise ValueError("positions must be contiguous in their last dimension")
    if not (slots.dtype is torch.int32 and slots.shape == (tokens,) and slots.is_contiguous()):
        _vector("slots", slots, tokens)
    index = q.get_device()
    if index < 0 or not (index == k.get_device() == v.get_device() == k_cache.get_device() == v_cache.get_device()
                         == positions.get_device() == slots.get_device() == inv_freq.get_device()) or (
            out is not None and out.get_device() != index):
        _device_error(q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache, positions=positions, slots=slots,
                      inv_freq=inv_freq, out=out)
    return _launch(_append, index, stream, q, k, v, k_cache, v_cache, q_strides, strides, positions, step[0], slots,
                   inv_freq, rotary_dim, axes, packed, interleaved, out)


def _append(handle, q, k, v, k_cache, v_cache, q_strides, strides, positions, axis_stride, slots, inv_freq, rotary_dim,
            axes, packed, interleaved, out):
    rows = q.shape
    if out is None:
        out = q.new_empty(rows)
    num_pages, kv_heads, page_size, dim = k_cache.shape
    status = _lib.load().fa_sm100_rotary_append(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        _STRIDES[14](*q_strides, *_rows("out", _written("out", out), rows), *strides), rows[0], rows[1], kv_heads, dim,
        page_size, num_pages, positions.data_ptr(), axis_stride, slots.data_ptr(), inv_freq.data_ptr(), rotary_dim,
        packed, axes, 1 if interleaved else 0, handle)
    if status:
        _check(status, "fa_sm100_rotary_append")
    return out


def paged_attention(q, k_cache, v_cache, plan, out=None, stream=None):
    """Attention of the plan's new tokens over the cache, scale 1/sqrt(head_dim).

    q: bf16 [plan.total_tokens, heads, head_dim], rows of a fused projection's output may be passed as
    they are. k_cache, v_cache: [plan.num_pages, kv_heads, page_size, head_dim] in any stride order with
    contiguous rows; the new tokens' K and V are in them. Returns out [total_tokens, heads, head_dim]
    (out may be q); padding rows are not written.
    """
    shape = plan.shape
    rows = (plan.total_tokens, shape.heads, shape.head_dim)
    cache = (plan.num_pages, shape.kv_heads, shape.page_size, shape.head_dim)
    q_strides = _rows("q", q, rows)
    strides = (*_rows("k_cache", k_cache, cache), *_rows("v_cache", v_cache, cache))
    index = plan.device_index
    if index < 0 or not (index == q.get_device() == k_cache.get_device() == v_cache.get_device()) or (
            out is not None and out.get_device() != index):
        _device_error(plan=plan._buffer, q=q, k_cache=k_cache, v_cache=v_cache, out=out)
    return _launch(_attention, index, stream, q, k_cache, v_cache, plan, q_strides, strides, rows, out)


def _attention(handle, q, k_cache, v_cache, plan, q_strides, strides, rows, out):
    if out is None:
        out = q.new_empty(rows)
    size = plan._workspace
    workspace = q.new_empty((size + 1) // 2) if size else None
    status = _lib.load().fa_sm100_paged_fwd(
        plan.c, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
        _STRIDES[10](*q_strides, *_rows("out", _written("out", out), rows), *strides),
        workspace.data_ptr() if size else None, size, handle)
    if status:
        _check(status, "fa_sm100_paged_fwd")
    return out
