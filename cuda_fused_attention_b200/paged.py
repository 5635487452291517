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
import ctypes
from dataclasses import dataclass

from . import _lib

__all__ = ["PagedShape", "PagedPlan", "paged_plan", "paged_attention", "rotary_embed", "rotary_append"]

_PAGE_SIZES = (16, 32, 64, 128, 256)
_INT_MAX = 2 ** 31 - 1


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

    def __init__(self, num_seqs, total_tokens, shape, device):
        import torch
        self.shape = shape
        self.num_seqs = num_seqs
        self.total_tokens = total_tokens
        self.device = device
        self.block_table = None
        self.causal = True
        schedule = 2 * (num_seqs + 1)
        words = (num_seqs + 1) + num_seqs + 2 * total_tokens + 1
        self._buffer = torch.empty(schedule + (words + 1) // 2, dtype=torch.int64, device=device)
        self._views = None
        base = int(self._buffer.data_ptr())
        at = base + 8 * schedule
        c = self.c = _lib.FaPagedPlan()
        c.num_seqs, c.total_tokens = num_seqs, total_tokens
        c.heads, c.kv_heads, c.head_dim, c.page_size = shape.heads, shape.kv_heads, shape.head_dim, shape.page_size
        c.schedule = base
        c.query_start = at
        c.kv_lens = at + 4 * (num_seqs + 1)
        c.positions = c.kv_lens + 4 * num_seqs
        c.slots = c.positions + 4 * total_tokens
        c.free_cursor = c.slots + 4 * total_tokens
        self._ref = ctypes.byref(c)

    def _split(self):
        if self._views is None:
            import torch
            b, t = self.num_seqs, self.total_tokens
            words = self._buffer.view(torch.int32)[4 * (b + 1):]
            self._views = words[: 2 * b + 2 + 2 * t].split([b + 1, b, t, t, 1])
        return self._views

    query_start = property(lambda self: self._split()[0])
    kv_lens = property(lambda self: self._split()[1])
    positions = property(lambda self: self._split()[2])
    slots = property(lambda self: self._split()[3])
    free_cursor = property(lambda self: self._split()[4])


def _check(status, what):
    if status:
        from . import FaError
        raise FaError(status, what)


def _device(**tensors):
    """The one CUDA device of the tensors."""
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
    return device


@contextlib.contextmanager
def _launching(device, stream):
    """Make `device` current and yield the stream's handle. What is allocated inside belongs to that
    stream, so that its memory is not handed to another one while the call still uses it."""
    import torch
    with contextlib.ExitStack() as stack:
        if torch.cuda.current_device() != device.index:
            stack.enter_context(torch.cuda.device(device))
        if stream is None:
            handle = int(torch.cuda.current_stream(device).cuda_stream)
        else:
            handle = stream if isinstance(stream, int) else int(stream.cuda_stream)
            if handle != int(torch.cuda.current_stream(device).cuda_stream):
                stack.enter_context(torch.cuda.stream(
                    torch.cuda.ExternalStream(handle, device=device) if handle
                    else torch.cuda.default_stream(device)))
        yield handle


def _int32(name, t, dims):
    import torch
    if t.dtype != torch.int32:
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
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    strides = t.stride()
    if strides[-1] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    # The stride of a dimension with one element is never used.
    strides = [s if n > 1 else shape[-1] for s, n in zip(strides[:-1], shape)]
    for s in strides:
        if s % 8:
            raise ValueError(f"{name} has rows off 16-byte boundaries (strides {list(t.stride())})")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must start on a 16-byte boundary")
    return strides


def _written(name, t):
    """An output (or cache) whose elements share no memory."""
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
    _vector("cached_lens", cached_lens)
    num_seqs = cached_lens.numel()
    _vector("new_lens", new_lens, num_seqs)
    _vector("free_pages", free_pages)
    _int32("block_table", block_table, 2)
    if block_table.shape[0] != num_seqs:
        raise ValueError(f"block_table must have {num_seqs} rows, got {block_table.shape[0]}")
    width = block_table.shape[1]
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
    device = _device(cached_lens=cached_lens, new_lens=new_lens, block_table=block_table, free_pages=free_pages,
                     free_cursor=free_cursor)
    with _launching(device, stream) as handle:
        if plan is None:
            plan = PagedPlan(num_seqs, total_tokens, shape, device)
        elif (plan.num_seqs, plan.total_tokens, plan.shape, plan.device) != (num_seqs, total_tokens, shape, device):
            raise ValueError("plan was made for other sizes or another device")
        plan.block_table = block_table
        plan.causal = bool(causal)
        c = plan.c
        c.max_new, c.num_pages, c.causal = max_new, num_pages, 1 if causal else 0
        c.table_width, c.table_stride = width, stride
        c.block_table = block_table.data_ptr()
        status = _lib.load().fa_sm100_paged_plan(plan._ref, cached_lens.data_ptr(), new_lens.data_ptr(),
                                                 free_pages.data_ptr(), free_pages.numel(),
                                                 free_cursor.data_ptr() if free_cursor is not None else None, handle)
    _check(status, "fa_sm100_paged_plan")
    return plan


def _frequencies(inv_freq, head_dim, sections):
    import torch
    if inv_freq.dtype != torch.float32:
        raise TypeError(f"inv_freq must be float32, got {inv_freq.dtype}")
    if inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous vector")
    pairs = inv_freq.numel()
    if pairs == 0 or pairs % 8 or 2 * pairs > head_dim:
        raise ValueError(f"inv_freq must have a multiple of 8 and at most {head_dim // 2} elements, got {pairs}")
    sections = (pairs,) if sections is None else tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError(f"sections must be 1 to 4 counts that add up to {pairs}, got {sections}")
    return 2 * pairs, sections


def rotary_embed(x, positions, inv_freq, sections=None, interleaved=False, inverse=False, out=None, stream=None):
    """Rotary positions over x [batch, heads, seq_len, head_dim] (bf16, head_dim 64 or 128).

    positions: int32 [seq_len], [axes, seq_len] or [axes, batch, seq_len]. inv_freq: float32, one
    frequency per pair (rotary_dim / 2 of them; elements from rotary_dim on are copied). sections:
    how many pairs take each axis, in order (default: all take the one axis). interleaved: pairs are
    neighbours (2p, 2p + 1) instead of (p, p + rotary_dim / 2). inverse: the opposite rotation, which
    is also the gradient: dL/dx = rotary_embed(dL/dout, ..., inverse=True). out may be x.
    """
    import torch
    if x.dim() != 4:
        raise ValueError("x must be [batch, heads, seq_len, head_dim]")
    shape = tuple(x.shape)
    batch, heads, tokens, dim = shape
    if dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {dim}")
    x_strides = _rows("x", x, shape)
    rotary_dim, sections = _frequencies(inv_freq, dim, sections)
    if positions.dim() == 1:
        positions = positions[None]
    _int32("positions", positions, 3 if positions.dim() == 3 else 2)
    expected = (len(sections), tokens) if positions.dim() == 2 else (len(sections), batch, tokens)
    if tuple(positions.shape) != expected:
        raise ValueError(f"positions must be {list(expected)}, got {list(positions.shape)}")
    if tokens > 1 and positions.stride(-1) != 1:
        raise ValueError("positions must be contiguous in their last dimension")
    strides = (positions.stride(0), positions.stride(1) if positions.dim() == 3 else 0)
    device = _device(x=x, positions=positions, inv_freq=inv_freq, out=out)
    with _launching(device, stream) as handle:
        if out is None:
            out = torch.empty(shape, dtype=x.dtype, device=device)
        out_strides = _rows("out", _written("out", out), shape)
        status = _lib.load().fa_sm100_rotary(
            x.data_ptr(), (ctypes.c_longlong * 3)(*x_strides), out.data_ptr(), (ctypes.c_longlong * 3)(*out_strides),
            batch, heads, tokens, dim, positions.data_ptr(), (ctypes.c_longlong * 2)(*strides), inv_freq.data_ptr(),
            rotary_dim, (ctypes.c_int * len(sections))(*sections), len(sections), 1 if interleaved else 0,
            1 if inverse else 0, handle)
    _check(status, "fa_sm100_rotary")
    return out


def _caches(k_cache, v_cache):
    if k_cache.dim() != 4:
        raise ValueError("k_cache must be [num_pages, kv_heads, page_size, head_dim]")
    shape = tuple(k_cache.shape)
    return shape, _rows("k_cache", k_cache, shape), _rows("v_cache", v_cache, shape)


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
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be [tokens, heads, head_dim]")
    cache_shape, k_cache_strides, v_cache_strides = _caches(_written("k_cache", k_cache), _written("v_cache", v_cache))
    num_pages, kv_heads, page_size, dim = cache_shape
    tokens, heads = q.shape[0], q.shape[1]
    if dim not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {dim}")
    if page_size not in _PAGE_SIZES:
        raise ValueError(f"page_size must be one of {_PAGE_SIZES}, got {page_size}")
    if num_pages * page_size > _INT_MAX:
        raise ValueError("a cache must hold fewer than 2^31 tokens")
    q_strides = _rows("q", q, (tokens, heads, dim))
    k_strides = _rows("k", k, (tokens, kv_heads, dim))
    v_strides = _rows("v", v, (tokens, kv_heads, dim))
    rotary_dim, sections = _frequencies(inv_freq, dim, sections)
    if positions.dim() == 1:
        positions = positions[None]
    _int32("positions", positions, 2)
    if tuple(positions.shape) != (len(sections), tokens):
        raise ValueError(f"positions must be {[len(sections), tokens]}, got {list(positions.shape)}")
    if tokens > 1 and positions.stride(1) != 1:
        raise ValueError("positions must be contiguous in their last dimension")
    _vector("slots", slots, tokens)
    device = _device(q=q, k=k, v=v, k_cache=k_cache, v_cache=v_cache, positions=positions, slots=slots,
                     inv_freq=inv_freq, out=out)
    with _launching(device, stream) as handle:
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
        out_strides = _rows("out", _written("out", out), (tokens, heads, dim))
        strides = (*q_strides, *out_strides, *k_strides, *v_strides, *k_cache_strides, *v_cache_strides)
        status = _lib.load().fa_sm100_rotary_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            (ctypes.c_longlong * 14)(*strides), tokens, heads, kv_heads, dim, page_size, num_pages,
            positions.data_ptr(), positions.stride(0), slots.data_ptr(), inv_freq.data_ptr(), rotary_dim,
            (ctypes.c_int * len(sections))(*sections), len(sections), 1 if interleaved else 0, handle)
    _check(status, "fa_sm100_rotary_append")
    return out


def paged_attention(q, k_cache, v_cache, plan, out=None, stream=None):
    """Attention of the plan's new tokens over the cache, scale 1/sqrt(head_dim).

    q: bf16 [plan.total_tokens, heads, head_dim], rows of a fused projection's output may be passed as
    they are. k_cache, v_cache: [plan.num_pages, kv_heads, page_size, head_dim] in any stride order with
    contiguous rows; the new tokens' K and V are in them. Returns out [total_tokens, heads, head_dim]
    (out may be q); padding rows are not written.
    """
    import torch
    shape, c = plan.shape, plan.c
    rows = (plan.total_tokens, shape.heads, shape.head_dim)
    q_strides = _rows("q", q, rows)
    cache = (c.num_pages, shape.kv_heads, shape.page_size, shape.head_dim)
    k_strides = _rows("k_cache", k_cache, cache)
    v_strides = _rows("v_cache", v_cache, cache)
    device = _device(q=q, k_cache=k_cache, v_cache=v_cache, out=out)
    if device != plan.device:
        raise ValueError(f"plan is on {plan.device}, other arguments on {device}")
    lib = _lib.load()
    with _launching(device, stream) as handle:
        if out is None:
            out = torch.empty(rows, dtype=q.dtype, device=device)
        out_strides = _rows("out", _written("out", out), rows)
        size = lib.fa_sm100_paged_workspace_bytes(plan._ref)
        workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        strides = (ctypes.c_longlong * 10)(*q_strides, *out_strides, *k_strides, *v_strides)
        status = lib.fa_sm100_paged_fwd(plan._ref, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                        out.data_ptr(), strides, workspace.data_ptr() if size else None, size, handle)
    _check(status, "fa_sm100_paged_fwd")
    return out
