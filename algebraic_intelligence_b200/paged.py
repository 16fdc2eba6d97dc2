"""Serving from a paged key/value cache on B200 (no reference counterpart).

A cache is a pair of tensors (pages, kv_heads, page_size, dim); request b keeps
token j in page ``block_table[b, j // page_size]``, row ``j % page_size``.
Lengths, tables and the stack of free pages live on the GPU, so a step needs no
host copy and can be captured into a CUDA graph. One step of a server, whether
its requests append a prompt, a token or a tree of drafted tokens:

* ``paged_plan``    block tables, slot maps, positions and tree masks from the
                    requests' lengths; refuses what does not fit
* ``paged_append``  rotates the new queries and keys (several position axes,
                    see ``apply_ago_rotations_axes``) and writes keys and
                    values into the cache
* ``afa_paged``     AFA of the new tokens over the cache: the math of
                    ``pallas_afa_forward`` (src/kernels/pallas_afa.py:104-151)
                    with the keys read through the block table
* ``paged_commit``  moves the accepted path of a verified tree to its front;
                    the next ``paged_plan`` takes back the other nodes' pages

The tensors are CUDA tensors on one device; calls run on its current stream.
The caches, the block table and the free stack are updated in place. Make the
first call of each on a device before any stream capture: it sets kernel
attributes and resolves the device status word.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._tensors import refuse_tangents, tangents_exist
from .ago import axis_arguments

__all__ = ["PagedPlan", "paged_plan", "paged_append", "afa_paged", "paged_commit", "paged_workspace_bytes"]


_I32 = torch.int32


class PagedPlan(NamedTuple):
    """What ``paged_plan`` returns (T = max_tokens, B requests)."""
    slots: torch.Tensor        # (T,) int64: cache row page * page_size + offset, -1 behind the last token
    rows: torch.Tensor         # (T,) int32: request, -1 behind the last token
    positions: torch.Tensor    # (T,) int32: position in the request (a tree's: its length before + depth)
    cu_tokens: torch.Tensor    # (B + 1,) int32: first new token of each request
    seq_lens: torch.Tensor     # (B,) int32: lengths with the new tokens
    page_counts: torch.Tensor  # (B,) int32: pages held
    free_count: torch.Tensor   # (1,) int32: pages left on the stack
    granted: torch.Tensor      # (B,) bool: False for a request whose tokens or pages did not fit
    ancestors: Optional[torch.Tensor]  # (T, ceil(nodes / 32)) int32 words, with parents


def _check_page_size(page_size) -> None:
    if not isinstance(page_size, int) or page_size < 16 or page_size > 256 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 256, got {page_size}")


def _ints(name, t, shape):
    if not isinstance(t, torch.Tensor) or t.dtype is not _I32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _one_device(*tensors):
    """The CUDA device that all tensors live on."""
    index = tensors[0].get_device()  # -1: the host
    for t in tensors:
        if t is not None and (index < 0 or t.get_device() != index):
            if not t.is_cuda or index < 0:
                raise ValueError("the paged operators need CUDA tensors")
            raise ValueError(f"tensors on different devices: {tensors[0].device} and {t.device}")
    return tensors[0].device


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")
    if tangents_exist():
        refuse_tangents(what, *tensors)


def _caches(k_cache, v_cache, ndims=(4,)):
    """Checks a pair of caches; returns (pages, kv_heads, page_size, dim)."""
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor):
        raise TypeError("the caches must be tensors")
    shape = k_cache.shape
    if len(shape) not in ndims or shape != v_cache.shape:
        raise ValueError("k_cache and v_cache must have the same (pages, kv_heads, page_size, dim) shape, got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if not k_cache.is_floating_point():
        raise TypeError("expected a floating point array")
    if k_cache.dtype != v_cache.dtype:
        raise TypeError("k_cache and v_cache must share a dtype")
    pages, heads, page_size, dim = shape[-4:]
    _check_page_size(page_size)
    if 0 in shape:
        raise ValueError(f"the caches must not be empty, got {tuple(shape)}")
    if k_cache.stride()[-1] != 1 or v_cache.stride()[-1] != 1:
        raise ValueError("a cache row's channels must be contiguous")
    return pages, heads, page_size, dim


@functools.lru_cache(maxsize=4096)
def _apart(shape, strides, behind) -> bool:
    """Whether the elements of a strided view, and of a second one ``behind`` elements further, all lie apart. (Views
    made by slicing, indexing and transposing do: each stride passes what the smaller ones span.)"""
    def nested(*axes):
        span = 0
        for stride, n in sorted(axes):
            if n > 1:
                if stride <= span:
                    return False
                span += stride * (n - 1)
        return True

    axes = tuple(zip(strides, shape))
    # Or the second lies between the first's rows of an axis, some rows on (odd pages behind even ones).
    return nested(*axes, (behind, 2)) or any(
        nested(*axes[:i], (stride, n + behind // stride), *axes[i + 1:], (behind % stride, 2))
        for i, (stride, n) in enumerate(axes) if n > 1 and 0 < stride < behind)


def _written(k_cache, v_cache):
    """Refuses caches whose rows share memory, as an expanded one's: moves and writes of rows would race."""
    behind = abs(k_cache.data_ptr() - v_cache.data_ptr())
    if k_cache.is_contiguous() and v_cache.is_contiguous() and behind >= k_cache.nbytes:
        return
    if k_cache.stride() == v_cache.stride():
        apart = _apart(k_cache.shape, k_cache.stride(), behind // k_cache.element_size())
    else:
        apart = behind > 0 and all(_apart(t.shape, t.stride(), 1 << 62) for t in (k_cache, v_cache))
    if not apart:
        raise ValueError("the caches are written to: their rows must not share memory")


def _rows(t):
    """A tensor whose last axis is contiguous."""
    return t if t.is_contiguous() or t.stride()[-1] == 1 else t.contiguous()


def paged_plan(block_table, page_counts, seq_lens, new_lens, free_pages, free_count, page_size: int, max_tokens: int,
               parents=None) -> PagedPlan:
    """Block tables, slot maps and tree masks of one step, from the requests' lengths.

    block_table (B, columns), page_counts (B,): the pages each request holds;
    seq_lens (B,): its tokens; new_lens (B,): tokens it appends (below 0 counts
    as 0); free_pages (N,), free_count (1,): the stack of free pages. All int32
    on the GPU. With need = ceil((seq_lens + new_lens) / page_size), pages a
    request holds behind ``need`` (it ended, or drafted tokens were rejected)
    are released onto the stack in request order; then the requests that need
    more take them from its top, in request order (a page belongs to one
    request: one that two held would join the stack twice). ``free_pages`` has
    room for every page of the cache, since all may be free at once: a released
    page that finds no room is lost, and not counted. ``block_table`` and
    ``free_pages`` are updated in place; lengths and counts come back in new
    tensors, so a call with the same inputs gives the same step.

    A request is refused (``granted`` False; it keeps what it holds and gets no
    tokens) when its row of the table is too short, when the tokens asked for
    up to and with it pass ``max_tokens``, or when the pages run out.

    ``parents`` (B, nodes <= 256) int32: each request's new tokens form a tree;
    ``parents[b, i]`` in [0, i) is token i's parent, any other value makes it a
    root. Positions are then seq_len + depth, and ``ancestors`` holds the words
    ``afa_paged`` takes.
    """
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.ndim != 2 or not block_table.is_contiguous() or block_table.numel() == 0:
        raise ValueError("block_table must be a contiguous (batch, columns) tensor")
    b, cols = block_table.shape
    if b > 4096:
        raise ValueError("paged_plan: batch must be in [1, 4096]")
    _check_page_size(page_size)
    if not isinstance(max_tokens, int) or not 0 <= max_tokens <= 2 ** 30:
        raise ValueError("max_tokens must be an integer in [0, 2^30]")
    shape = (b,)
    _ints("page_counts", page_counts, shape)
    _ints("seq_lens", seq_lens, shape)
    _ints("new_lens", new_lens, shape)
    _ints("free_count", free_count, (1,))
    if not isinstance(free_pages, torch.Tensor) or free_pages.dtype != torch.int32:
        raise TypeError("free_pages must be an int32 tensor")
    if free_pages.ndim != 1 or not free_pages.is_contiguous() or free_pages.numel() == 0:
        raise ValueError("free_pages must be a contiguous one-dimensional tensor")
    nodes = 0
    if parents is not None:
        if not isinstance(parents, torch.Tensor) or parents.ndim != 2:
            raise ValueError("parents must have shape (batch, nodes)")
        nodes = parents.shape[1]
        _ints("parents", parents, (b, nodes))
        if not 1 <= nodes <= 256:
            raise ValueError("a tree may have at most 256 nodes")
    dev = _one_device(block_table, page_counts, seq_lens, new_lens, free_pages, free_count, parents)
    page_counts, seq_lens, new_lens = page_counts.contiguous(), seq_lens.contiguous(), new_lens.contiguous()
    parents = parents.contiguous() if parents is not None else None
    # One allocation, cut up: int64 slots first, then 32-bit words.
    words, t = (nodes + 31) // 32, max_tokens
    w, g = t * words, (b + 3) // 4
    buf = torch.empty(4 * t + 3 * b + 2 + w + g, dtype=torch.int32, device=dev)
    slots, rows, positions, cu, lens_out, held_out, free_out, ancestors, granted = buf.split_with_sizes(
        (2 * t, t, t, b + 1, b, b, 1, w, g))
    per_request = buf.data_ptr() + 16 * t  # cu_tokens
    behind = per_request + 12 * b + 8      # ancestors
    rc = _lib.call(
        dev, _lib.load().afa_paged_plan, block_table.data_ptr(), page_counts.data_ptr(), seq_lens.data_ptr(),
        new_lens.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), parents.data_ptr() if nodes else None,
        per_request - 16 * t, per_request - 8 * t, per_request - 4 * t, per_request, per_request + 4 * b + 4,
        per_request + 8 * b + 4, behind - 4, behind + 4 * w, behind, b, cols, page_size, free_pages.shape[0], t, nodes)
    if rc:
        _lib.check(rc, "afa_paged_plan")
    increment_version((block_table, free_pages))
    return PagedPlan(slots.view(torch.int64), rows, positions, cu, lens_out, held_out, free_out,
                     granted.view(torch.bool)[:b], ancestors.view(max_tokens, words) if nodes else None)


def paged_append(k, v, k_cache, v_cache, slots, q=None, rotary_params=None, positions=None, sections=None):
    """Writes new keys and values into a paged cache, rotating on the way.

    k, v (tokens, kv_heads, dim) go to cache rows ``slots`` (tokens,) int64 (a
    ``PagedPlan``'s); a slot outside the cache, such as a padded token's -1, is
    skipped, and slots inside it are distinct. With ``rotary_params``,
    ``positions`` (axes, tokens) and ``sections`` as in
    ``apply_ago_rotations_axes`` the keys are rotated, and so is ``q`` (tokens,
    heads, dim), which comes back; without q the result is None. Rows start on a
    channel pair (views off one are refused). The caches may be strided views
    (such as a (pages, page_size, heads, dim) cache transposed) whose rows lie
    apart.
    """
    pages, heads, page_size, dim = _caches(k_cache, v_cache)
    if k.ndim != 3 or k.shape != v.shape or k.shape[1:] != (heads, dim):
        raise ValueError(f"k and v must have shape (tokens, {heads}, {dim}), got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    tokens = k.shape[0]
    if q is not None and (q.ndim != 3 or q.shape[0] != tokens or q.shape[2] != dim or q.shape[1] == 0):
        raise ValueError(f"q must have shape ({tokens}, heads, {dim}), got {tuple(q.shape)}")
    dtype = k_cache.dtype
    if k.dtype != dtype or v.dtype != dtype or (q is not None and q.dtype != dtype):
        raise TypeError("k, v, q and the caches must share a dtype")
    if k_cache.dtype == torch.float16:
        raise TypeError("float16 is not supported; use bfloat16 or float32")
    if not isinstance(slots, torch.Tensor) or slots.dtype not in (torch.int64, torch.int32):
        raise TypeError("slots must be an int64 tensor")
    if slots.shape != (tokens,):
        raise ValueError(f"slots must have shape ({tokens},), got {tuple(slots.shape)}")
    if dim % 2 != 0:
        raise ValueError(f"Feature dimension must be even, got {dim}")
    if rotary_params is None and (q is not None or positions is not None or sections is not None):
        raise ValueError("q, positions and sections go with rotary_params")
    _no_gradient("paged_append", k, v, q, k_cache, v_cache)
    dev = _one_device(k_cache, v_cache, k, v, q, slots)
    _written(k_cache, v_cache)
    axes = axis_arguments(rotary_params, positions, sections, dim, (tokens,), dev) if rotary_params is not None \
        else None
    k, v = _rows(k), _rows(v)
    if slots.dtype != torch.int64:
        slots = slots.to(torch.int64)
    slots = slots.contiguous()
    out = None
    if q is not None:
        q = _rows(q)
        out = torch.empty((tokens, q.shape[1], dim), dtype=q.dtype, device=dev)
    if axes is not None:
        c, p = axes.c, axes.positions
        pos = (c.data_ptr(), axes.s.data_ptr(), _lib.dtype_code(c.dtype), c.shape[0], p.data_ptr(),
               _lib.longs(*p.stride()), p.dtype == torch.int64, axes.sections, p.shape[0])
    else:
        pos = (None, None, 0, 0, None, None, 0, None, 0)
    rc = _lib.call(
        dev, _lib.load().afa_paged_append, k.data_ptr(), _lib.longs(*k.stride()[:2]), v.data_ptr(),
        _lib.longs(*v.stride()[:2]), k_cache.data_ptr(), _lib.longs(*k_cache.stride()[:3]), v_cache.data_ptr(),
        _lib.longs(*v_cache.stride()[:3]),
        slots.data_ptr(), None if q is None else q.data_ptr(),
        None if q is None else _lib.longs(*q.stride()[:2]), None if out is None else out.data_ptr(),
        0 if q is None else q.shape[1], *pos, tokens, heads, dim, pages, page_size,
        _lib.dtype_code(k_cache.dtype))
    if rc:
        _lib.check(rc, "afa_paged_append")
    increment_version((k_cache, v_cache))
    return out


def paged_workspace_bytes(tokens: int, q_heads: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16) -> int:
    """Scratch bytes ``afa_paged`` needs for this shape."""
    return int(_lib.load().afa_paged_workspace_bytes(tokens, q_heads, kv_heads, head_dim, _lib.dtype_code(dtype)))


def afa_paged(q, k_cache, v_cache, block_table, seq_lens, cu_tokens, ancestors=None, sink_omega: float = 0.5,
              return_denominator: bool = False, out: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None):
    """AFA of new tokens over a paged cache: single tokens, prompt chunks, drafted trees.

    q (tokens, heads, dim): the requests' new tokens one after the other,
    request b's from ``cu_tokens[b]`` to ``cu_tokens[b + 1]``; heads a multiple
    of the cache's, head h reading key head h // (heads / kv_heads).
    ``seq_lens`` (B,) counts a request's keys, its n new tokens (already in the
    cache) included. A new token sees the seq_len - n keys before them, and of
    the new ones those up to itself or, with ``ancestors`` (tokens, words) int32
    (bit j of word j // 32: new token j of its request), those whose bit is set.
    Keys whose table entry names no page of the cache are not seen; a row that
    sees no key gives output 0 and d_total = sink_omega. Cached rows of a
    request must be finite; what lies behind its last token does not matter.

    Returns out (tokens, heads, dim), with ``return_denominator`` also d_total
    (tokens, heads) in the accumulation dtype. Rows of q behind the last request
    are not computed: with ``out`` given they are left as they were, otherwise
    their contents are unspecified. ``workspace`` (see
    ``paged_workspace_bytes``) is overwritten; calls that may overlap need one
    each. bfloat16 with dim 64 or 128 runs on the tensor cores.
    """
    if not 0 <= sink_omega < float("inf"):
        raise ValueError("sink_omega must be finite and nonnegative")
    pages, kv_heads, page_size, dim = _caches(k_cache, v_cache)
    if not isinstance(q, torch.Tensor) or not q.is_floating_point():
        raise TypeError("expected a floating point array")
    if q.ndim != 3 or q.shape[2] != dim or q.shape[1] == 0 or q.shape[1] % kv_heads != 0:
        raise ValueError(f"q must have shape (tokens, heads, {dim}) with heads a multiple of {kv_heads}, got "
                         f"{tuple(q.shape)}")
    if q.dtype != k_cache.dtype:
        raise TypeError("q and the caches must share a dtype")
    code = _lib.dtype_code(q.dtype)
    if code == _lib.AFA_F16:
        raise TypeError("float16 is not supported: rho(s)^8 overflows float16 for s > 2.4; use bfloat16 or float32")
    tokens, heads, _ = q.shape
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.ndim != 2 or block_table.numel() == 0:
        raise ValueError("block_table must have shape (batch, columns)")
    b, cols = block_table.shape
    _ints("seq_lens", seq_lens, (b,))
    _ints("cu_tokens", cu_tokens, (b + 1,))
    words = 0
    if ancestors is not None:
        if not isinstance(ancestors, torch.Tensor) or ancestors.dtype != torch.int32:
            raise TypeError("ancestors must be an int32 tensor")
        if ancestors.ndim != 2 or ancestors.shape[0] != tokens or ancestors.shape[1] == 0:
            raise ValueError(f"ancestors must have shape ({tokens}, words), got {tuple(ancestors.shape)}")
        words = ancestors.shape[1]
        ancestors = _rows(ancestors)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor of q's shape and dtype")
    _no_gradient("afa_paged", q, k_cache, v_cache, out)
    dev = _one_device(q, k_cache, v_cache, block_table, seq_lens, cu_tokens, ancestors, out, workspace)
    q, block_table = _rows(q), _rows(block_table)
    seq_lens, cu_tokens = seq_lens.contiguous(), cu_tokens.contiguous()
    given = out is not None
    if not given:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=dev)
    den = torch.empty((tokens, heads), dtype=_lib.accum_dtype(q.dtype), device=dev) if return_denominator else None
    lib = _lib.load()
    need = lib.afa_paged_workspace_bytes(tokens, heads, kv_heads, dim, code)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    elif not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace must be a contiguous tensor of at least {need} bytes")
    elif workspace.data_ptr() % 16:
        raise ValueError("workspace must start on a 16-byte boundary")
    rc = _lib.call(
        dev, lib.afa_paged, q.data_ptr(), _lib.longs(*q.stride()[:2]), k_cache.data_ptr(), v_cache.data_ptr(),
        _lib.longs(*k_cache.stride()[:3]), _lib.longs(*v_cache.stride()[:3]), out.data_ptr(),
        None if den is None else den.data_ptr(), block_table.data_ptr(), block_table.stride()[0],
        seq_lens.data_ptr(), cu_tokens.data_ptr(), ancestors.data_ptr() if words else None,
        ancestors.stride(0) if words else 0, words, b, tokens, heads, kv_heads, dim, cols, page_size, pages, code,
        float(sink_omega), workspace.data_ptr(), need)
    if rc:
        _lib.check(rc, "afa_paged")
    if given:
        increment_version(out)
    return (out, den) if return_denominator else out


def paged_commit(k_cache, v_cache, block_table, base_lens, seq_lens, accepted) -> torch.Tensor:
    """Moves the accepted path of each request's drafted tree to its front.

    ``base_lens`` (B,): tokens before the tree; ``seq_lens`` (B,): with it;
    ``accepted`` (B, path <= 256): the accepted nodes from the root on, -1
    behind the last. Cache row base + i becomes row base + accepted[i] for the
    longest prefix of ``accepted`` that ascends strictly, lies in the tree and
    whose pages are in the cache. The caches may hold several layers, (layers,
    pages, kv_heads, page_size, dim). Returns the lengths base + accepted (B,)
    int32, the next ``paged_plan``'s ``seq_lens``.
    """
    pages, heads, page_size, dim = _caches(k_cache, v_cache, (4, 5))
    if k_cache.dtype == torch.float16:
        raise TypeError("float16 is not supported; use bfloat16 or float32")
    if not isinstance(block_table, torch.Tensor) or block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.ndim != 2 or block_table.numel() == 0:
        raise ValueError("block_table must have shape (batch, columns)")
    b, cols = block_table.shape
    _ints("base_lens", base_lens, (b,))
    _ints("seq_lens", seq_lens, (b,))
    if not isinstance(accepted, torch.Tensor) or accepted.ndim != 2:
        raise ValueError("accepted must have shape (batch, path)")
    path = accepted.shape[1]
    _ints("accepted", accepted, (b, path))
    if path > 256:
        raise ValueError("an accepted path may have at most 256 tokens")
    _no_gradient("paged_commit", k_cache, v_cache)
    dev = _one_device(k_cache, v_cache, block_table, base_lens, seq_lens, accepted)
    _written(k_cache, v_cache)
    block_table, accepted = _rows(block_table), _rows(accepted)
    base_lens, seq_lens = base_lens.contiguous(), seq_lens.contiguous()
    lens = torch.empty(b, dtype=torch.int32, device=dev)
    layers = k_cache.shape[0] if k_cache.ndim == 5 else 1
    strides = [(0, *t.stride()[:3]) if t.ndim == 4 else t.stride()[:4] for t in (k_cache, v_cache)]
    rc = _lib.call(
        dev, _lib.load().afa_paged_commit, k_cache.data_ptr(), _lib.longs(*strides[0]), v_cache.data_ptr(),
        _lib.longs(*strides[1]), block_table.data_ptr(), block_table.stride(0), base_lens.data_ptr(),
        seq_lens.data_ptr(), accepted.data_ptr(),
        accepted.stride(0) if path else 0, lens.data_ptr(), b, path, layers, heads, dim, cols, pages, page_size,
        _lib.dtype_code(k_cache.dtype))
    if rc:
        _lib.check(rc, "afa_paged_commit")
    increment_version((k_cache, v_cache))
    return lens
