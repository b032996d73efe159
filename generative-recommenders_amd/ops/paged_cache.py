"""Rotated positions, and a paged K/V cache held in 4 bits with the attention that reads it.

``qk_norm_rope``: norms of q and k for each head and the rotation by position in one pass, between the producer of q, k, v
(``hstu_compute_uqvk``) and the attention; differentiable.  ``append_paged_kv`` puts new K and V rows into the pages of a
cache, normed and rotated on the way; ``read_paged_kv`` gives rows of it back as values, for the operators that read 16-bit K
and V; ``delta_hstu_mha_paged`` is ``delta_hstu_mha`` on such a cache.  The reference has none of them: its layers take
positions from an embedding, and its cache is a jagged 16-bit tensor that it concatenates anew
(``generative_recommenders/modules/stu.py:84-173``).

Device tensors only; hand-written gfx950 kernels behind ``include/hstu_cache.h`` (``csrc/hstu_norm_rope.h``,
``csrc/hstu_paged_rows.h``, ``csrc/hstu_paged_attention_kernel.h``), called through the native front.  The functions below
check what it leaves: tensors that need a copy first, and calls that are refused.
"""

from typing import NamedTuple, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import hip_backend, native
from .hstu_attention import _check_forward_only, _kernel_layout, _require_device


class PagedKVCache(NamedTuple):
    """Pages of K and V rows in 4 bits.  A row is ``dim`` codes, two to a byte (the even column in the low half), and a pair
    (step, lowest value) in the type of K and V; a column's value is ``lowest + step * code``.  Any four tensors in this order
    will do wherever a cache is asked for."""

    k_codes: torch.Tensor  # uint8 [pages, heads, page_size, dqk / 2]
    k_scales: torch.Tensor  # [pages, heads, page_size, 2]
    v_codes: torch.Tensor  # uint8 [pages, heads, page_size, dv / 2]
    v_scales: torch.Tensor  # [pages, heads, page_size, 2]


def allocate_paged_kv_cache(pages: int, page_size: int, heads: int, dqk: int, dv: int, dtype: torch.dtype = torch.bfloat16,
                            device: torch.device = torch.device("cuda")) -> PagedKVCache:
    """A cache of ``pages`` pages, all rows zero.  ``page_size``: a power of two from 16 to 1024; head dims 32, 64, 128 or 256."""
    torch._assert(dtype in (torch.bfloat16, torch.float16), "a cache is of K and V in bf16 or fp16")
    torch._assert(pages > 0 and heads > 0, "a cache holds at least one page and one head")
    if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise NotImplementedError("page_size must be a power of two from 16 to 1024")
    if any(d not in (32, 64, 128, 256) for d in (dqk, dv)):
        raise NotImplementedError("head dims of a cache are 32, 64, 128 or 256")
    shape = (pages, heads, page_size)
    return PagedKVCache(
        torch.zeros(shape + (dqk // 2,), dtype=torch.uint8, device=device), torch.zeros(shape + (2,), dtype=dtype, device=device),
        torch.zeros(shape + (dv // 2,), dtype=torch.uint8, device=device), torch.zeros(shape + (2,), dtype=dtype, device=device),
    )


def make_rotary_table(positions: int, rotary_dim: int, base: float = 10000.0, device: torch.device = torch.device("cuda")) -> torch.Tensor:
    """``[positions, rotary_dim]`` fp32: cosines, then sines, of ``position * base ** (-2 i / rotary_dim)``.  Angles are formed in
    64 bits: in 32 those of far positions would be off by up to position * 2**-24."""
    torch._assert(positions > 0 and rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_dim must be even and positions at least 1")
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device).view(-1, 1) * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


def _index(x: torch.Tensor, name: str, size: int, device: torch.device) -> torch.Tensor:
    _require_device(x, name)
    torch._assert(x.dtype in (torch.int32, torch.int64), f"{name} must be int32 or int64")
    torch._assert(x.dim() == 1 and x.numel() == size, f"{name} must hold {size} values")
    torch._assert(x.device == device, f"{name} must be on the device of the others")
    return x.contiguous()


def _parameter(x: Optional[torch.Tensor], name: str, dim: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    if x is None:
        return None
    _require_device(x, name)
    torch._assert(x.dim() == 1 and x.shape[0] == dim, f"{name} must hold one value per column of a head")
    torch._assert(x.dtype == like.dtype and x.device == like.device, f"{name} must have the type and device of what it weighs")
    return _dense(x)


def _dense(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _rotary(table: Optional[torch.Tensor], dim: int, interleaved: bool, device: torch.device) -> Optional[torch.Tensor]:
    if table is None:
        return None
    _require_device(table, "rotary_table")
    torch._assert(table.dim() == 2 and table.dtype == torch.float32, "rotary_table must be a 2-D float32 tensor")
    torch._assert(table.device == device, "rotary_table must be on the device of the others")
    torch._assert(0 < table.shape[1] <= dim, "rotary_table must not be wider than a head")
    if table.shape[1] % (8 if interleaved else 16) != 0:
        raise NotImplementedError("rotated columns come in multiples of 16 (interleaved pairs: of 8)")
    if torch.is_grad_enabled() and table.requires_grad:
        raise NotImplementedError("the HIP backend has no gradient for rotary_table; detach it")
    return _dense(table)


def _check_no_tangents(*tensors: Optional[torch.Tensor]) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the HIP backend has no forward-mode derivatives; pass tensors without tangents")


def _check_positions(positions: torch.Tensor, table: torch.Tensor) -> None:
    if positions.numel() and not bool(((positions >= 0) & (positions < table.shape[0])).all()):
        raise ValueError("hstu_cache: positions outside of the rotary table")


def _served(out, name: str):
    if out is None or out is False:
        raise RuntimeError(f"hstu_cache: {name} has no kernel for this call")
    return out


def qk_norm_rope(
    q: torch.Tensor,
    k: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    rotary_table: Optional[torch.Tensor] = None,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``x / sqrt(mean(x^2) + eps) * weight`` for each head of q and k, then the rotation of ``positions``; returns both, dense.

    ``q`` ``[L, Hq, D]``, ``k`` ``[L, Hk, D]`` or None; bf16, fp16 or fp32, any row and head strides.  A weight (``[D]``, shared
    by the heads) that is None leaves its norm out; no ``rotary_table`` (``make_rotary_table``), no rotation.  The table's width is
    how many columns of a head turn: pairs ``(i, i + width / 2)``, or ``(2 i, 2 i + 1)`` with ``interleaved``.  fp32 inside, one
    rounding at the end.  ``positions``: ``[L]``; a row whose position is not in the table comes back NaN
    (``HSTU_HIP_CHECK_CONTRACT=1`` raises instead).  Gradients for q, k and both weights; a weight's are summed in fp32 and,
    over the lanes, in 64 bits, in an order that only depends on the sizes.  Tensors with forward-mode tangents are refused.
    """
    out = native.front.qk_norm_rope(q, k, positions, rotary_table, q_weight, k_weight, eps, interleaved, False)
    if out is not None:
        return out
    _require_device(q, "q")
    torch._assert(q.dim() == 3, "q must be 3-D")
    torch._assert(q.dtype in (torch.bfloat16, torch.float16, torch.float32), "qk_norm_rope takes bf16, fp16 and fp32")
    rows, _, dim = q.shape
    if k is not None:
        _require_device(k, "k")
        torch._assert(k.dim() == 3, "k must be 3-D")
        torch._assert(k.shape[0] == rows and k.shape[2] == dim, "k must have q's rows and head dim")
        torch._assert(k.dtype == q.dtype and k.device == q.device, "q and k must have the same dtype and device")
    torch._assert(k is not None or k_weight is None, "k_weight without k")
    torch._assert(rotary_table is not None or q_weight is not None or k_weight is not None, "neither a norm weight nor a rotary table")
    _check_no_tangents(q, k, q_weight, k_weight, rotary_table)
    q_weight, k_weight = _parameter(q_weight, "q_weight", dim, q), _parameter(k_weight, "k_weight", dim, q)
    rotary_table = _rotary(rotary_table, dim, interleaved, q.device)
    if rotary_table is not None:
        torch._assert(positions is not None, "a rotation needs positions")
        positions = _index(positions, "positions", rows, q.device)
        if hip_backend.contract_checks_enabled():
            _check_positions(positions, rotary_table)
    if dim % 8 != 0 or dim > 512:
        raise NotImplementedError("head dims are multiples of 8 up to 512")
    if q.numel() == 0 or (k is not None and k.numel() == 0):
        if q.numel() == 0 and (k is None or k.numel() == 0):
            # nothing in them; the graph, if there is one, goes on, to gradients of zero for the weights too
            return q * (1 if q_weight is None else q_weight), None if k is None else k * (1 if k_weight is None else k_weight)
        raise NotImplementedError("q and k must both have heads")
    q = _copied(q)
    k = None if k is None else _copied(k)
    return _served(native.front.qk_norm_rope(q, k, positions, rotary_table, q_weight, k_weight, eps, interleaved, True), "qk_norm_rope")


def _copied(x: torch.Tensor) -> torch.Tensor:
    """``x`` with rows the kernels can read; a copy that gradients flow through where it needs one."""
    y = _kernel_layout(x)
    per16 = 16 // x.element_size()
    if any(y.shape[d] > 1 and (y.stride(d) % per16 or y.stride(d) < 0) for d in (0, 1)):
        y = y.clone(memory_format=torch.contiguous_format)
    return y


def _cache_tensors(cache: Sequence[torch.Tensor], page_table: torch.Tensor) -> Tuple[torch.Tensor, ...]:
    torch._assert(len(cache) == 4, "a cache is codes and scales of K, then of V")
    k_codes, k_scales, v_codes, v_scales = cache
    for x, name in zip(cache, PagedKVCache._fields):
        _require_device(x, name)
        torch._assert(x.dim() == 4 and x.is_contiguous() and x.data_ptr() % 16 == 0, f"{name} must be a dense, 16-byte aligned 4-D tensor")
        torch._assert(x.device == k_codes.device, "the cache's tensors must be on one device")
        torch._assert(x.shape[:3] == k_codes.shape[:3], "the cache's tensors must agree in pages, heads and page size")
        torch._assert(not x.requires_grad, "a cache has no gradient")
    torch._assert(k_codes.dtype == torch.uint8 and v_codes.dtype == torch.uint8, "codes are uint8, two to a byte")
    torch._assert(k_scales.dtype in (torch.bfloat16, torch.float16) and v_scales.dtype == k_scales.dtype, "scales are bf16 or fp16")
    torch._assert(k_scales.shape[3] == 2 and v_scales.shape[3] == 2, "scales are pairs (step, lowest value)")
    torch._assert(k_codes.shape[0] > 0 and k_codes.shape[1] > 0, "a cache holds at least one page and one head")
    page = k_codes.shape[2]
    if page < 16 or page > 1024 or page & (page - 1):
        raise NotImplementedError("page_size must be a power of two from 16 to 1024")
    if any(2 * x.shape[3] not in (32, 64, 128, 256) for x in (k_codes, v_codes)):
        raise NotImplementedError("head dims of a cache are 32, 64, 128 or 256")
    _require_device(page_table, "page_table")
    torch._assert(page_table.dim() == 2 and page_table.dtype in (torch.int32, torch.int64), "page_table must be 2-D, int32 or int64")
    torch._assert(page_table.device == k_codes.device, "page_table must be on the cache's device")
    torch._assert(page_table.shape[0] > 0 and page_table.shape[1] > 0, "page_table must hold at least one sequence and one page")
    return tuple(cache)


def _pages(page_table: torch.Tensor) -> torch.Tensor:
    return page_table if page_table.stride(1) == 1 and page_table.stride(0) >= 0 else page_table.contiguous()


def _check_places(cache, page_table: torch.Tensor, start: torch.Tensor, offsets: Optional[torch.Tensor], rows: int) -> None:
    """The caller contract of rows start[b] .. start[b] + count[b] - 1 of every sequence (synchronises)."""
    page, pages = cache[0].shape[2], cache[0].shape[0]
    batch = page_table.shape[0]
    if offsets is None:
        count = torch.full((batch,), rows // batch, dtype=torch.int64, device=start.device)
    else:
        count = (offsets[1:] - offsets[:-1]).long()
        if bool((count < 0).any()) or int(offsets[0]) != 0 or int(offsets[-1]) > rows:
            raise ValueError("hstu_cache: seq_offsets decrease, do not begin at 0 or end behind the rows")
    end = start.long() + count
    if bool(((start < 0) | (end > page_table.shape[1] * page)).any()):
        raise ValueError("hstu_cache: a sequence does not fit its row of the page table")
    column = torch.arange(page_table.shape[1], device=start.device).view(1, -1)
    used = (column >= (start.long() // page).view(-1, 1)) & (column < ((end + page - 1) // page).view(-1, 1)) & (count > 0).view(-1, 1)
    if bool((used & ((page_table < 0) | (page_table >= pages))).any()):
        raise ValueError("hstu_cache: page_table names a page that the cache does not have")


def _check_once(cache, page_table: torch.Tensor, start: torch.Tensor, count: torch.Tensor) -> None:
    """No two of the rows start[b] .. start[b] + count[b] - 1, whose places there are, have one (synchronises)."""
    page, count = cache[0].shape[2], count.long()
    of = torch.repeat_interleave(torch.arange(count.numel(), device=count.device), count)
    place = start.long()[of] + torch.arange(of.numel(), device=count.device) - (count.cumsum(0) - count)[of]
    row = page_table[of, place // page].long() * page + place % page
    if row.unique().numel() != row.numel():
        raise ValueError("hstu_cache: two rows of the call have one place")


def _first_seen(lengths: torch.Tensor, targets: Optional[torch.Tensor], delta: int, max_attn_len: int, contextual: int) -> torch.Tensor:
    """The first position that any of the newest ``delta`` positions of each sequence sees."""
    top = (lengths - delta).clamp(min=0)
    history = lengths if targets is None else lengths - targets.long()
    ids = torch.minimum(top, history) - (contextual - 1 if contextual else 0)
    lowest = (ids - max_attn_len + (contextual - 1 if contextual else 0)) if max_attn_len else torch.zeros_like(ids)
    first = torch.where(ids > max_attn_len, lowest, torch.zeros_like(ids))
    if contextual:
        return torch.where(top < contextual, torch.zeros_like(ids), first)
    return torch.where(ids > 0, first, top)


def append_paged_kv(
    cache: Sequence[torch.Tensor],
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    start: torch.Tensor,
    seq_offsets: Optional[torch.Tensor] = None,
    rotary_table: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> None:
    """Put new K and V rows into their pages, in place: the norm of every head of K (``k_weight``) and its rotation
    (``rotary_table``) as ``qk_norm_rope`` does them, the result rounded to K's type and then, as V, to 4 bits.

    Row ``seq_offsets[b] + i`` of ``k`` ``[L, H, dqk]`` and ``v`` ``[L, H, dv]`` is position ``start[b] + i`` of sequence ``b``;
    without ``seq_offsets`` every sequence has ``L / batch`` rows.  Position ``p`` lies in page ``page_table[b][p // page_size]``.
    ``positions`` (``[L]``): the positions to rotate by, where they are not the places in the sequence (candidates that all
    stand behind the same history).  A row is kept as (step, lowest value) in K's type and codes 0 .. 15: half a step off at
    most, and the rounding of the step.  A row with a NaN or an infinity becomes NaN.

    Caller contract: every place has a page, no two rows of a call have one place (``HSTU_HIP_CHECK_CONTRACT=1`` raises where
    either does not hold).  Rows without a page are not stored; what two rows leave in one place is neither's; rows behind the
    last sequence are no one's and not stored either.
    No gradients.
    """
    if native.front.append_paged_kv(tuple(cache), k, v, page_table, start, seq_offsets, rotary_table, positions, k_weight, eps, interleaved, False):
        return
    cache = _cache_tensors(cache, page_table)
    heads, dqk, dv = cache[0].shape[1], 2 * cache[0].shape[3], 2 * cache[2].shape[3]
    for x, name, dim in ((k, "k", dqk), (v, "v", dv)):
        _require_device(x, name)
        torch._assert(x.dim() == 3 and x.shape[1] == heads and x.shape[2] == dim, f"{name} must be [rows, {heads}, {dim}] as the cache's rows")
        torch._assert(x.dtype == cache[1].dtype and x.device == cache[1].device, f"{name} must have the cache's type and device")
    torch._assert(v.shape[0] == k.shape[0], "k and v must have the same rows")
    rows, batch = k.shape[0], page_table.shape[0]
    start = _index(start, "start", batch, k.device)
    if seq_offsets is not None:
        seq_offsets = _index(seq_offsets, "seq_offsets", batch + 1, k.device)
    else:
        torch._assert(rows % batch == 0, "without seq_offsets all sequences have the same number of rows")
    k_weight = _parameter(k_weight, "k_weight", dqk, k)
    rotary_table = _rotary(rotary_table, dqk, interleaved, k.device)
    if positions is not None:
        positions = _index(positions, "positions", rows, k.device)
    _check_forward_only(k, v, *([] if k_weight is None else [k_weight]))
    _check_no_tangents(k, v, k_weight, rotary_table)
    if rows == 0:
        return
    if hip_backend.contract_checks_enabled():
        _check_places(cache, page_table, start, seq_offsets, rows)
        count = torch.full_like(start, rows // batch) if seq_offsets is None else seq_offsets[1:] - seq_offsets[:-1]
        _check_once(cache, page_table, start, count)
        if rotary_table is not None:
            if positions is None:
                _check_positions((start + count - 1)[count > 0], rotary_table)
            else:  # (rows behind the last sequence are no one's)
                _check_positions(positions if seq_offsets is None else positions[: int(seq_offsets[-1])], rotary_table)
    _served(native.front.append_paged_kv(cache, _copied(k), _copied(v), _pages(page_table), start, seq_offsets, rotary_table, positions,
                                         k_weight, eps, interleaved, True), "append_paged_kv")


def read_paged_kv(
    cache: Sequence[torch.Tensor],
    rows: int,
    page_table: torch.Tensor,
    start: torch.Tensor,
    seq_offsets: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of a cache as values in its type: ``k [rows, H, dqk]`` and ``v [rows, H, dv]``, row ``seq_offsets[b] + i`` being position
    ``start[b] + i`` of sequence ``b`` (without ``seq_offsets``: ``rows / batch`` positions of each).  Rows behind the last sequence
    are zero; one whose place has no page is NaN (``HSTU_HIP_CHECK_CONTRACT=1`` raises instead)."""
    out = native.front.read_paged_kv(tuple(cache), rows, page_table, start, seq_offsets, False)
    if out is not None:
        return out
    cache = _cache_tensors(cache, page_table)
    torch._assert(rows >= 0, "rows must not be negative")
    batch, device = page_table.shape[0], cache[1].device
    start = _index(start, "start", batch, device)
    if seq_offsets is not None:
        seq_offsets = _index(seq_offsets, "seq_offsets", batch + 1, device)
    else:
        torch._assert(rows % batch == 0, "without seq_offsets all sequences have the same number of rows")
    if rows == 0:
        return tuple(torch.empty((0, cache[0].shape[1], 2 * c.shape[3]), dtype=cache[1].dtype, device=device) for c in (cache[0], cache[2]))
    if hip_backend.contract_checks_enabled():
        _check_places(cache, page_table, start, seq_offsets, rows)
    return _served(native.front.read_paged_kv(cache, rows, _pages(page_table), start, seq_offsets, True), "read_paged_kv")


def delta_hstu_mha_paged(
    max_seq_len: int,
    alpha: float,
    delta_q: torch.Tensor,
    cache: Sequence[torch.Tensor],
    page_table: torch.Tensor,
    seq_lengths: torch.Tensor,
    num_targets: Optional[torch.Tensor] = None,
    max_attn_len: int = 0,
    contextual_seq_len: int = 0,
    kv_splits: int = 0,
) -> torch.Tensor:
    """``delta_hstu_mha`` on a paged cache in 4 bits: ``delta_q`` ``[batch * delta, Hq, dqk]`` holds the newest ``delta`` positions
    of every sequence, whose K and V rows are in the cache already (``append_paged_kv``); ``seq_lengths`` counts them.  Head ``h`` of
    ``delta_q`` reads head ``h // (Hq / H)`` of the cache.  Returns ``[batch * delta, Hq, dv]`` in the dtype of ``delta_q``.

    The masks are those of ``delta_hstu_mha``.  K and V enter as they are stored, unrounded (``lowest + step * code``); sums are in
    fp32.  A sequence shorter than ``delta`` has zeros in the rows in front of its first position; one that does not fit its row
    of the page table comes back NaN, and so does every row that sees a position on a page that the cache does not have (other rows
    of its sequence may; ``HSTU_HIP_CHECK_CONTRACT=1`` raises instead).  Pages that end in front of the first position that any of
    the ``delta`` rows sees, behind a window, may be gone: they are not looked at.  ``kv_splits``: at most so many runs per row block
    (0 = automatic); it changes the order of the fp32 sums.
    """
    out = native.front.delta_hstu_mha_paged(max_seq_len, alpha, delta_q, tuple(cache), page_table, seq_lengths, num_targets, max_attn_len,
                                            contextual_seq_len, kv_splits, False)
    if out is not None:
        return out
    cache = _cache_tensors(cache, page_table)
    torch._assert(0 < max_seq_len < 2**31, "max_seq_len must be larger than 0")
    torch._assert(min(max_attn_len, contextual_seq_len, kv_splits) >= 0 and max(max_attn_len, contextual_seq_len, kv_splits) < 2**31,
                  "max_attn_len, contextual_seq_len and kv_splits must not be negative")
    _require_device(delta_q, "delta_q")
    torch._assert(delta_q.dim() == 3, "delta_q must be 3-D")
    batch, heads, dqk = page_table.shape[0], cache[0].shape[1], 2 * cache[0].shape[3]
    torch._assert(delta_q.shape[2] == dqk, "delta_q must have the head dim of the cache's K")
    torch._assert(delta_q.shape[1] % heads == 0, "delta_q must have a multiple of the cache's heads")
    torch._assert(delta_q.shape[0] % batch == 0, "delta_q must be padded")
    torch._assert(delta_q.dtype == cache[1].dtype and delta_q.device == cache[1].device, "delta_q must have the cache's type and device")
    if 256 in (dqk, 2 * cache[2].shape[3]) and cache[0].shape[3] != cache[2].shape[3]:
        raise NotImplementedError("a head dim of 256 is built for K and V alike")
    seq_lengths = _index(seq_lengths, "seq_lengths", batch, delta_q.device)
    if num_targets is not None:
        num_targets = _index(num_targets, "num_targets", batch, delta_q.device)
    _check_forward_only(delta_q)
    _check_no_tangents(delta_q)
    if delta_q.numel() == 0:
        return torch.empty((delta_q.shape[0], delta_q.shape[1], 2 * cache[2].shape[3]), dtype=delta_q.dtype, device=delta_q.device)
    if hip_backend.contract_checks_enabled():
        first = _first_seen(seq_lengths.long(), num_targets, delta_q.shape[0] // batch, max_attn_len, contextual_seq_len)
        count = seq_lengths - first
        _check_places(cache, page_table, first, torch.nn.functional.pad(count.cumsum(0), (1, 0)), int(count.sum()))
        if bool((seq_lengths > max_seq_len).any()):
            raise ValueError("hstu_cache: a sequence is longer than max_seq_len")
        if num_targets is not None and bool(((num_targets < 0) | (num_targets > seq_lengths)).any()):
            raise ValueError("hstu_cache: num_targets outside [0, length]")
        if bool(((seq_lengths - (0 if num_targets is None else num_targets) < contextual_seq_len) & (seq_lengths > 0)).any()):
            raise ValueError("hstu_cache: fewer non-target positions than contextual_seq_len")
    return _served(native.front.delta_hstu_mha_paged(max_seq_len, alpha, _copied(delta_q), cache, _pages(page_table), seq_lengths, num_targets,
                                                     max_attn_len, contextual_seq_len, kv_splits, True), "delta_hstu_mha_paged")
