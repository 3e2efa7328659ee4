"""Paged 4-bit KV cache: requests of different lengths that come and go share a pool of pages, and attention of their new
tokens - one each, drafts, prompt chunks - reads the pages as they lie.  The four-segment cache
(:mod:`hyquant_b200.d_stage_kv_cache`) serves one batch of equal lengths; this one serves a ragged batch, with every
token in 4 bits from the start (no counterpart in the reference).

One layer's pool is ``pages`` uint8 ``[num_pages, H_KV, page_size // 16, 2112]`` (:func:`paged_pages`); a block of sixteen
tokens is 16 x 64 bytes of K codes, 16 x 64 bytes of V codes, 16 bf16 K scales and 16 bf16 V scales.  A row's scale is
max|x| / 7 rounded up to bf16, within [2^-17, 9344], and its codes are clamp(rint(x / scale), -7, 7), packed as
:func:`hyquant_b200.quantize_per_token` packs four bits.  Every value code * scale is an fp16 number: attention works on the
cache's values without rounding them again.  Values beyond +-65408 saturate; a NaN takes code -7.

A step is: :func:`page_advance` (block tables, slots, positions - once for all layers), then per layer :func:`paged_append`
and :func:`paged_attention`.  All of it stays on the device, allocates only its outputs (and attention its scratch) and
can be captured in a CUDA graph.  Nothing here has gradients.  :class:`PagedKVCache` keeps the state of a whole model.
"""

from __future__ import annotations

import ctypes as C
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import HyQuantError, PageAdvanceArgs, PagedAttentionArgs

BLOCK = 16                  # tokens of a block
BLOCK_BYTES = 2112
PAGE_SIZES = (16, 32, 64, 128)
STATUS = {1: "too few free pages", 2: "a request longer than its table row", 4: "more new tokens than max_tokens",
          8: "arguments that do not fit the state"}

_I32, _I64 = torch.int32, torch.int64


# Argument blocks as bytes: a block is read during the call and not kept, and packing one costs a fifth of filling a ctypes
# structure.  The fields are those of PageAdvanceArgs and PagedAttentionArgs.
_ADVANCE_BYTES, _ARGS_BYTES = C.sizeof(PageAdvanceArgs), C.sizeof(PagedAttentionArgs)
_pack_advance, _pack_args = struct.Struct("@6i15q").pack, struct.Struct("@10ifi14q").pack


class PageStep(NamedTuple):
    """What :func:`page_advance` gives.  ``slots`` int64 [max_tokens] (-1 behind the last token), ``positions`` int32 [max_tokens],
    ``cu_q`` int32 [R + 1]; ``kv_lens``, ``held`` int32 [R] and ``free_count`` int32 [1] are the state after the step;
    ``status`` int32 [1] is 0 unless the step was refused (:data:`STATUS`)."""
    kv_lens: torch.Tensor
    held: torch.Tensor
    free_count: torch.Tensor
    cu_q: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    status: torch.Tensor


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)       # without the check for a first use


def _call(fn, dev, *args) -> int:
    """One library call on the current stream of ``dev``, which need not be the current device."""
    if dev.index != _current_device():
        with torch.cuda.device(dev):
            return fn(*args, _lib.stream_ptr(dev))
    return fn(*args, _lib.stream_ptr(dev))


def paged_pages(num_pages: int, num_kv_heads: int, page_size: int = 64, device="cuda") -> torch.Tensor:
    """An empty pool of one layer."""
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return torch.zeros(num_pages, num_kv_heads, page_size // BLOCK, BLOCK_BYTES, dtype=torch.uint8, device=device)


def _pool(pages: torch.Tensor) -> Tuple[int, int, int]:
    """(num_pages, H_KV, page_size) of a pool."""
    if not pages.is_cuda:
        _lib.require_cuda(pages, "pages")
    shape = pages.shape
    if pages.dtype is not torch.uint8 or len(shape) != 4 or shape[3] != BLOCK_BYTES or not pages.is_contiguous():
        raise HyQuantError(f"pages must be contiguous uint8 [num_pages, H_KV, page_size // {BLOCK}, {BLOCK_BYTES}]")
    page_size = shape[2] * BLOCK
    if page_size not in PAGE_SIZES:
        raise HyQuantError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return shape[0], shape[1], page_size


def _vector(t: torch.Tensor, n: int, dtype, device, name: str) -> int:
    """Address of a contiguous one-dimensional tensor of n entries (-1: any number)."""
    if t.dtype is dtype and t.device == device and t.dim() == 1 and (n < 0 or t.numel() == n) and t.is_contiguous():
        return t.data_ptr()
    raise HyQuantError(f"{name} must be contiguous {dtype} [{'n' if n < 0 else n}] on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _table(page_table: torch.Tensor, R: int, device) -> Tuple[int, int, int]:
    """(address, row stride, columns) of a block table."""
    if page_table.dtype is not _I32 or page_table.device != device or page_table.dim() != 2 or page_table.size(0) != R:
        raise HyQuantError(f"page_table must be int32 [{R}, max_pages] on {device}")
    cols = page_table.size(1)
    stride, one = page_table.stride()
    if cols > 1 and one != 1:
        raise HyQuantError("page_table rows must be contiguous")
    return page_table.data_ptr(), stride if R > 1 else max(cols, 1), cols


def page_advance(kv_lens: torch.Tensor, held: torch.Tensor, add: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
                 free_count: torch.Tensor, *, page_size: int, max_tokens: int, keep: Optional[torch.Tensor] = None,
                 in_place: bool = False) -> PageStep:
    """Block tables, slots and positions of one step, on the device (:class:`PageStep`).

    Request r keeps its first ``keep[r]`` cached tokens (default all of ``kv_lens[r]``; fewer drops rejected drafts, 0 ends
    the request) and takes ``add[r]`` new ones (0 is allowed).  Pages it no longer needs go onto the stack
    ``free_pages[:free_count]`` in request and page order, then missing ones are taken from its top.  ``page_table`` int32
    [R, max_pages] and ``free_pages`` change in place; ``held`` int32 [R] says how many pages a row holds.  ``max_tokens`` is
    the length of ``slots`` and ``positions``, at least the sum of ``add``.  ``in_place`` writes the new ``kv_lens``, ``held`` and
    ``free_count`` over the old.

    A step that cannot be done changes nothing and sets ``status``; its ``cu_q`` is 0 throughout and its slots -1, so that appending
    and attention do nothing with it."""
    if not kv_lens.is_cuda:
        _lib.require_cuda(kv_lens, "kv_lens")
    if kv_lens.dim() != 1:
        raise HyQuantError("kv_lens must be int32 [R]")
    dev, R = kv_lens.device, kv_lens.numel()
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if max_tokens < 0:
        raise ValueError(f"max_tokens must be >= 0, got {max_tokens}")
    lens_p, held_p, add_p = _vector(kv_lens, R, _I32, dev, "kv_lens"), _vector(held, R, _I32, dev, "held"), _vector(add, R, _I32, dev, "add")
    keep_p = 0 if keep is None else _vector(keep, R, _I32, dev, "keep")
    free_p, count_p = _vector(free_pages, -1, _I32, dev, "free_pages"), _vector(free_count, 1, _I32, dev, "free_count")
    table_p, stride, cols = _table(page_table, R, dev)
    slots = kv_lens.new_empty(max_tokens, dtype=_I64)
    if in_place:
        ints = kv_lens.new_empty(R + 2 + max_tokens)
        cu_q, positions, status = ints.unsafe_split_with_sizes((R + 1, max_tokens, 1))
        lens2, held2, count2, lens2_p, held2_p, count2_p = kv_lens, held, free_count, lens_p, held_p, count_p
        base = ints.data_ptr()
    else:
        ints = kv_lens.new_empty(3 * R + 3 + max_tokens)
        cu_q, positions, status, lens2, held2, count2 = ints.unsafe_split_with_sizes((R + 1, max_tokens, 1, R, R, 1))
        base = ints.data_ptr()
        lens2_p = base + 4 * (R + 2 + max_tokens)
        held2_p, count2_p = lens2_p + 4 * R, lens2_p + 8 * R
    rc = _call(_lib.lib().hq_page_advance, dev, _pack_advance(
        _ADVANCE_BYTES, R, max_tokens, page_size, cols, free_pages.numel(), lens_p, held_p, add_p, keep_p, table_p, stride, free_p, count_p,
        lens2_p, held2_p, count2_p, base, slots.data_ptr(), base + 4 * (R + 1), base + 4 * (R + 1 + max_tokens)))
    if rc != 0:
        _lib.check(rc, "hq_page_advance")
    return PageStep(lens2, held2, count2, cu_q, slots, positions, status)


def paged_append(pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise rows ``k``, ``v`` [T, H_KV, 128] (bf16, fp16 or fp32, views are fine) into their slots of ``pages``.  Slots that are -1
    or outside the pool are skipped; the others of one call are distinct."""
    num_pages, H, page_size = _pool(pages)
    T, dev = slots.numel(), pages.device
    if k.shape != (T, H, 128) or v.shape != k.shape or k.dtype is not v.dtype or k.device != dev or v.device != dev:
        raise HyQuantError(f"k and v must be [{T}, {H}, 128] of one dtype on {dev}, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
    code = _lib.dtype_code(k.dtype)
    slots_p = _vector(slots, T, _I64, dev, "slots")
    k, k_p, k_st, k_sh = _rows(k)
    v, v_p, v_st, v_sh = _rows(v)
    rc = _call(_lib.lib().hq_paged_append, dev, k_p, v_p, code, k_st, k_sh, v_st, v_sh, T, H, slots_p, pages.data_ptr(), num_pages, page_size)
    if rc != 0:
        _lib.check(rc, "hq_paged_append")


def _rows(x: torch.Tensor):
    """(x, address, strides) with rows of 128 that the kernels read in 16-byte pieces; of a copy if x has none."""
    st, sh, sd = x.stride()
    address = x.data_ptr()
    if sd == 1 and not (st | sh) & 7 and not address & 15:
        return x, address, st, sh
    T, H, _ = x.shape
    st, sh = st if T > 1 else 0, sh if H > 1 else 0                        # an index of one value has no stride
    if sd != 1 or (st | sh) & 7 or address & 15:
        x = x.clone(memory_format=torch.contiguous_format)                 # (contiguous() would give back one that lies at an odd offset)
        address, st, sh = x.data_ptr(), H * 128, 128
    return x, address, st, sh


def paged_read(pages: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cache's values of ``slots`` as rows (k, v) [T, H_KV, 128] (fp16 and fp32 hold them exactly); zeros for slots outside the pool."""
    num_pages, H, page_size = _pool(pages)
    code = _lib.dtype_code(dtype)
    T, dev = slots.numel(), pages.device
    slots_p = _vector(slots, T, _I64, dev, "slots")
    k, v = pages.new_empty(T, H, 128, dtype=dtype), pages.new_empty(T, H, 128, dtype=dtype)
    rc = _call(_lib.lib().hq_paged_read, dev, pages.data_ptr(), num_pages, page_size, slots_p, T, H, code, k.data_ptr(), v.data_ptr())
    if rc != 0:
        _lib.check(rc, "hq_paged_read")
    return k, v


def paged_attention(q: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor, *,
                    cu_q: Optional[torch.Tensor] = None, max_q_len: int = 1, sm_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of new tokens ``q`` [T, H_Q, 128] (bf16 or fp16) over the cache, which holds them already -> [T, H_Q, 128].

    Request r has the rows ``cu_q[r] .. cu_q[r + 1]`` of ``q`` (without ``cu_q``: row r, one each) and ``kv_lens[r]`` cached tokens
    with them; its token i of n sees the first ``kv_lens[r] - n + i + 1`` of them, and gets zeros if there is none.  A length past the
    table counts as the table's.
    ``max_q_len`` is the most tokens of a request (tokens beyond it are not computed).  ``sm_scale`` (0 or more) is 128 ** -0.5 by default.
    ``out`` may be ``q`` and shares nothing else with the arguments; its rows do not overlap, and those behind the last token stay
    as they are (without ``out`` they are not initialised)."""
    num_pages, H, page_size = _pool(pages)
    dev, dtype, shape = pages.device, q.dtype, q.shape
    if len(shape) != 3 or shape[2] != 128 or q.device != dev:
        raise HyQuantError(f"q must be [T, H_Q, 128] on {dev}, got {tuple(shape)} on {q.device}")
    if dtype is torch.bfloat16:
        code = _lib.HQ_BF16
    elif dtype is torch.float16:
        code = _lib.HQ_F16
    else:
        raise HyQuantError(f"q must be bf16 or fp16, got {dtype}")
    T, H_Q, _ = shape
    R = kv_lens.numel()
    lens_p = _vector(kv_lens, R, _I32, dev, "kv_lens")
    table_p, stride, cols = _table(page_table, R, dev)
    if cu_q is None:
        if T != R or max_q_len != 1:
            raise HyQuantError(f"without cu_q every request has one token: q has {T} rows, kv_lens {R}, max_q_len {max_q_len}")
        cu_p = 0
    else:
        cu_p = _vector(cu_q, R + 1, _I32, dev, "cu_q")
        if max_q_len < 1:
            raise ValueError(f"max_q_len must be >= 1, got {max_q_len}")
    q, q_p, q_st, q_sh = _rows(q)
    if out is None:
        out = q.new_empty(T, H_Q, 128)
        o_st, o_sh = H_Q * 128, 128
    else:
        if out.shape != shape or out.dtype is not dtype or out.device != dev or out.stride(2) != 1:
            raise HyQuantError(f"out must be {tuple(shape)} {dtype} on {dev} with contiguous rows")
        o_st, o_sh, _ = out.stride()
    a = [_ARGS_BYTES, R, T, H_Q, H, 128, page_size, cols, max_q_len, code, 128 ** -0.5 if sm_scale is None else sm_scale, 0, num_pages,
         q_p, q_st, q_sh, pages.data_ptr(), table_p, stride, lens_p, cu_p, out.data_ptr(), o_st, o_sh, 0, 0]
    need = _workspace_bytes(a, dev)
    if need:
        ws = pages.new_empty(need)
        a[24], a[25] = ws.data_ptr(), need
    rc = _call(_lib.lib().hq_paged_attention, dev, _pack_args(*a))
    if rc != 0:
        _lib.check(rc, "hq_paged_attention")
    return out


_workspace: dict = {}


def _workspace_bytes(a, dev) -> int:
    """Scratch of a call.  It depends on the heads, the longest request and, for short tables, the number of requests, so that the
    answers for a device are few."""
    key = dev.index, a[3], a[4], a[8], a[1] if a[1] == 0 or a[6] * a[7] <= 1024 else -1, a[2] > 0
    need = _workspace.get(key)
    if need is None:
        n = C.c_int64()
        _lib.check(_call(lambda block, out, stream: _lib.lib().hq_paged_attention_workspace_bytes(block, out), dev, _pack_args(*a), C.byref(n)),
                   "hq_paged_attention_workspace_bytes")
        if len(_workspace) > 4096:
            _workspace.clear()
        need = _workspace[key] = n.value
    return need


class PagedKVCache:
    """State of a model's paged cache: a pool of pages per layer, one block table, stack of free pages and set of lengths for
    all layers.  ``advance`` once per step, then ``append`` and ``attention`` per layer; buffers keep their addresses, so that a
    whole step can be captured in a CUDA graph (``add`` and ``keep`` are read on the device).

    Requests live in ``max_requests`` rows; a row of length 0 is free.  ``kv_lens`` are the cached tokens of each row."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, *, max_requests: int, max_pages_per_request: int,
                 page_size: int = 64, device="cuda"):
        if min(num_layers, num_pages, num_kv_heads, max_requests, max_pages_per_request) < 1:
            raise ValueError("sizes of a paged cache must be positive")
        self.page_size = page_size
        self.pages = [paged_pages(num_pages, num_kv_heads, page_size, device) for _ in range(num_layers)]
        dev = self.pages[0].device
        self.page_table = torch.full((max_requests, max_pages_per_request), -1, dtype=_I32, device=dev)
        self.kv_lens = torch.zeros(max_requests, dtype=_I32, device=dev)
        self.held = torch.zeros(max_requests, dtype=_I32, device=dev)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=_I32, device=dev)      # page 0 on top
        self.free_count = torch.full((1,), num_pages, dtype=_I32, device=dev)
        self.step: Optional[PageStep] = None

    def __len__(self):
        return len(self.pages)

    def advance(self, add: torch.Tensor, *, max_tokens: int, keep: Optional[torch.Tensor] = None) -> PageStep:
        """Next step: ``add`` [max_requests] new tokens, ``keep`` tokens of the cached ones (:func:`page_advance`)."""
        self.step = page_advance(self.kv_lens, self.held, add, self.page_table, self.free_pages, self.free_count,
                                 page_size=self.page_size, max_tokens=max_tokens, keep=keep, in_place=True)
        return self.step

    def check(self) -> None:
        """Raise if the last step was refused (reads the status: waits for the device)."""
        why = 0 if self.step is None else int(self.step.status.item())
        if why:
            raise HyQuantError("the step was refused: " + ", ".join(text for bit, text in STATUS.items() if why & bit))

    def _step(self) -> PageStep:
        if self.step is None:
            raise HyQuantError("advance() comes before append(), attention() and read()")
        return self.step

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The step's rows of one layer, [max_tokens, H_KV, 128] (:func:`paged_append`)."""
        paged_append(self.pages[layer], k, v, self._step().slots)

    def attention(self, layer: int, q: torch.Tensor, *, max_q_len: int, sm_scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The step's tokens of one layer, [max_tokens, H_Q, 128] (:func:`paged_attention`)."""
        return paged_attention(q, self.pages[layer], self.page_table, self.kv_lens, cu_q=self._step().cu_q, max_q_len=max_q_len,
                               sm_scale=sm_scale, out=out)

    def read(self, layer: int, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        """Rows of one layer by slot (:func:`paged_read`)."""
        return paged_read(self.pages[layer], slots, dtype)
