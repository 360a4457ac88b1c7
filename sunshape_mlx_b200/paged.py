"""Serving over paged KV caches held in 4 bits.

The reference's caches hold sequences of equal length in one array per layer
(cache.py:59-336). A server's requests have lengths of their own and come and
go, so here tokens live in pages that a table assigns to requests:

  plan_step / release_pages   block tables, slot maps and lengths, on the GPU
  int4_append / int4_fetch    rows quantised into pages by slot, and read back
  int4_attention              attention of ragged requests over the pages
  PageTables                  the tables and the free pages of a server
  Int4PagedKVCache            one layer's pages

A page pool is uint8 (n_pages, n_kv_heads, page_size * head_dim * 5 / 4): keys
and values in groups of 32 dims with an fp16 scale and zero, 5 bits a value
(``value = code * scale + zero``, as ``quantize_values`` defines it).
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib as L
from .attention import workspace_for

__all__ = ["StepPlan", "plan_step", "release_pages", "int4_append", "int4_fetch",
           "int4_attention", "int4_pool", "PageTables", "Int4PagedKVCache"]

_HEAD_DIMS = (64, 128, 256)
_INT_MAX = 2 ** 31 - 1  # of the C interface's sizes
_STATUS = {1: "the page pool has too few free pages", 2: "a request needs more pages than its table row holds",
           4: "the new tokens exceed n_tokens", 8: "more pages were released than the pool has out"}


class StepPlan(NamedTuple):
    """What a step needs to know about its requests, all on the GPU.

    cu_q (n + 1,) int32: first token of each request; positions, requests
    int32 and slots int64 (n_tokens,): of each token (0, -1, -1 past the last
    one); seq_lens (n,) int32 and n_free (1,) int32: after the step; status
    (1,) int32: 0, or why nothing was allocated (``PageTables.check``).
    """

    cu_q: torch.Tensor
    positions: torch.Tensor
    requests: torch.Tensor
    slots: torch.Tensor
    seq_lens: torch.Tensor
    n_free: torch.Tensor
    status: torch.Tensor


_I32, _I64, _U8 = torch.int32, torch.int64, torch.uint8


def _int32(name: str, t: torch.Tensor, dims: int, index: int) -> None:
    if t.dtype is not _I32 or t.dim() != dims or t.get_device() != index or (t.size(-1) > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be a contiguous {dims}-D int32 tensor on CUDA device {index}")


def _check_tables(seq_lens, block_table, free_pages, n_free, page_size) -> int:
    """Checks what a step's tables share; returns the index of their device."""
    if not seq_lens.is_cuda:
        L.require_cuda(seq_lens)
    index = seq_lens.get_device()
    _int32("seq_lens", seq_lens, 1, index)
    _int32("block_table", block_table, 2, index)
    _int32("free_pages", free_pages, 1, index)
    _int32("n_free", n_free, 1, index)
    if block_table.size(0) != seq_lens.size(0) or n_free.size(0) != 1:
        raise ValueError("block_table needs a row per request, n_free one element")
    if block_table.size(0) > 1 and block_table.stride(0) < block_table.size(1):
        raise ValueError("the rows of block_table must not overlap")
    if page_size < 16 or page_size % 16 or page_size > _INT_MAX:
        raise ValueError(f"page_size must be a multiple of 16 below 2^31, got {page_size}")
    return index


def _row_stride(table: torch.Tensor) -> int:
    return max(table.stride(0), table.size(1))  # a single row has any stride


def plan_step(seq_lens: torch.Tensor, q_lens: torch.Tensor, block_table: torch.Tensor,
              free_pages: torch.Tensor, n_free: torch.Tensor, *, page_size: int,
              n_tokens: int) -> StepPlan:
    """Block tables and slot maps of a step, from the requests' lengths.

    seq_lens, q_lens (n,) int32: tokens held and new tokens of each request.
    New pages are popped from the stack ``free_pages[:n_free]`` and entered
    into ``block_table`` (n, width), the only argument that changes: lengths
    and the count of free pages after the step are returned, so a repeated
    call repeats its result. The stack has a place for every page of the pool
    (its length is the pool's size: a page past it maps to slot -1).
    ``n_tokens`` is the number of token places (a
    step of fewer tokens leaves slots of -1 at the end). If the step does not
    fit, nothing is allocated and ``status`` says why.
    """
    t = (L._fast or L.fast()).plan_step(seq_lens, q_lens, block_table, free_pages, n_free, page_size, n_tokens)
    if t is not None:
        return StepPlan._make(t)
    index = _check_tables(seq_lens, block_table, free_pages, n_free, page_size)
    _int32("q_lens", q_lens, 1, index)
    n = seq_lens.size(0)
    if q_lens.size(0) != n:
        raise ValueError("q_lens and seq_lens must have one element per request")
    if n_tokens < 0:
        raise ValueError("n_tokens must not be negative")
    slots = torch.empty(n_tokens, dtype=_I64, device=seq_lens.device)
    out = torch.empty(2 * n + 3 + 2 * n_tokens, dtype=_I32, device=seq_lens.device)
    cu, pos, req, lens, left, status = out.split_with_sizes((n + 1, n_tokens, n_tokens, n, 1, 1))
    at = out.data_ptr()
    at_pos = at + 4 * (n + 1)
    at_req = at_pos + 4 * n_tokens
    at_lens = at_req + 4 * n_tokens
    L.launch("ss_plan_step", index, seq_lens.data_ptr(), q_lens.data_ptr(), n, block_table.data_ptr(),
             _row_stride(block_table), block_table.size(1), free_pages.data_ptr(), free_pages.size(0),
             n_free.data_ptr(), page_size, n_tokens, at, at_pos, at_req, slots.data_ptr(), at_lens,
             at_lens + 4 * n, at_lens + 4 * n + 4)
    return StepPlan(cu, pos, req, slots, lens, left, status)


def release_pages(seq_lens: torch.Tensor, done: torch.Tensor, block_table: torch.Tensor,
                  free_pages: torch.Tensor, n_free: torch.Tensor, *, page_size: int):
    """Pushes the pages of every request with ``done`` (n,) bool back onto the
    stack ``free_pages`` and clears its table row (-1). Returns (seq_lens,
    n_free, status) after it."""
    index = _check_tables(seq_lens, block_table, free_pages, n_free, page_size)
    n = seq_lens.size(0)
    if done.dtype is not torch.bool or done.shape != (n,) or done.get_device() != index or not done.is_contiguous():
        raise ValueError("done must be a contiguous bool tensor with one element per request")
    lens, left, status = torch.empty(n + 2, dtype=_I32, device=seq_lens.device).split_with_sizes((n, 1, 1))
    L.launch("ss_release_pages", index, seq_lens.data_ptr(), done.data_ptr(), n, block_table.data_ptr(),
             _row_stride(block_table), block_table.size(1), free_pages.data_ptr(), free_pages.size(0),
             n_free.data_ptr(), page_size, lens.data_ptr(), left.data_ptr(), status.data_ptr())
    return lens, left, status


# ------------------------------------------------------------------ pages

def int4_pool(n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, device="cuda") -> torch.Tensor:
    """A page pool: uint8 (n_pages, n_kv_heads, page_size * head_dim * 5 / 4),
    uninitialised (bits that no token was written to are never used)."""
    if n_pages < 1 or n_kv_heads < 1:
        raise ValueError("n_pages and n_kv_heads must be positive")
    _page_tokens(page_size * head_dim * 5 // 4, head_dim)
    return torch.empty((n_pages, n_kv_heads, page_size * head_dim * 5 // 4), dtype=torch.uint8, device=device)


def _page_tokens(nbytes: int, head_dim: int) -> int:
    """page_size of a pool whose pages of one head have nbytes."""
    if head_dim not in _HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if nbytes < 20 * head_dim or nbytes % (20 * head_dim):
        raise ValueError(f"pages of {nbytes} bytes do not hold a multiple of 16 tokens of head_dim {head_dim}")
    return nbytes * 4 // (5 * head_dim)


def _check_pool(pages: torch.Tensor, head_dim: int) -> int:
    if not pages.is_cuda:
        L.require_cuda(pages)
    if pages.dtype is not _U8 or pages.dim() != 3 or pages.stride(2) != 1 or not pages.size(0) or not pages.size(1):
        raise ValueError("pages must be uint8 (n_pages, n_kv_heads, bytes), not empty, contiguous in the last dim")
    return _page_tokens(pages.size(2), head_dim)


def _check_slots(slots: torch.Tensor, n: int, index: int) -> None:
    if slots.dtype is not _I64 or slots.dim() != 1 or slots.size(0) != n or slots.get_device() != index or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int64 tensor with one element per token, on the pages' device")


def int4_append(keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor, pages: torch.Tensor) -> None:
    """Quantises keys and values (n, n_kv_heads, head_dim), fp32, fp16 or
    bf16, into the pages at ``slots`` (n,) int64; -1 skips a token. Slots of
    one call must differ. No gradient reaches what is stored. Magnitudes above 2^15 saturate; a NaN makes its
    group of 32 dims read as NaN."""
    if (L._fast or L.fast()).append(keys, values, slots, pages):
        return
    if not (keys.is_cuda and values.is_cuda):
        L.require_cuda(keys, values)
    if keys.dim() != 3 or keys.shape != values.shape or keys.dtype is not values.dtype:
        raise ValueError("keys and values must be (n, n_kv_heads, head_dim) of one shape and dtype")
    n, h, d = keys.shape
    page = _check_pool(pages, d)
    index = pages.get_device()
    if pages.size(1) != h:
        raise ValueError(f"the pages hold {pages.size(1)} kv heads, got {h}")
    if keys.get_device() != index or values.get_device() != index:
        raise ValueError("keys, values and pages must be on one device")
    ks, vs = keys.stride(), values.stride()
    if n and (ks[2] != 1 or vs[2] != 1):
        raise ValueError("keys and values must be contiguous in head_dim")
    _check_slots(slots, n, index)
    L.launch("ss_int4_append", index, keys.data_ptr(), values.data_ptr(), L.dtype_code(keys.dtype), ks[0], ks[1],
             vs[0], vs[1], slots.data_ptr(), n, h, d, pages.data_ptr(), pages.size(0), pages.stride(0),
             pages.stride(1), page)


def int4_fetch(slots: torch.Tensor, pages: torch.Tensor, head_dim: int, *,
               dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values (n, n_kv_heads, head_dim) as the pages hold them at
    ``slots``; zeros where a slot is -1."""
    dt = L.dtype_code(dtype)
    kv = (L._fast or L.fast()).fetch(slots, pages, head_dim, dt)
    if kv is not None:
        return kv
    page = _check_pool(pages, head_dim)
    index, n, h = pages.get_device(), slots.numel(), pages.size(1)
    _check_slots(slots, n, index)
    k = torch.empty((n, h, head_dim), dtype=dtype, device=pages.device)
    v = torch.empty_like(k)
    L.launch("ss_int4_fetch", index, slots.data_ptr(), n, h, head_dim, pages.data_ptr(), pages.size(0),
             pages.stride(0), pages.stride(1), page, k.data_ptr(), v.data_ptr(), dt)
    return k, v


# ------------------------------------------------------------------ attention

def int4_attention(queries: torch.Tensor, pages: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, cu_q: torch.Tensor, scale: float, *, max_q: int,
                   causal: bool = True, window: int = 0, return_lse: bool = False):
    """Attention of ragged requests over 4-bit pages.

    queries (n_tokens, n_q_heads, head_dim), fp16 or bf16; tokens
    ``cu_q[b]:cu_q[b + 1]`` belong to request b, whose keys are the first
    ``seq_lens[b]`` tokens of row b of ``block_table`` (the new tokens
    included), and stand at its last positions. ``causal`` hides later keys;
    ``window > 0`` also hides keys at ``position - window`` and before.
    ``max_q`` is the most query tokens of a request. Stored values enter as
    fp16(code * scale + zero), probabilities as fp16 (as a sum of two where the
    output is fp16); sums are fp32. Returns the output
    (n_tokens, n_q_heads, head_dim) in the queries' dtype and, with
    ``return_lse``, the natural log-sum-exp (n_tokens, n_q_heads) in fp32. A
    row that sees no key gives 0 and -inf, as does a token outside ``cu_q``.
    There is no gradient: queries that want one are refused.
    """
    L.poll_device_errors()
    if queries.is_cuda and pages.is_cuda and queries.dim() == 3 and queries.size(2) in _HEAD_DIMS:
        t = (L._fast or L.fast()).attention(queries, pages, block_table, seq_lens, cu_q, scale, max_q, causal, window, return_lse,
                                            _workspace(pages, queries.size(2)))
        if t is not None:
            return t if return_lse else t[0]
    if not queries.is_cuda:
        L.require_cuda(queries)
    L.refuse_graph("int4_attention", queries)
    if queries.dim() != 3:
        raise ValueError("queries must be (n_tokens, n_q_heads, head_dim)")
    n, hq, d = queries.shape
    page = _check_pool(pages, d)
    index, hkv = pages.get_device(), pages.size(1)
    if queries.dtype is not torch.float16 and queries.dtype is not torch.bfloat16:
        raise TypeError(f"queries must be fp16 or bf16, got {queries.dtype}")
    if queries.get_device() != index:
        raise ValueError("queries and pages must be on one device")
    if hq < 1 or hq % hkv:
        raise ValueError("n_q_heads must be a multiple of n_kv_heads")
    if n and queries.stride(2) != 1:
        raise ValueError("queries must be contiguous in head_dim")
    _int32("block_table", block_table, 2, index)
    _int32("seq_lens", seq_lens, 1, index)
    _int32("cu_q", cu_q, 1, index)
    b = seq_lens.size(0)
    if not b or block_table.size(0) != b or cu_q.size(0) != b + 1 or not block_table.size(1):
        raise ValueError("block_table and seq_lens need a row per request, cu_q one element more")
    if max_q < 1 or window < 0:
        raise ValueError("max_q must be positive and window not negative")
    out = torch.empty((n, hq, d), dtype=queries.dtype, device=pages.device)
    lse = torch.empty((n, hq), dtype=torch.float32, device=pages.device) if return_lse else None
    if n:
        ws = _workspace(pages, d)
        a = L.Int4AttnArgs(queries.data_ptr(), L.dtype_code(queries.dtype), queries.stride(0),
                           queries.stride(1), n, hq, hkv, d, pages.data_ptr(), pages.size(0),
                           pages.stride(0), pages.stride(1), page, block_table.data_ptr(),
                           block_table.stride(0), block_table.size(1), seq_lens.data_ptr(),
                           cu_q.data_ptr(), b, min(max_q, _INT_MAX), scale, 1 if causal else 0, min(window, _INT_MAX),
                           out.data_ptr(), lse.data_ptr() if return_lse else None, ws.data_ptr(), ws.numel())
        L.launch("ss_int4_attention", index, C.byref(a))
    return (out, lse) if return_lse else out


# The kernels' scratch belongs to a stream: (device, stream, head_dim) -> workspace.
_WS: dict[tuple, torch.Tensor] = {}
# That of captured calls to their graph, which may run on any stream and at any time: the same
# key -> (capture, workspace) of the last capture.
_GRAPH_WS: dict[tuple, tuple] = {}


def _workspace(pages: torch.Tensor, head_dim: int) -> torch.Tensor:
    index = pages.get_device()
    if L.current_device() != index:
        with torch.cuda.device(index):
            return _workspace(pages, head_dim)
    key = (index, L.raw_stream(index), head_dim)
    if L.capturing():
        return _graph_workspace(pages.device, key)
    ws = _WS.get(key)
    if ws is None:
        ws = workspace_for(pages.device, L.entry("ss_int4_attention_workspace")(head_dim), f"int4-{head_dim}")
        _WS[key] = ws
    return ws


def _graph_workspace(device: torch.device, key: tuple) -> torch.Tensor:
    """Scratch of the calls that one capture has on this stream, in the graph's own
    memory, its counters cleared by the graph before the first of them."""
    now = C.c_ulonglong()
    L.call("ss_stream_capture_id", key[1], C.byref(now))
    held = _GRAPH_WS.get(key)
    if held is None or held[0] != now.value:
        ws = torch.empty(L.entry("ss_int4_attention_workspace")(key[2]), dtype=torch.uint8, device=device)
        ws[:L.entry("ss_int4_attention_counters")()].zero_()
        # kept while the capture goes on; afterwards the graph's memory stays the graph's
        held = _GRAPH_WS[key] = now.value, ws
    return held[1]


# ------------------------------------------------------------------ a server's state

class PageTables:
    """The block tables, lengths and free pages of a server's requests,
    shared by the caches of all layers. Rows are request slots: a row whose
    request ended (``release``) serves a new one from length 0."""

    def __init__(self, n_pages: int, page_size: int, max_requests: int, max_pages: int, device="cuda"):
        if n_pages < 1 or max_requests < 1 or max_pages < 1:
            raise ValueError("n_pages, max_requests and max_pages must be positive")
        if page_size < 16 or page_size % 16 or page_size > _INT_MAX:
            raise ValueError(f"page_size must be a multiple of 16 below 2^31, got {page_size}")
        self.n_pages, self.page_size = n_pages, page_size
        self.device = torch.device(device)
        self.block_table = torch.full((max_requests, max_pages), -1, dtype=torch.int32, device=self.device)
        self.seq_lens = torch.zeros(max_requests, dtype=torch.int32, device=self.device)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=self.device)
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)

    def plan(self, q_lens: torch.Tensor, n_tokens: int) -> StepPlan:
        """Allocates the step's pages and returns its plan. A step that does
        not fit allocates nothing and maps no token; ``check`` raises then."""
        p = plan_step(self.seq_lens, q_lens, self.block_table, self.free_pages, self.n_free,
                      page_size=self.page_size, n_tokens=n_tokens)
        self.seq_lens, self.n_free = p.seq_lens, p.n_free
        self.status = self.status | p.status
        return p

    def release(self, done: torch.Tensor) -> None:
        """Ends the requests with ``done``: their pages are free again."""
        self.seq_lens, self.n_free, status = release_pages(
            self.seq_lens, done, self.block_table, self.free_pages, self.n_free, page_size=self.page_size)
        self.status = self.status | status

    def check(self) -> None:
        """Waits for the GPU and raises if a step since the last check did not fit."""
        code = int(self.status.item())
        if code:
            self.status = torch.zeros_like(self.status)
            raise RuntimeError("; ".join(m for bit, m in _STATUS.items() if code & bit))


class Int4PagedKVCache:
    """One layer's keys and values in 4-bit pages, placed by a ``PageTables``."""

    def __init__(self, tables: PageTables, n_kv_heads: int, head_dim: int):
        self.tables, self.n_kv_heads, self.head_dim = tables, n_kv_heads, head_dim
        self.pages = int4_pool(tables.n_pages, n_kv_heads, tables.page_size, head_dim, tables.device)

    def append(self, keys: torch.Tensor, values: torch.Tensor, plan: StepPlan) -> None:
        """Stores the step's keys and values (n_tokens, n_kv_heads, head_dim)."""
        int4_append(keys, values, plan.slots, self.pages)

    def fetch(self, slots: torch.Tensor, dtype: torch.dtype = torch.float32):
        """Keys and values as stored at ``slots``."""
        return int4_fetch(slots, self.pages, self.head_dim, dtype=dtype)

    def attend(self, queries: torch.Tensor, plan: StepPlan, scale: float, *, max_q: int,
               causal: bool = True, window: int = 0, return_lse: bool = False):
        """Attention of the step's queries over everything the requests hold."""
        return int4_attention(queries, self.pages, self.tables.block_table, plan.seq_lens, plan.cu_q,
                              scale, max_q=max_q, causal=causal, window=window, return_lse=return_lse)

    @property
    def nbytes(self) -> int:
        return self.pages.numel()
