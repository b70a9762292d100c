"""Many sequences over one pool of resident pages.

A page is a resident block (16 tokens) of every kv head of a layer, in the form of
:class:`latticequant_amd.llm.resident.ResidentKV`; a sequence is a row of page numbers,
so sequences of any lengths share a pool, grow by a page at a time and may share pages
(a common prompt).  Where the cache of the reference grows every sequence of a batch
together (llm/compressed_kv_cache.py:384-395), here each has its own length.

* ``PagedKV`` is the pool: ``write`` quantises rows into pages, ``read`` gives them back;
* ``paged_decode_attention`` attends one new token of each sequence to its pages and its
  fp16 / bf16 tail, and keeps account of the softmax weight that each page received;
* ``evict_pages`` shortens the sequences to the pages of most weight: their numbers leave
  the table, nothing is copied.

None of it waits for the device, except ``write``: of more than 64 blocks (pages times heads), and
where only the count of exceptions tells whether the list is long enough.
"""
from __future__ import annotations

import ctypes
from array import array
from typing import NamedTuple, Optional

import torch

from .. import _lib as L
from .._dev import int32_on
from .resident import HD, RB, ResidentKV
from .tree import _DTYPES, _ints, _rows

PAGE = RB        # tokens of a page


def _no_grad(what: str, *ts) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: detach its inputs or call it under torch.no_grad()")


class _Pool(ResidentKV):
    """The resident form behind a PagedKV: its exception list has the entries' records beside it."""

    _by_number = True

    def __init__(self, n_heads: int, n_pages: int, device, exc_cap: int):
        super().__init__(n_heads, n_pages * PAGE, device=device, exc_cap=exc_cap)
        self.n_tokens = n_pages * PAGE
        self.room = torch.zeros(n_heads * n_pages, dtype=torch.int32, device=self.a.device)
        self.rec = torch.zeros(exc_cap, dtype=torch.uint8, device=self.a.device)
        self._pages = self._pages_of = None

    def _grow_exc(self, cap: int, keep: int) -> None:
        grown = torch.zeros(cap, dtype=torch.uint8, device=self.device)
        grown[:keep] = self.rec[:keep]
        super()._grow_exc(cap, keep)           # (where memory runs out, both are as they were)
        self.rec = grown

    def pages(self) -> L.Pages:
        """The buffers as the C ABI's lq_pages (cached with the struct() that it holds)."""
        st = self.struct()
        if self._pages_of is not st:
            self._pages, self._pages_of = L.Pages(r=st, room=self.room.data_ptr(), rec=self.rec.data_ptr()), st
        return self._pages


class PagedKV:
    """A pool of n_pages pages of n_heads kv heads (K or V of a layer).

    exc_cap: room for exceptions (vectors outside the 5-bit range), by default eight a
    page and head.  ``write`` lengthens the list, which moves it, where it is too short: where
    the entries in use and 256 more for each page and head that is written (of which a write
    of more than 64 counts only those it turns out to need) do not fit.  A page has the next power
    of two of its largest number of exceptions in use, and under as many again of
    earlier ones: 512 a page and head and 256 a page and head of a write always suffice.
    A graph captured over the pool holds the list as it was: capture again when
    ``exc_cap`` has grown.  Calls on one pool from several streams are the caller's to order,
    whichever pages they name: a write may move the list that the others read."""

    def __init__(self, n_heads: int, n_pages: int, device=None, exc_cap: Optional[int] = None):
        if n_heads < 1 or n_pages < 1:
            raise ValueError("n_heads and n_pages must be positive")
        if n_heads * n_pages > 2 ** 31 - 1:
            raise ValueError("a pool has fewer than 2^31 pages in all its heads")
        if exc_cap is None:
            exc_cap = max(4096, 8 * n_heads * n_pages)
        self.pool = _Pool(n_heads, n_pages, device, exc_cap)
        self.n_heads, self.n_pages, self.device = int(n_heads), int(n_pages), self.pool.a.device

    @property
    def exc_cap(self) -> int:
        return self.pool.exc_cap

    def struct(self) -> L.Pages:
        return self.pool.pages()

    def _numbers(self, pages: torch.Tensor, shape, write: bool) -> torch.Tensor:
        if not isinstance(pages, torch.Tensor) or pages.dtype not in (torch.int32, torch.int64):
            raise ValueError("pages must be an int32 or int64 tensor")
        if shape is not None and pages.shape != shape:
            raise ValueError(f"pages must have shape {tuple(shape)}, not {tuple(pages.shape)}")
        if pages.device.type == "cpu" or L.debug_checks():
            if pages.numel() and (int(pages.min()) < 0 or int(pages.max()) >= self.n_pages):
                raise ValueError("page number outside the pool")
            if write and pages.unique().numel() != pages.numel():
                raise ValueError("a page stands twice")
        return int32_on(pages, self.device)

    def write(self, x: torch.Tensor, pages: torch.Tensor, scale32: Optional[torch.Tensor] = None,
              scale16: Optional[torch.Tensor] = None, bits: int = 4) -> None:
        """Quantise x (n, n_heads, T, 128) fp16 / bf16 / fp32 (T a multiple of 16) into pages
        (n, T / 16), each the next 16 tokens of its row.  scale32 / scale16: the rows'
        scales per head, n * n_heads of each (those of the chunk codec give its points);
        without them they are taken from x at `bits` bits per dimension.  What the pages held
        is gone; all their numbers are to differ.  Numbers on the device that are outside the
        pool write nothing (from the host such, and equal ones, are refused)."""
        if x.dim() != 4 or x.shape[1] != self.n_heads or x.shape[3] != HD:
            raise ValueError(f"x must be (n, {self.n_heads}, T, 128)")
        n, H, T, _ = x.shape
        if T % PAGE:
            raise ValueError(f"pages hold {PAGE} tokens: write a multiple of {PAGE} (keep the rest in the tail)")
        if (scale32 is None) != (scale16 is None):
            raise ValueError("scale32 and scale16 go together")
        if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise ValueError("x must be fp16, bf16 or fp32")
        if pages.shape != (n, T // PAGE):
            raise ValueError(f"pages must have shape {(n, T // PAGE)}, not {tuple(pages.shape)}")
        if n * T == 0:
            return
        _no_grad("a write to pages", x, scale32, scale16)
        num = self._numbers(pages, None, True)
        lib, r = L.lib(), self.pool
        with L.on_device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a write may lengthen the exception list: not while a graph is captured")
            xc = x.to(self.device).contiguous()
            if scale32 is None:
                from ..codec import _head_scales
                _, s32, s16, _, _ = _head_scales(xc[None], bits, None)
            else:
                s32 = scale32.to(device=self.device, dtype=torch.float32).contiguous().view(-1)
                s16 = scale16.to(device=self.device, dtype=torch.float16).contiguous().view(-1)
            if s32.numel() != n * H or s16.numel() != n * H:
                raise ValueError("one scale per row and head expected")

            def launch():
                L.check(lib.lq_page_quantize(xc.data_ptr(), L.dtype_code(xc.dtype), n, T, s32.data_ptr(), s16.data_ptr(),
                                             ctypes.addressof(r.pages()), num.data_ptr(), L.raw_stream(self.device)),
                        "lq_page_quantize")
            r._with_exceptions(n * H * T * (HD // 8), launch, anew=False)

    def read(self, pages: torch.Tensor, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """(n, n_heads, m * 16, 128): the rows of pages (n, m), lattice point times the stored
        fp16 scale, rounded once (the values _decompress_chunk writes); zeros for numbers
        outside the pool."""
        if pages.dim() != 2:
            raise ValueError("pages must be (n, m) whole numbers")
        n, m = pages.shape
        out = torch.empty(n, self.n_heads, m * PAGE, HD, dtype=out_dtype, device=self.device)
        if out.numel():
            with L.on_device(self.device):
                num = self._numbers(pages, None, False)
                L.check(L.lib().lq_page_dequant(ctypes.addressof(self.struct()), num.data_ptr(), n, m, out.data_ptr(),
                                                L.dtype_code(out_dtype), L.raw_stream(self.device)), "lq_page_dequant")
        return out


def paged_workspace_size(n_seq: int, n_heads: int, group: int, max_pages: int, tail_cap: int, weights: bool = False) -> int:
    """Bytes of workspace of paged_decode_attention over pools of n_heads kv heads."""
    n = L.load().lq_paged_attn_workspace(n_seq, n_heads, group, max_pages, tail_cap, int(weights))
    if n < 0:
        raise ValueError("bad paged attention geometry")
    return n


def paged_attn_workspace(n_seq: int, n_heads: int, group: int, max_pages: int, tail_cap: int, weights: bool = False,
                         device=None) -> torch.Tensor:
    """paged_workspace_size bytes on the device, uninitialised."""
    return torch.empty(paged_workspace_size(n_seq, n_heads, group, max_pages, tail_cap, weights), dtype=torch.uint8,
                       device=device)


def _apart(out: torch.Tensor) -> bool:
    """Whether the rows of out (B, Hq, 1, 128) share no element."""
    if out.is_contiguous():
        return True
    (a, n), (b, m) = sorted(zip(out.stride()[:2], out.shape[:2]))
    if n == 1 or m == 1:
        return n * m == 1 or (b if n == 1 else a) >= HD
    return a >= HD and b >= (n - 1) * a + HD


def paged_decode_attention(k: PagedKV, v: PagedKV, q: torch.Tensor, pages: torch.Tensor, n_pages: torch.Tensor,
                           tail_k: Optional[torch.Tensor] = None, tail_v: Optional[torch.Tensor] = None,
                           tail_len: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                           decay: float = 1.0, work: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One new token of each of B sequences: softmax(q K^T / sqrt(128)) V over its pages and
    its tail (which has the new token's own K / V).

    q: (B, Hq, 1, 128) fp16 or bf16, Hq = group * n_heads (group 1..16); pages: (B, W)
    whole numbers, sequence b's pages in order in its first n_pages[b] (B,) places (the
    others are not read; W may be 0); tail_k / tail_v: (B, n_heads, cap, 128) of q's type,
    of which sequence b has the first tail_len[b] (all cap without tail_len).  Counts
    are clamped to W and cap; page numbers outside the pool read its last page.  A sequence
    without any token gets zeros.
    weights: (B, W) fp32, contiguous, the pages' accumulated weights: weights[b, j] becomes
    decay * weights[b, j] + the softmax weight that all Hq heads gave page j (decay 0: that
    alone, whatever stood there); places past n_pages[b] stay as they are.
    Any strides with a contiguous last dimension are read in place.  work:
    paged_attn_workspace, used until the call's work on the stream is done; out: where to
    write, of q's shape and type.  Returns (B, Hq, 1, 128).  The products are fp16 as
    resident_tree_attention's are; a page's value is its lattice coordinate times its scale,
    V's unrounded, K's rounded to fp16 (as ``read`` rounds it) with weights and unrounded
    without (so asking for weights moves the result by what that rounding does); coordinates
    of exceptions beyond 1024 (K's without weights 1008) have fp16's 11 bits.  The same inputs give the same bits."""
    dev = k.device
    dt, shape = q.dtype, q.shape
    if len(shape) != 4 or dt not in _DTYPES or shape[2] != 1 or shape[3] != HD:
        raise ValueError("q must be (B, Hq, 1, 128) fp16 or bf16")
    B, Hq, _, _ = shape
    H = k.n_heads
    if v.n_heads != H or v.n_pages != k.n_pages or v.device != dev:
        raise ValueError("the K and V pools must have the same heads, pages and device")
    if B < 1 or Hq < 1 or Hq % H or Hq // H > 16:
        raise ValueError("query heads must be 1..16 times the pools' heads")
    wide = pages.shape
    if len(wide) != 2 or wide[0] != B:
        raise ValueError("pages must be (B, W) whole numbers")
    W = wide[1]
    given = [q]
    cap = 0
    if tail_k is not None and tail_v is not None:
        rows = tail_k.shape
        if len(rows) != 4 or rows != tail_v.shape or rows[0] != B or rows[1] != H or rows[3] != HD:
            raise ValueError("tail K / V must be (B, n_heads, cap, 128)")
        cap = rows[2]
        if cap:
            given += [tail_k, tail_v]
    elif tail_k is not None or tail_v is not None:
        raise ValueError("tail K and V go together")
    elif tail_len is not None:
        raise ValueError("tail_len without a tail")
    for t in given:
        if t.dtype is not dt or t.device != dev:
            raise ValueError("q and the tail must be of one type, on the pools' device")
    _no_grad("paged_decode_attention", *given, weights, out)
    if weights is not None and (weights.shape != (B, W) or weights.dtype is not torch.float32 or weights.device != dev or
                                not weights.is_contiguous()):
        raise ValueError("weights must be (B, W) fp32, contiguous, on the pools' device")
    if out is not None and (out.shape != q.shape or out.dtype is not dt or out.device != dev or out.stride(3) != 1 or
                            any(s % 8 for s in out.stride()[:2]) or out.data_ptr() % 16 or not _apart(out)):
        raise ValueError("out must be like q, its rows 16-byte aligned and apart")
    lib = L.lib()
    with L.on_device(dev):
        tab = _ints(pages, wide, "pages", dev)
        cnt = _ints(n_pages, (B,), "n_pages", dev)
        tl = None if tail_len is None else _ints(tail_len, (B,), "tail_len", dev)
        if L.debug_checks():
            on = torch.arange(W, device=dev) < cnt[:, None]
            if bool((cnt < 0).any()) or bool((cnt > W).any()) or bool((on & ((tab < 0) | (tab >= k.n_pages))).any()):
                raise ValueError("page count or number out of range")
            if tl is not None and (bool((tl < 0).any()) or bool((tl > cap).any())):
                raise ValueError("tail_len out of range")
        if work is None:
            work = paged_attn_workspace(B, H, Hq // H, W, cap, weights is not None, device=dev)
        elif work.device != dev or not work.is_contiguous():
            raise ValueError("the attention workspace must be contiguous, on the pools' device")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        keep, flat = [], []                    # the copies stay until the launch; four lq_rows
        for t in given:
            t, r = _rows(t)
            keep.append(t)
            flat += r
        flat += (out.data_ptr(),) + out.stride()[:3]
        rows = array("q", flat)
        at = rows.buffer_info()[0]
        rc = lib.lq_paged_attention(
            ctypes.addressof(k.struct()), ctypes.addressof(v.struct()), at, B, Hq // H, tab.data_ptr(), W,
            cnt.data_ptr(), at + 32 if cap else None, at + 64 if cap else None, cap, None if tl is None else tl.data_ptr(),
            None if weights is None else weights.data_ptr(), decay, 0 if dt is torch.float16 else 1, work.data_ptr(),
            work.numel() * work.element_size(), at + 32 * len(given), L.raw_stream(dev))
        if rc:
            need = lib.lq_paged_attn_workspace(B, H, Hq // H, W, cap, int(weights is not None))
            if need < 0:
                raise ValueError("too many sequences, heads or tokens for one call")
            if rc == L.LQ_ERR_ARG and work.numel() * work.element_size() < need:
                raise ValueError("attention workspace too small")
            L.check(rc, "lq_paged_attention")
    return out


class Eviction(NamedTuple):
    """What evict_pages returns."""
    pages: torch.Tensor      # (B, W) int32: the kept pages in order, then -1
    n_pages: torch.Tensor    # (B,) int32
    weights: torch.Tensor    # (B, W) fp32: theirs, then 0
    freed: torch.Tensor      # (B, W) int32: the others in order, then -1


def evict_pages(pages: torch.Tensor, n_pages: torch.Tensor, weights: torch.Tensor, keep: int, sink: int = 0,
                recent: int = 0, out: Optional[Eviction] = None) -> Eviction:
    """Each sequence's pages down to `keep`, by the weights that paged_decode_attention
    accumulated: the first `sink` and the last `recent` stay, and of those between the
    ones of most weight (NaN above all; of equal ones the earlier), in their order.
    pages (B, W) whole numbers, n_pages (B,), weights (B, W) fp32, all on one device; a
    sequence of `keep` pages or fewer stays whole.  The inputs are left as they are; out: an
    earlier result whose tensors are written again.  A page freed by one sequence may still
    be another's (shared prompts): the caller counts."""
    if not isinstance(weights, torch.Tensor) or weights.dim() != 2 or weights.dtype is not torch.float32:
        raise ValueError("weights must be (B, W) fp32")
    B, W = weights.shape
    dev = weights.device
    if not 1 <= B < 2 ** 22:
        raise ValueError("at least one sequence, and fewer than 2^22")
    if sink < 0 or recent < 0 or keep < sink + recent:
        raise ValueError("keep must be at least sink + recent, and neither below 0")
    _no_grad("evict_pages", weights)
    if dev.type != "cuda":
        raise ValueError("weights must be on the GPU")
    lib = L.lib()
    with L.on_device(dev):
        tab = _ints(pages, (B, W), "pages", dev)
        cnt = _ints(n_pages, (B,), "n_pages", dev)
        w = weights.contiguous()
        if out is None:
            out = Eviction(torch.empty_like(tab), torch.empty_like(cnt), torch.empty_like(w), torch.empty_like(tab))
        else:
            for t, like in zip(out, (tab, cnt, w, tab)):
                if t.shape != like.shape or t.dtype is not like.dtype or t.device != dev or not t.is_contiguous():
                    raise ValueError("out must be an Eviction of the same shapes and device")
            spans = sorted((t.data_ptr(), t.nbytes) for t in (*out, tab, cnt, w))
            if any(at + size > behind for (at, size), (behind, _) in zip(spans, spans[1:])) and W:
                raise ValueError("out must be apart from the inputs")
        if W == 0:
            out.n_pages.zero_()
            return out
        L.check(lib.lq_evict_pages(tab.data_ptr(), cnt.data_ptr(), w.data_ptr(), B, W, min(keep, 2 * W), min(sink, W),
                                   min(recent, W), out.pages.data_ptr(), out.n_pages.data_ptr(),
                                   out.weights.data_ptr(), out.freed.data_ptr(), L.raw_stream(dev)), "lq_evict_pages")
    return out
