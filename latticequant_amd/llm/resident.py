"""Resident (fixed-width) form of a compressed KV prefix and decode attention over it.

The rANS chunks of :mod:`latticequant_amd.codec` are the cache's at-rest form,
bit-exact with the reference's bitstreams.  A decode step needs the prefix at
every step, and re-running rANS over 32k tokens per step is instruction-bound,
so the cache also keeps the same lattice points as one b = 5 fixed-rate code
word per vector (the ``pack_e8`` word of core/compact_storage.py:87-154,
split into a 32-bit and an 8-bit plane laid out for the attention kernel's
MFMA operands), with an exception entry (the lattice point as int16 2c) for
every vector outside the 5-bit range -- the representable / fallback split of
llm/fused_triton_merge.py:33-130.  At 4 bits/dim a prefix costs about 5.3 B
per 8-dim vector here, against 16 B for the fp16 cache the reference keeps
resident beside its chunks (llm/compressed_kv_cache.py:384-395).

``resident_decode_attention`` is one decode step of
softmax(q K^T / sqrt(128)) V over a resident K / V prefix plus an fp16 tail
(lq_resident_attention: MFMA for Q K^T and P V, online softmax, split-token
records merged in the same launch).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from .. import _lib as L
from .._dev import int32_on

RB = 16          # tokens per resident block
HD = 128


class ResidentKV:
    """Resident prefix of n_heads kv heads (B * H_kv), capacity cap_tokens tokens each.

    n_seq: of how many sequences the heads are (B), where a selection is to know without
    being told: given here, or that of the rows appended; None where rows of different
    groupings were."""

    _by_number = False   # a pool of pages: a block keeps its place, and exception entries of its own

    def __init__(self, n_heads: int, cap_tokens: int, device=None, exc_cap: Optional[int] = None,
                 n_seq: Optional[int] = None):
        if n_heads <= 0 or cap_tokens <= 0:
            raise ValueError("n_heads and cap_tokens must be positive")
        if n_seq is not None and (n_seq < 1 or n_heads % n_seq):
            raise ValueError("n_heads must be a multiple of n_seq")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        nb = (cap_tokens + RB - 1) // RB
        self.device = dev
        self.n_heads = int(n_heads)
        self.n_seq = n_seq
        self._n_seq_given = n_seq is not None
        self.cap_blocks = nb
        self.a = torch.zeros(n_heads * nb * 64 * 4, dtype=torch.int32, device=dev)
        self.b = torch.zeros(n_heads * nb * 64 * 4, dtype=torch.uint8, device=dev)
        self.mask = torch.zeros(n_heads * nb * 4, dtype=torch.int64, device=dev)
        self.meta = torch.zeros(n_heads * nb * 4, dtype=torch.int32, device=dev)
        self.scale = torch.zeros(n_heads * nb * RB, dtype=torch.float16, device=dev)
        self.n_exc = torch.zeros(1, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        cap = exc_cap if exc_cap is not None else max(256, n_heads * nb * 4)
        self.exc = torch.zeros(cap * 8, dtype=torch.int16, device=dev)
        self.n_tokens = 0
        # exception count as the host knows it without waiting: a count read
        # back earlier (pinned copy + event), the vectors appended after it
        # (each may add one exception), and the newest read still in flight
        self._exc_known = 0
        self._exc_since = 0
        self._exc_read = None   # (pinned count, event, vectors appended after its snapshot)
        self._st = None         # the ctypes view of the buffers, rebuilt when one is reallocated

    @property
    def exc_cap(self) -> int:
        return self.exc.numel() // 8

    def struct(self) -> L.Resident:
        """The buffers as the C ABI's lq_resident (cached: the pointers and
        capacities change only when reserve() or the exception list grows)."""
        if self._st is None:
            self._st = L.Resident(a=self.a.data_ptr(), b=self.b.data_ptr(), mask=self.mask.data_ptr(),
                                  meta=self.meta.data_ptr(), exc=self.exc.data_ptr(), scale=self.scale.data_ptr(),
                                  n_exc=self.n_exc.data_ptr(), status=self.status.data_ptr(), n_heads=self.n_heads,
                                  cap_blocks=self.cap_blocks, exc_cap=self.exc_cap)
        return self._st

    def nbytes(self) -> int:
        """Bytes a decode step reads per token range: records, masks, bases, scales, exceptions in use."""
        nb = (self.n_tokens + RB - 1) // RB
        per_blk = 64 * 4 * 4 + 64 * 4 + 16 + RB * 2   # records, meta, scales
        return self.n_heads * nb * per_blk + int(self.n_exc.item()) * 16

    def reserve(self, cap_tokens: int) -> None:
        """Grow the capacity to at least cap_tokens tokens per head (copies the blocks in use)."""
        nb = (cap_tokens + RB - 1) // RB
        if nb <= self.cap_blocks:
            return
        if self._by_number:
            raise ValueError("a pool of pages keeps its size")
        H, ob = self.n_heads, self.cap_blocks
        used = (self.n_tokens + RB - 1) // RB

        def grow(t, per_blk):
            n = torch.zeros(H * nb * per_blk, dtype=t.dtype, device=t.device)
            n.view(H, nb, per_blk)[:, :used].copy_(t.view(H, ob, per_blk)[:, :used])
            return n
        self.a = grow(self.a, 64 * 4)
        self.b = grow(self.b, 64 * 4)
        self.mask = grow(self.mask, 4)
        self.meta = grow(self.meta, 4)
        self.scale = grow(self.scale, RB)
        self.cap_blocks = nb
        self._st = None

    # appends of at most this many vectors run without a host read: the
    # exception list is grown (device copy) whenever the host's upper bound of
    # the count could pass its capacity; larger appends (a prefill) read the
    # count back instead, so that the list does not grow to the bound
    ASYNC_MAX_VECTORS = 1 << 14

    def append(self, x: torch.Tensor, scale32: torch.Tensor, scale16: torch.Tensor) -> None:
        """Quantize x (B, H, T, 128) with the per-head scales of its chunk
        (B*H of each; the points are those the chunk codec codes with the same
        scale32) and append it: T must be a multiple of 16.  Small appends (a
        decode step's flush) make no host read; larger ones grow the exception
        list to its exact need (one or two host reads of the count)."""
        if x.dim() != 4 or x.shape[3] != HD:
            raise ValueError("x must be (B, H, T, 128)")
        B, H, T, _ = x.shape
        if B * H != self.n_heads:
            raise ValueError(f"x has {B * H} heads, the resident prefix {self.n_heads}")
        if self._n_seq_given and B != self.n_seq:
            raise ValueError(f"x has {B} sequences, the resident prefix {self.n_seq}")
        if T % RB:
            raise ValueError(f"resident blocks hold {RB} tokens: append a multiple of {RB} (keep the rest in the tail)")
        if self.n_tokens % RB:
            raise ValueError("resident prefix ends inside a block")
        if self.n_tokens + T > self.cap_blocks * RB:
            raise ValueError("resident prefix capacity exceeded")
        lib = L.lib()
        xc = x.to(self.device).contiguous()
        s32 = scale32.to(device=self.device, dtype=torch.float32).contiguous().view(-1)
        s16 = scale16.to(device=self.device, dtype=torch.float16).contiguous().view(-1)
        if s32.numel() != self.n_heads or s16.numel() != self.n_heads:
            raise ValueError("one scale per head expected")
        work = torch.empty(int(lib.lq_resident_workspace(self.n_heads, T)), dtype=torch.uint8, device=self.device)
        blk0 = self.n_tokens // RB
        n_new = self.n_heads * T * (HD // 8)   # vectors appended: each can be one exception

        def launch():
            st = self.struct()
            L.check(lib.lq_resident_quantize(xc.data_ptr(), L.dtype_code(xc.dtype), self.n_heads, T,
                                             s32.data_ptr(), s16.data_ptr(), ctypes.addressof(st), 0, blk0,
                                             work.data_ptr(), L.stream_ptr(self.device)), "lq_resident_quantize")

        with torch.cuda.device(self.device):
            self._with_exceptions(n_new, launch, anew=True)
        if B != self.n_seq:
            self.n_seq = None if self.n_tokens else B
        self.n_tokens += T

    def _with_exceptions(self, n_new: int, launch, anew: bool) -> None:
        """launch(), which may add n_new exception entries, with room for them.  anew: where
        the list was too short and launch runs again, its entries are numbered again (else
        those that have numbers keep them, and a graph may hold the list: it moves only where
        the entries in use and n_new do not fit, which the host may have to wait for)."""
        if n_new <= self.ASYNC_MAX_VECTORS:
            if self._exc_read is not None and self._exc_read[1].query():
                host, _, after = self._exc_read
                self._exc_known, self._exc_since, self._exc_read = int(host[0]), after, None
            need = self._exc_known + self._exc_since + n_new
            if need > self.exc_cap >= self._exc_known + n_new and not anew:
                self._exc_known, self._exc_since, self._exc_read = int(self.n_exc.item()), 0, None
                need = self._exc_known + n_new
            if need > self.exc_cap:
                self._grow_exc(self._longer(need), self.exc_cap)
            launch()
            self._exc_since += n_new
            if self._exc_read is not None:
                host, ev, after = self._exc_read
                self._exc_read = (host, ev, after + n_new)
            else:
                host = torch.empty(1, dtype=torch.int32, pin_memory=True)
                host.copy_(self.n_exc, non_blocking=True)
                ev = torch.cuda.Event()
                ev.record(torch.cuda.current_stream(self.device))
                self._exc_read = (host, ev, 0)
        else:
            n0 = int(self.n_exc.item())
            for attempt in range(2):
                launch()
                n1 = int(self.n_exc.item())
                if n1 <= self.exc_cap:
                    break
                # grow the exception list to the exact need and launch again
                if not anew:
                    self._exc_known, self._exc_since, self._exc_read = n1, 0, None   # if there is no room for it
                self._grow_exc(self._longer(n1), n0 if anew else self.exc_cap)
                if anew:
                    self.n_exc.fill_(n0)
                self.status.zero_()
            self._exc_known, self._exc_since, self._exc_read = n1, 0, None

    def _longer(self, need: int) -> int:
        """The length of a list that gets too short for `need` entries."""
        if need >= 2 ** 31 - 1:
            raise RuntimeError("an exception list has fewer than 2^31 entries")
        return min(max(2 * self.exc_cap, need), 2 ** 31 - 2)

    def _grow_exc(self, cap: int, keep: int) -> None:
        """A longer exception list holding the first `keep` entries."""
        grown = torch.zeros(cap * 8, dtype=torch.int16, device=self.device)
        grown[:keep * 8] = self.exc[:keep * 8]
        self.exc = grown
        self._st = None

    def exceptions(self) -> torch.Tensor:
        """(n, 8) int16: the exception entries in use (a host read of their number unless
        the host knows it)."""
        known = self._exc_since == 0 and self._exc_read is None
        n = self._exc_known if known else int(self.n_exc.item())
        return self.exc[:min(n, self.exc_cap) * 8].view(-1, 8)

    def reorder(self, index: torch.Tensor, t_from: int = 0) -> None:
        """reorder_sequences of this prefix alone."""
        reorder_sequences([self], index, t_from)

    def select(self, index: torch.Tensor, n_seq: Optional[int] = None, blocks: Optional[torch.Tensor] = None,
               cap_tokens: Optional[int] = None) -> "ResidentKV":
        """A new prefix of chosen sequences, and of chosen blocks of each: fork, drop,
        evict and compact.  This prefix is n_seq sequences of n_heads / n_seq heads (by
        default its own n_seq: that of the rows appended, of its construction or of the
        selection that made it); sequence r of the new one is sequence index[r] (index: (R,)
        whole numbers) and, with blocks (R, n), holds that sequence's 16-token blocks blocks[r]
        in the order given, else all of them.  The new prefix has its own exception list,
        with the entries of the chosen blocks only (their number is read back: one host
        wait), and room for cap_tokens tokens (those it holds by default).  Indices are
        clamped to their ranges."""
        if n_seq is None:
            n_seq = self.n_seq
            if n_seq is None:
                raise ValueError("how many sequences the prefix holds is not known: give n_seq")
        if n_seq < 1 or self.n_heads % n_seq:
            raise ValueError("n_heads must be a multiple of n_seq")
        if index.dim() != 1 or index.numel() < 1 or index.dtype not in (torch.int32, torch.int64):
            raise ValueError("index must be a list of sequences (int32 or int64)")
        if self.n_tokens % RB:
            raise ValueError("resident prefix ends inside a block")
        R, used, dev = index.numel(), self.n_tokens // RB, self.a.device
        if blocks is not None and (blocks.dim() != 2 or blocks.shape[0] != R or
                                   blocks.dtype not in (torch.int32, torch.int64)):
            raise ValueError("blocks must be (R, n) whole numbers")
        nb = used if blocks is None else blocks.shape[1]
        cap = max(1, nb, 0 if cap_tokens is None else (int(cap_tokens) + RB - 1) // RB)
        if nb and not used:
            raise ValueError("no blocks to choose from")
        if L.debug_checks() and (bool((index < 0).any()) or bool((index >= n_seq).any()) or
                                 (blocks is not None and nb and (bool((blocks < 0).any()) or bool((blocks >= used).any())))):
            raise ValueError("sequence or block out of range")
        heads = R * (self.n_heads // n_seq)
        if nb == 0:
            new = self._bare(heads, cap, self.n_exc.new_zeros(1), self.status.new_zeros(1))
            new.exc, new.n_seq = self.exc.new_empty(8), R
            return new
        lib = L.lib()
        need = lib.lq_select_workspace(heads, nb)
        if need < 0:
            raise ValueError("too many heads or blocks for one selection")
        read, total = ctypes.c_void_p(), ctypes.c_int64()
        with L.on_device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a selection reads its exception count back: not while a graph is captured")
            idx = int32_on(index, dev)
            blk = None if blocks is None else int32_on(blocks, dev)
            work, n_exc, status = idx.new_empty(need + 3 >> 2), self.n_exc.new_empty(1), self.status.new_empty(1)
            stream = L.raw_stream(dev)
            args = (ctypes.addressof(self.struct()), n_seq, used, idx.data_ptr(), R, L.ptr(blk), nb)
            L.check(lib.lq_select_count(*args, work.data_ptr(), need, n_exc.data_ptr(), status.data_ptr(),
                                        ctypes.addressof(read), stream), "lq_select_count")
            try:                               # the planes are allocated while the device counts
                new = self._bare(heads, cap, n_exc, status)
                dst = new.struct()
                L.check(lib.lq_resident_select(*args, ctypes.addressof(dst), work.data_ptr(), need, stream),
                        "lq_resident_select")
            finally:
                rc = lib.lq_select_total(read, ctypes.addressof(total))
            L.check(rc, "lq_select_total")
            n = total.value
            new.exc = self.exc.new_empty(max(1, n) * 8)
            dst.exc, dst.exc_cap = new.exc.data_ptr(), max(1, n)
            if n:
                L.check(lib.lq_resident_select_exceptions(*args, ctypes.addressof(dst), stream),
                        "lq_resident_select_exceptions")
        new._exc_known, new.n_tokens, new.n_seq = n, nb * RB, R
        return new

    def _bare(self, n_heads: int, nb: int, n_exc: torch.Tensor, status: torch.Tensor) -> "ResidentKV":
        """nb blocks of room per head where this prefix lies, uninitialised, with the given
        counters."""
        r = ResidentKV.__new__(ResidentKV)
        r.device, r.n_heads, r.cap_blocks, r.n_seq, r._n_seq_given = self.a.device, n_heads, nb, None, False
        n = n_heads * nb
        r.a, r.b, r.mask = self.a.new_empty(n * 256), self.b.new_empty(n * 256), self.mask.new_empty(n * 4)
        r.meta, r.scale = self.meta.new_empty(n * 4), self.scale.new_empty(n * RB)
        r.n_exc, r.status = n_exc, status
        r.exc = r.scale.view(torch.int16)[:8]   # no entry yet
        r.n_tokens = r._exc_known = r._exc_since = 0
        r._exc_read = r._st = None
        return r

    def dequant(self, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """(n_heads, n_tokens, 128): lattice point times the stored fp16 scale,
        rounded once (the values _decompress_chunk writes)."""
        lib = L.lib()
        nb = self.n_tokens // RB
        out = torch.empty(self.n_heads, nb * RB, HD, dtype=out_dtype, device=self.device)
        if nb:
            st = self.struct()
            with torch.cuda.device(self.device):
                L.check(lib.lq_resident_dequant(ctypes.addressof(st), 0, self.n_heads, 0, nb, out.data_ptr(),
                                                L.dtype_code(out_dtype), L.stream_ptr(self.device)),
                        "lq_resident_dequant")
        return out


def from_chunk(x: torch.Tensor, enc, cap_tokens: Optional[int] = None) -> ResidentKV:
    """Resident form of one chunk (x (B, H, T, 128) and its EncodedBatch enc of
    one chunk): the same lattice points as enc's bitstreams."""
    B, H, T, _ = x.shape
    r = ResidentKV(B * H, cap_tokens or T, device=x.device)
    r.append(x, enc.scale32.view(-1)[:B * H], enc.scale16.view(-1)[:B * H])
    return r


MAX_REORDER = 128   # sequences of one in-place reorder


def reorder_sequences(residents: Sequence[ResidentKV], index: torch.Tensor, t_from: int = 0) -> None:
    """Permute the sequences of resident prefixes in place (beam search): sequence i
    becomes sequence index[i] as it was, from token t_from (a multiple of 16) on; what
    lies before is the same in all sequences (the beams' prompt) and stays.  residents:
    K and V of all layers (one launch per 64), all of the same heads and tokens, on one
    device; index: (B,) whole numbers, B <= 128, heads split evenly over B.  A number may
    stand several times; one out of range leaves its sequence as it is.  No second copy
    of the cache is made; exception entries are shared by the copies."""
    if not len(residents):
        return
    r0 = residents[0]
    if index.dim() != 1 or index.dtype not in (torch.int32, torch.int64):
        raise ValueError("index must be a list of sequences (int32 or int64)")
    B, dev = index.numel(), r0.a.device
    if B < 1 or B > MAX_REORDER or r0.n_heads % B:
        raise ValueError(f"index must name 1..{MAX_REORDER} sequences that the heads divide into evenly "
                         "(more: ResidentKV.select makes a reordered copy)")
    H, T = r0.n_heads, r0.n_tokens
    if any(r._by_number for r in residents):
        raise ValueError("the blocks of a pool of pages keep their places: reorder the tables")
    for r in residents:
        if r.n_heads != H or r.n_tokens != T or r.a.device != dev:
            raise ValueError("the prefixes must have the same heads, tokens and device")
    if len(set(map(id, residents))) != len(residents):
        raise ValueError("a prefix stands twice in the list")
    if t_from < 0 or t_from % RB or t_from > r0.n_tokens or r0.n_tokens % RB:
        raise ValueError("t_from must be a multiple of 16 within the prefix")
    nb = (r0.n_tokens - t_from) // RB
    if nb == 0 or B == 1:
        return
    lib = L.lib()
    with L.on_device(dev):
        idx = int32_on(index, dev)
        if L.debug_checks() and (bool((idx < 0).any()) or bool((idx >= B).any())):
            raise ValueError("sequence out of range")
        table = b"".join([r.struct() for r in residents])   # lq_resident[]
        L.check(lib.lq_resident_reorder(table, len(residents), B, idx.data_ptr(), t_from // RB, nb, L.raw_stream(dev)),
                "lq_resident_reorder")


def attn_workspace(n_heads: int, group: int, t_prefix: int, t_tail: int, device=None) -> torch.Tensor:
    """Workspace of lq_resident_attention (counters zeroed; each call leaves them zero)."""
    n = L.lib().lq_resident_attn_workspace(n_heads, group, t_prefix, t_tail)
    if n < 0:
        raise ValueError("bad attention geometry")
    return torch.zeros(int(n), dtype=torch.uint8, device=device)


def resident_decode_attention(k: ResidentKV, v: ResidentKV, q: torch.Tensor, tail_k: Optional[torch.Tensor] = None,
                              tail_v: Optional[torch.Tensor] = None, work: Optional[torch.Tensor] = None,
                              out: Optional[torch.Tensor] = None, t_prefix: Optional[int] = None) -> torch.Tensor:
    """q: (B, Hq, 1, 128) fp16, Hq = group * H_kv (group 1..16); k / v: resident
    prefixes of B * H_kv heads; tail_k / tail_v: (B, H_kv, Tt, 128) fp16 or None.
    Returns (B, Hq, 1, 128) fp16 = softmax(q K^T / sqrt(128)) V over prefix + tail."""
    lib = L.lib()
    if k.n_heads != v.n_heads or k.n_tokens != v.n_tokens:
        raise ValueError("K and V resident prefixes must have the same geometry")
    tp = k.n_tokens if t_prefix is None else int(t_prefix)
    if tp < 0 or tp > k.n_tokens or tp % RB:
        raise ValueError("t_prefix must be a multiple of 16 within the resident prefix")
    if q.dtype != torch.float16 or q.dim() != 4 or q.shape[2] != 1 or q.shape[3] != HD:
        raise ValueError("q must be (B, Hq, 1, 128) fp16")
    B, Hq = q.shape[0], q.shape[1]
    if B < 1 or k.n_heads % B:
        raise ValueError("the resident prefix must hold B * H_kv heads")
    Hkv = k.n_heads // B
    if Hq % Hkv:
        raise ValueError("query heads must be a multiple of the kv heads")
    group = Hq // Hkv
    if not 1 <= group <= 16:
        raise ValueError("group (query heads per kv head) must be 1..16")
    dev = k.device
    tt = 0
    pk = pv = None
    if tail_k is not None and tail_k.shape[2] > 0:
        if tail_v is None or tail_k.shape != tail_v.shape or tail_k.shape[:2] != (B, Hkv) or tail_k.shape[3] != HD:
            raise ValueError("tail K / V must be (B, H_kv, Tt, 128)")
        tt = int(tail_k.shape[2])
        pk = tail_k.to(device=dev, dtype=torch.float16).contiguous()
        pv = tail_v.to(device=dev, dtype=torch.float16).contiguous()
    if tp + tt == 0:
        raise ValueError("empty prefix and tail")
    need = lib.lq_resident_attn_workspace(k.n_heads, group, tp, tt)
    if work is None:
        work = attn_workspace(k.n_heads, group, tp, tt, dev)
    elif work.numel() < need:
        raise ValueError("attention workspace too small")
    qc = q.to(dev).contiguous()
    if out is None:
        out = torch.empty(B, Hq, 1, HD, dtype=torch.float16, device=dev)
    ks, vs = k.struct(), v.struct()

    def call():
        L.check(lib.lq_resident_attention(ctypes.addressof(ks), ctypes.addressof(vs), tp, qc.data_ptr(), group,
                                          L.ptr(pk), L.ptr(pv), tt, work.data_ptr(), out.data_ptr(),
                                          L.stream_ptr(dev)), "lq_resident_attention")
    if dev.index == torch.cuda.current_device():
        call()
    else:
        with torch.cuda.device(dev):
            call()
    return out
