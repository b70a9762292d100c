"""Drafted tokens over a resident compressed cache.

A drafter proposes a few tokens per sequence, as a chain or as a tree: node 0 is
the newest token (its K / V are not in the cache yet), every other node continues
an earlier one.  One pass of the model scores all of them:

* ``resident_tree_attention`` attends every node to the resident prefix, the
  fp16 / bf16 tail and the node's own ancestors.  Several query tokens would
  otherwise read a prefix dequantised to memory (``ResidentKVCache.materialise``,
  the read path of the reference's cache, llm/compressed_kv_cache.py:384-395).
* ``accept_drafts`` finds the path of drafts that the model's own choices confirm;
* ``append_accepted`` puts those nodes' K / V behind the tails, all layers at once.

None of it waits for the device; lengths, trees and counts stay there.
"""
from __future__ import annotations

import ctypes
from array import array
from functools import reduce
from operator import attrgetter, or_
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib as L
from .resident import HD, RB, ResidentKV

MAX_NODES = L.LQ_TREE_MAX_NODES
_DTYPES = (torch.float16, torch.bfloat16)


def _rows(t: torch.Tensor):
    """(t, pointer and strides of (B, H, T, 128) rows): as it lies where the kernels can
    read 16 bytes at a time, else a copy.  (contiguous() makes none of a tensor that is
    contiguous and unaligned, or whose odd stride is that of a length of one.)"""
    sb, sh, st, se = t.stride()
    p = t.data_ptr()
    if se != 1 or (sb | sh | st) & 7 or p & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        sb, sh, st, _ = t.stride()
        p = t.data_ptr()
    return t, (p, sb, sh, st)


def _ints(t, shape, name: str, dev) -> torch.Tensor:
    """Whole numbers of the given shape as a contiguous int32 tensor on dev."""
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    if t.dtype is torch.int32 and t.device == dev and t.is_contiguous():
        return t
    return t.to(device=dev, dtype=torch.int32).contiguous()


def _parents(parents, B: int, N: int, dev) -> torch.Tensor:
    if isinstance(parents, torch.Tensor) and parents.dim() == 1:
        parents = parents[None].expand(B, -1)
    p = _ints(parents, (B, N), "parents", dev)
    if L.debug_checks():
        bad = (p >= torch.arange(N, device=dev, dtype=torch.int32)).any()
        if bool(bad):
            raise ValueError("a node's parent must be an earlier node of its sequence, -1 (root) or -2 (padding)")
    return p


def node_depths(parents: torch.Tensor) -> torch.Tensor:
    """(B, N) int64: how many ancestors each node has (0 for roots and padding), by
    doubling: after k rounds up[i] is the node 2^k generations above i."""
    B, N = parents.shape
    idx = torch.arange(N, device=parents.device)
    up = torch.where((parents >= 0) & (parents < idx), parents.long(), idx)
    depth = (up != idx).long()
    k = 1
    while k < N:
        depth = depth + depth.gather(1, up)
        up = up.gather(1, up)
        k *= 2
    return depth


def tree_workspace_size(n_heads: int, group: int, n_nodes: int, t_prefix: int, tail_cap: int) -> int:
    """Bytes of workspace of resident_tree_attention over n_heads resident heads (all
    sequences' kv heads), n_nodes nodes per sequence."""
    n = L.load().lq_tree_attn_workspace(1, n_heads, n_nodes, group, t_prefix, tail_cap)
    if n < 0:
        raise ValueError("bad tree attention geometry")
    return n


def tree_attn_workspace(n_heads: int, group: int, n_nodes: int, t_prefix: int, tail_cap: int,
                        device=None) -> torch.Tensor:
    """tree_workspace_size bytes on the device, uninitialised."""
    return torch.empty(tree_workspace_size(n_heads, group, n_nodes, t_prefix, tail_cap), dtype=torch.uint8, device=device)


def resident_tree_attention(k: ResidentKV, v: ResidentKV, q: torch.Tensor, draft_k: torch.Tensor,
                            draft_v: torch.Tensor, parents: torch.Tensor, tail_k: Optional[torch.Tensor] = None,
                            tail_v: Optional[torch.Tensor] = None, tail_len: Optional[torch.Tensor] = None,
                            start: Optional[torch.Tensor] = None, work: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None, t_prefix: Optional[int] = None) -> torch.Tensor:
    """Attention of N drafted nodes per sequence: softmax(q K^T / sqrt(128)) V, each
    node over the cache, itself and its ancestors.

    q: (B, Hq, N, 128) fp16 or bf16, Hq = group * H_kv (group 1..16, N 1..256);
    draft_k / draft_v: (B, H_kv, N, 128) of q's type, the nodes' own K / V;
    parents: (B, N) or (N,) whole numbers: an earlier node, -1 for a root, -2 for
    padding (padding and its descendants see nothing; their rows are zero).
    k / v: resident prefixes of B * H_kv heads, read up to t_prefix tokens (a multiple
    of 16, all of them by default); tail_k / tail_v: (B, H_kv, cap, 128) of q's type,
    of which sequence b has the first tail_len[b] (all cap without tail_len); start[b]:
    the first prefix / tail token that sequence b sees (left padding).
    Any strides with a contiguous last dimension are read in place.  work:
    tree_attn_workspace, used until the call's work on the stream is done; out: where
    to write, of q's shape and type.  Returns (B, Hq, N, 128).  The products are
    fp16: bf16 values beyond its range become infinities, those below 2^-14 lose bits and
    below 2^-25 are zero.  The same inputs give the same bits, and tokens that a row does
    not see do not change its."""
    lib = L.lib()
    dev = k.a.device
    if q.dim() != 4 or q.dtype not in _DTYPES or q.shape[3] != HD:
        raise ValueError("q must be (B, Hq, N, 128) fp16 or bf16")
    dt = q.dtype
    B, Hq, N, _ = q.shape
    if k.n_heads != v.n_heads or k.n_tokens != v.n_tokens or dev != v.a.device:
        raise ValueError("K and V resident prefixes must have the same geometry and device")
    if B < 1 or k.n_heads % B:
        raise ValueError("the resident prefix must hold B * H_kv heads")
    Hkv = k.n_heads // B
    if Hq < 1 or Hq % Hkv or Hq // Hkv > 16:
        raise ValueError("query heads must be 1..16 times the kv heads")
    if not 1 <= N <= MAX_NODES:
        raise ValueError(f"1..{MAX_NODES} nodes per sequence")
    tp = k.n_tokens if t_prefix is None else int(t_prefix)
    if tp < 0 or tp > k.n_tokens or tp % RB:
        raise ValueError("t_prefix must be a multiple of 16 within the resident prefix")
    if draft_k.shape != (B, Hkv, N, HD) or draft_v.shape != draft_k.shape:
        raise ValueError("draft K / V must be (B, H_kv, N, 128)")
    given = [q, draft_k, draft_v]
    cap = 0
    if tail_k is not None and tail_v is not None:
        if tail_k.dim() != 4 or tail_k.shape != tail_v.shape or tail_k.shape[:2] != (B, Hkv) or tail_k.shape[3] != HD:
            raise ValueError("tail K / V must be (B, H_kv, cap, 128)")
        cap = tail_k.shape[2]
        given += [tail_k, tail_v]
    elif tail_k is not None or tail_v is not None:
        raise ValueError("tail K and V go together")
    elif tail_len is not None:
        raise ValueError("tail_len without a tail")
    for t in given:
        if t.dtype is not dt or t.device != dev:
            raise ValueError("q, the drafts and the tail must be of one type, on the resident prefix's device")
    if out is not None and (out.shape != q.shape or out.dtype is not dt or out.device != dev or out.stride(3) != 1 or
                            any(s % 8 or (s == 0 and n > 1) for s, n in zip(out.stride()[:3], out.shape)) or
                            out.data_ptr() % 16):
        raise ValueError("out must be like q, its rows 16-byte aligned and apart")
    with L.on_device(dev):
        par = _parents(parents, B, N, dev)
        tl = None if tail_len is None else _ints(tail_len, (B,), "tail_len", dev)
        st = None if start is None else _ints(start, (B,), "start", dev)
        if work is None:
            work = tree_attn_workspace(k.n_heads, Hq // Hkv, N, tp, cap, device=dev)
        elif work.device != dev or not work.is_contiguous():
            raise ValueError("the attention workspace must be contiguous, on the resident prefix's device")
        if out is None:
            out = q.new_empty(q.shape)
        keep, flat = [], []                    # the copies stay until the launch; six lq_rows
        for t in given:
            t, r = _rows(t)
            keep.append(t)
            flat += r
        flat += (out.data_ptr(),) + out.stride()[:3]
        rows = array("q", flat)
        at = rows.buffer_info()[0]
        rc = lib.lq_resident_tree_attention(
            ctypes.addressof(k.struct()), ctypes.addressof(v.struct()), tp, at, at + 32, at + 64, par.data_ptr(), B, N,
            Hq // Hkv, at + 96 if cap else None, at + 128 if cap else None, cap, None if tl is None else tl.data_ptr(),
            None if st is None else st.data_ptr(), 0 if dt is torch.float16 else 1, work.data_ptr(),
            work.numel() * work.element_size(), at + 32 * len(given), L.raw_stream(dev))
        if rc:
            if rc == L.LQ_ERR_ARG and work.numel() * work.element_size() < lib.lq_tree_attn_workspace(
                    B, Hkv, N, Hq // Hkv, tp, cap):
                raise ValueError("attention workspace too small")
            L.check(rc, "lq_resident_tree_attention")
    return out


def accept_drafts(tokens: torch.Tensor, parents: torch.Tensor, logits: Optional[torch.Tensor] = None,
                  choice: Optional[torch.Tensor] = None, work: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The drafts of each sequence that the model confirms.

    tokens: (B, N) int64, the drafted tokens (node 0: the newest token); parents:
    (B, N) or (N,), as in resident_tree_attention; logits: (B, N, V) fp16, bf16 or
    fp32, the model's at each node, whose argmax (lowest index of equal ones, NaN
    above all) is the node's choice -- or choice: (B, N) int64, e.g. a sample of each
    node's distribution.  From node 0 the walk goes to the lowest-numbered child whose
    token is the node's choice, until there is none.  Returns (path (B, N) int32: the
    nodes walked, then -1; count (B,) int32: how many, 0 where node 0 is padding;
    next (B,) int64: the last one's choice, -1 there), on tokens' device."""
    lib = L.lib()
    if (logits is None) == (choice is None):
        raise ValueError("either logits or choice")
    if tokens.dim() != 2 or tokens.dtype != torch.int64 or not tokens.is_cuda:
        raise ValueError("tokens must be (B, N) int64 on the GPU")
    B, N = tokens.shape
    dev = tokens.device
    if B < 1 or not 1 <= N <= MAX_NODES:
        raise ValueError(f"at least one sequence of 1..{MAX_NODES} nodes")
    vocab = dt = sb = sn = 0
    if logits is not None:
        if logits.dim() != 3 or logits.shape[:2] != (B, N) or logits.device != dev or logits.shape[2] < 1:
            raise ValueError("logits must be (B, N, V) on the tokens' device")
        if logits.dtype not in _DTYPES and logits.dtype is not torch.float32:
            raise ValueError("logits must be fp16, bf16 or fp32")
        vocab, dt = logits.shape[2], L.dtype_code(logits.dtype)
    elif choice.shape != (B, N) or choice.dtype is not torch.int64 or choice.device != dev:
        raise ValueError("choice must be (B, N) int64 on the tokens' device")
    with L.on_device(dev):
        nbytes = 0
        if logits is not None:
            if logits.stride(2) != 1:
                logits = logits.contiguous()
            sb, sn, _ = logits.stride()
            if work is None:
                nbytes = lib.lq_accept_workspace(B, N, vocab)
                if nbytes < 0:
                    raise ValueError("too many nodes (65535 in all) or too large a vocabulary")
                work = tokens.new_empty(nbytes + 7 >> 3)
            elif work.device != dev or not work.is_contiguous():
                raise ValueError("the acceptance workspace must be contiguous, on the tokens' device")
            else:
                nbytes = work.numel() * work.element_size()
        else:
            choice = choice.contiguous()
        par, tok = _parents(parents, B, N, dev), tokens.contiguous()
        path, count, nxt = par.new_empty((B, N)), par.new_empty(B), tokens.new_empty(B)
        rc = lib.lq_accept_drafts(None if logits is None else logits.data_ptr(), dt, sb, sn, vocab, L.ptr(choice),
                                  tok.data_ptr(), par.data_ptr(), B, N, None if logits is None else work.data_ptr(),
                                  nbytes, path.data_ptr(), count.data_ptr(), nxt.data_ptr(), L.raw_stream(dev))
        if rc:
            if logits is not None and not 0 <= lib.lq_accept_workspace(B, N, vocab) <= nbytes:
                raise ValueError("acceptance workspace too small, or too many nodes")
            L.check(rc, "lq_accept_drafts")
    return path, count, nxt


def accept_workspace(n_seq: int, n_nodes: int, vocab: int, device=None) -> torch.Tensor:
    """Workspace of accept_drafts with logits; uninitialised."""
    n = L.load().lq_accept_workspace(n_seq, n_nodes, vocab)
    if n < 0:
        raise ValueError("bad acceptance geometry")
    return torch.empty(int(n), dtype=torch.uint8, device=device)


_stride, _data_ptr, _get_device = torch.Tensor.stride, torch.Tensor.data_ptr, torch.Tensor.get_device
_shape, _dtype = attrgetter("shape"), attrgetter("dtype")


def _pairs(dst: Sequence[torch.Tensor], src: Sequence[torch.Tensor], what: str):
    """Checked (destination, source) lists of row tensors (B, H, rows, width), grouped by
    layout: [(how many, pointers, pointers, strides, strides in bytes, sources kept)].
    A model's lists are long (K and V of every layer): their properties are taken by
    maps over the list, a tenth of a microsecond each, and compared as sets."""
    if not len(dst) or len(dst) != len(src):
        raise ValueError(f"{what}: as many destinations as sources, one at least")
    ds, ss = set(map(_shape, dst)), set(map(_shape, src))
    if len(ds) != 1 or len(ss) != 1 or len(set(map(_dtype, dst)) | set(map(_dtype, src))) != 1:
        raise ValueError(f"{what}: destinations of one shape, sources of one shape, all of one type")
    ds, ss, el = ds.pop(), ss.pop(), dst[0].element_size()
    if len(ds) != 4 or len(ss) != 4:
        raise ValueError(f"{what}: tensors of (B, H, rows, width)")
    on = set(map(_get_device, dst)) | set(map(_get_device, src))
    if len(on) != 1 or on.pop() < 0 or ds[3] != ss[3] or ds[3] * el % 16 or not 16 <= ds[3] * el <= 4096:
        raise ValueError(f"{what}: rows on one GPU, of one width, a multiple of 16 bytes")

    def fits(strides):
        return strides[3] == 1 and not any(x * el % 16 for x in strides[:3])
    dt, st = list(map(_stride, dst)), list(map(_stride, src))
    dp, sp = list(map(_data_ptr, dst)), list(map(_data_ptr, src))
    if (not all(fits(t) and not any(x == 0 and n > 1 for x, n in zip(t, ds)) for t in set(dt)) or
            reduce(or_, dp) & 15 or len(set(dp)) < len(dp)):
        raise ValueError(f"{what}: destination rows must be contiguous, apart and 16-byte aligned")
    src = list(src)
    if not all(map(fits, set(st))) or reduce(or_, sp) & 15:
        for i, t in enumerate(src):
            if not fits(st[i]) or sp[i] & 15:
                src[i] = t.clone(memory_format=torch.contiguous_format)
                st[i], sp[i] = src[i].stride(), src[i].data_ptr()

    def group(td, ts, d, s):
        return (len(d), array("Q", d), array("Q", s), array("q", [x * el for x in td[:3]]),
                array("q", [x * el for x in ts[:3]]), src)
    n = len(dst)
    if dt.count(dt[0]) == n and st.count(st[0]) == n:
        return [group(dt[0], st[0], dp, sp)]
    kinds = list(zip(dt, st))
    return [group(*kind, [p for p, x in zip(dp, kinds) if x == kind], [p for p, x in zip(sp, kinds) if x == kind])
            for kind in dict.fromkeys(kinds)]


def _addresses(group):
    """A group of _pairs as the C ABI takes it."""
    n, d, s, sd, ss, _ = group
    return d.buffer_info()[0], s.buffer_info()[0], n, sd.buffer_info()[0], ss.buffer_info()[0]


def append_accepted(tails: Sequence[torch.Tensor], drafts: Sequence[torch.Tensor], path: torch.Tensor,
                    count: torch.Tensor, tail_len: torch.Tensor) -> torch.Tensor:
    """Accepted drafts into the tails, in place: row tail_len[b] + j of every tail
    (B, H, cap, width) becomes row path[b][j] of its draft (B, H, N, width), j < count[b];
    the other rows stay.  tails / drafts: lists (K and V of all layers: one launch per
    128 of one layout); path (B, N), count and tail_len (B,) as accept_drafts and the
    tails have them.  No draft may lie in a tail.  Returns the new lengths (B,) int32, tail_len + count.  The caller
    keeps cap >= tail_len + count: rows past cap are left out (the length stops there)."""
    lib = L.lib()
    groups = _pairs(tails, drafts, "append_accepted")
    B, H, cap, width = tails[0].shape
    N, dev = drafts[0].shape[2], tails[0].device
    if drafts[0].shape[:2] != (B, H) or B < 1 or H < 1 or cap < 1 or not 1 <= N <= MAX_NODES:
        raise ValueError(f"drafts must be (B, H, N, width) of the tails' B and H, N 1..{MAX_NODES}")
    with L.on_device(dev):
        pt, ct = _ints(path, (B, N), "path", dev), _ints(count, (B,), "count", dev)
        ln = _ints(tail_len, (B,), "tail_len", dev)
        if L.debug_checks() and (bool((ln + ct > cap).any()) or bool((ct > N).any())):
            raise ValueError("accepted rows do not fit the tails")
        new = ln.new_empty(B)
        for g in groups:
            L.check(lib.lq_append_rows(*_addresses(g), B, H, cap, N, width * tails[0].element_size(), pt.data_ptr(),
                                       ct.data_ptr(), ln.data_ptr(), new.data_ptr(), L.raw_stream(dev)),
                    "lq_append_rows")
    return new


def gather_tails(tails: Sequence[torch.Tensor], index: torch.Tensor) -> list:
    """New tails of the sequences index[r] of every tail (B, H, T, width): what
    torch.index_select(tail, 0, index) gives for each, in one launch per 128.  Indices
    are clamped to 0 .. B - 1."""
    lib = L.lib()
    if not len(tails):
        return []
    t0 = tails[0]
    if t0.dim() != 4 or index.dim() != 1 or index.numel() < 1:
        raise ValueError("tails of (B, H, T, width) and a list of sequences")
    out = [torch.empty((index.numel(),) + tuple(t.shape[1:]), dtype=t.dtype, device=t.device) for t in tails]
    if t0.shape[2] == 0 or t0.shape[1] == 0:
        return out
    groups = _pairs(out, tails, "gather_tails")
    B, H, T, width = t0.shape
    with L.on_device(t0.device):
        idx = _ints(index, (index.numel(),), "index", t0.device)
        if B < 1:
            raise ValueError("no sequences to choose from")
        for g in groups:
            L.check(lib.lq_gather_rows(*_addresses(g), B, index.numel(), H, T, width * t0.element_size(),
                                       idx.data_ptr(), L.raw_stream(t0.device)), "lq_gather_rows")
    return out
