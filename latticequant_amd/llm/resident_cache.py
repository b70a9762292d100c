"""HF cache whose decode steps attend straight over the compressed prefix.

The reference's ``CompressedKVCache.update`` (llm/compressed_kv_cache.py:342-395)
compresses every update and hands HF attention fully decompressed fp16 K / V
(kept resident beside the chunks and ``torch.cat``-ed each step).  Here:

* every layer keeps its newest tokens (up to ``tail_tokens`` + 15) as an fp16
  residual tail; older tokens are flushed in blocks of 16 into
  - E8 + rANS chunks (:func:`codec.encode_batch`, the reference's bitstream
    format: the at-rest form, what ``compressed_bytes`` counts), and
  - the resident fixed-width form of the same lattice points
    (:class:`ResidentKV`) that decode attention reads;
* the at-rest chunks are not read by decode steps: ``offload_at_rest()``
  moves them to host memory in the wire form (the device then keeps the
  resident form and the tail), ``restore_at_rest()`` brings them back;
* ``update`` returns, for a one-token step, marker views that carry the cache
  and layer, and the registered attention ``"lq_resident"`` runs
  ``lq_resident_attention`` over resident prefix + tail (no fp16 prefix is
  ever materialised); for a prompt (several query tokens) it returns the
  materialised K / V (resident prefix dequantised as ``_decompress_chunk``
  writes it, then the tail) for HF's causal SDPA;
* drafted tokens (``draft`` / ``verify``): the next forward's tokens are the nodes of
  a tree that attend to the cache and their own ancestors
  (:func:`resident_tree_attention`); the path that the model confirms goes into the
  cache, the rest is dropped;
* beams: ``reorder_cache`` permutes the sequences in place
  (:func:`reorder_sequences`), ``batch_repeat_interleave`` and
  ``batch_select_indices`` make the cache of chosen ones.

Use::

    from latticequant_amd.llm.resident_cache import ResidentKVCache, register
    register()                                   # adds attn_implementation "lq_resident"
    model = AutoModelForCausalLM.from_config(cfg, attn_implementation="lq_resident")
    out = model.generate(ids, past_key_values=ResidentKVCache(bits_per_dim=4), ...)

    cache.draft(parents)                         # the tree: parents[i] < i, -1 for node 0
    logits = model(tokens, position_ids=cache.draft_positions(), past_key_values=cache).logits
    accepted, nxt = cache.verify(tokens, logits=logits)
"""
from __future__ import annotations

from typing import List, Optional

import torch
from transformers.cache_utils import DynamicCache

from .. import codec
from .resident import MAX_REORDER, RB, ResidentKV, attn_workspace, reorder_sequences, resident_decode_attention
from .tree import (MAX_NODES, accept_drafts, append_accepted, gather_tails, node_depths, resident_tree_attention,
                   tree_workspace_size)

ATTN_NAME = "lq_resident"


class ResidentKVCache(DynamicCache):
    """HF cache: rANS chunks at rest + resident b=5 prefix + fp16 residual tail."""

    def __init__(self, bits_per_dim: int = 4, tail_tokens: int = 128):
        super().__init__()
        if bits_per_dim not in (3, 4, 5):
            raise ValueError("bits_per_dim must be 3, 4 or 5")
        if tail_tokens < 0 or tail_tokens % RB:
            raise ValueError(f"tail_tokens must be a non-negative multiple of {RB}")
        self.bits = bits_per_dim
        self.tail_tokens = tail_tokens
        self._empty()

    # -- storage ----------------------------------------------------------
    def _empty(self):
        self.res_k: List[Optional[ResidentKV]] = []
        self.res_v: List[Optional[ResidentKV]] = []
        self.tail_k: List[Optional[torch.Tensor]] = []
        self.tail_v: List[Optional[torch.Tensor]] = []
        self.chunks: List[list] = []          # per layer: [(_AtRest K, _AtRest V)] rANS chunks at rest
        self._epochs = _Epochs()
        self._work = None
        self._work_heads = 0
        self._parents = self._start = None    # drafted tree of the next forward
        self._drafts = {}                     # layer -> the drafts' (K, V)
        self._room = {}                       # layer -> (K, V) buffers that the tails are the first tokens of
        self._tree_work = None

    def _ensure(self, layer_idx: int):
        while len(self.res_k) <= layer_idx:
            self.res_k.append(None)
            self.res_v.append(None)
            self.tail_k.append(None)
            self.tail_v.append(None)
            self.chunks.append([])

    def _flush(self, layer_idx: int, n: int):
        """Compress the oldest n (a multiple of 16) tail tokens of the layer."""
        tk, tv = self.tail_k[layer_idx], self.tail_v[layer_idx]
        B, H, _, hd = tk.shape
        xk, xv = tk[:, :, :n].contiguous(), tv[:, :, :n].contiguous()
        # no host sync: the at-rest chunks are settled on first access
        enc, _, pend = codec.encode_batch_deferred(torch.stack([xk, xv]), self.bits)
        s32, s16 = enc.scale32.view(2, -1), enc.scale16.view(2, -1)   # the K and V chunks' head scales
        for i, (res, x) in enumerate(((self.res_k, xk), (self.res_v, xv))):
            r = res[layer_idx]
            if r is None:
                r = ResidentKV(B * H, max(4 * n, 1024), device=x.device)
                res[layer_idx] = r
            elif r.n_tokens + n > r.cap_blocks * RB:
                r.reserve(max(2 * r.cap_blocks * RB, r.n_tokens + n))
            r.append(x, s32[i], s16[i])
        since = self._epochs.now()
        self.chunks[layer_idx].append((_AtRest(pend, 0, since), _AtRest(pend, 1, since)))
        self._room.pop(layer_idx, None)
        self.tail_k[layer_idx] = tk[:, :, n:].contiguous()
        self.tail_v[layer_idx] = tv[:, :, n:].contiguous()

    # -- HF Cache interface ----------------------------------------------
    def update(self, key_states, value_states, layer_idx, cache_kwargs=None, *args, **kwargs):
        if key_states.shape[-1] != 128:
            raise ValueError("ResidentKVCache needs head_dim 128")
        self._ensure(layer_idx)
        if self._parents is not None:
            if (key_states.shape[0], key_states.shape[2]) != tuple(self._parents.shape):
                raise ValueError("the forward's tokens are not the drafted nodes: verify() or discard() the draft first")
            self._drafts[layer_idx] = (key_states, value_states)
            return self._marked(key_states, value_states, layer_idx)
        self._room.pop(layer_idx, None)
        if self.tail_k[layer_idx] is None:
            self.tail_k[layer_idx] = key_states.contiguous()
            self.tail_v[layer_idx] = value_states.contiguous()
        else:
            self.tail_k[layer_idx] = torch.cat([self.tail_k[layer_idx], key_states], 2)
            self.tail_v[layer_idx] = torch.cat([self.tail_v[layer_idx], value_states], 2)
        over = self.tail_k[layer_idx].shape[2] - self.tail_tokens
        if over >= RB:
            self._flush(layer_idx, over // RB * RB)
        if key_states.shape[2] == 1:
            # decode step: marker views carrying the cache; the attention reads
            # the resident prefix and the tail itself
            return self._marked(key_states, value_states, layer_idx)
        return self.materialise(layer_idx)

    def _marked(self, k, v, layer_idx: int):
        mk, mv = k.view_as(k), v.view_as(v)
        mk._lq_cache = mv._lq_cache = self
        mk._lq_layer = mv._lq_layer = layer_idx
        return mk, mv

    def materialise(self, layer_idx: int):
        """Full (B, H, T, hd) K / V of the layer: the resident prefix dequantised
        (lattice point x fp16 scale, rounded once) followed by the tail."""
        tk, tv = self.tail_k[layer_idx], self.tail_v[layer_idx]
        rk, rv = self.res_k[layer_idx], self.res_v[layer_idx]
        if rk is None or rk.n_tokens == 0:
            return tk, tv
        B, H = tk.shape[:2]
        pk = rk.dequant(tk.dtype).view(B, H, -1, 128)
        pv = rv.dequant(tv.dtype).view(B, H, -1, 128)
        return torch.cat([pk, tk], 2), torch.cat([pv, tv], 2)

    def attend(self, layer_idx: int, query: torch.Tensor) -> torch.Tensor:
        """One decode step of the layer: query (B, Hq, 1, 128) -> (B, Hq, 1, 128)."""
        tk, tv = self.tail_k[layer_idx], self.tail_v[layer_idx]
        B, H = tk.shape[:2]
        rk, rv = self._prefix(layer_idx, B * H, tk.device)
        group = query.shape[1] // H
        n = attn_workspace_size(B * H, group, rk.n_tokens, tk.shape[2])
        # the workspace's completion counters sit at [0, 256 * kv heads): a new
        # head count would put split records where counters were, so re-zero
        if (self._work is None or self._work.numel() < n or self._work.device != tk.device or
                self._work_heads != B * H):
            self._work = attn_workspace(B * H, group, rk.n_tokens, tk.shape[2], device=tk.device)
            self._work_heads = B * H
        out = resident_decode_attention(rk, rv, query.to(torch.float16), tk.to(torch.float16),
                                        tv.to(torch.float16), work=self._work)
        return out.to(query.dtype)

    def _prefix(self, layer_idx: int, heads: int, device):
        if self.res_k[layer_idx] is None:   # nothing flushed yet: an empty prefix
            self.res_k[layer_idx] = ResidentKV(heads, 1024, device=device)
            self.res_v[layer_idx] = ResidentKV(heads, 1024, device=device)
        return self.res_k[layer_idx], self.res_v[layer_idx]

    # -- drafted trees ------------------------------------------------------
    def draft(self, parents, start=None) -> None:
        """The next forward's tokens are drafted nodes: parents (B, N) or (N,) whole
        numbers (tensor or nested lists), an earlier node, -1 for the root, node 0 (the
        newest token, not in the cache yet); -2 for padding.  start (B,): the first cached
        token each sequence sees (left padding).  The forward leaves the cache as it is;
        its attention is the tree's (the model's mask is not read), so its positions are
        draft_positions().  verify() or discard() ends the draft."""
        if self._parents is not None:
            raise ValueError("a draft is pending: verify() or discard() it first")
        if not self.tail_k:
            raise ValueError("nothing is cached yet: the prompt comes first")
        B, dev = self.tail_k[0].shape[0], self.tail_k[0].device
        par = torch.as_tensor(parents)
        if par.is_floating_point() or par.dtype == torch.bool or par.dim() not in (1, 2):
            raise ValueError("parents must be (B, N) or (N,) whole numbers")
        if par.dim() == 1:
            par = par[None].expand(B, -1)
        if par.shape[0] != B or not 1 <= par.shape[1] <= MAX_NODES:
            raise ValueError(f"one tree of 1..{MAX_NODES} nodes per sequence")
        st = None if start is None else torch.as_tensor(start)
        if st is not None and (st.shape != (B,) or st.dtype not in (torch.int32, torch.int64)):
            raise ValueError("start must be (B,) whole numbers")
        self._parents = par.to(device=dev, dtype=torch.int32).contiguous()
        self._start = None if st is None else st.to(device=dev, dtype=torch.int32)
        self._drafts = {}

    def draft_positions(self) -> torch.Tensor:
        """(B, N) int64: the nodes' positions, cached tokens + depth in the tree."""
        if self._parents is None:
            raise ValueError("no draft is pending")
        pos = self.get_seq_length() + node_depths(self._parents)
        return pos if self._start is None else pos - self._start[:, None].long()

    def attend_drafts(self, layer_idx: int, query: torch.Tensor) -> torch.Tensor:
        """The drafted nodes' attention: query (B, Hq, N, 128) -> (B, N, Hq, 128)."""
        dk, dv = self._drafts[layer_idx]
        tk, tv = self.tail_k[layer_idx], self.tail_v[layer_idx]
        dt = query.dtype if query.dtype in (torch.float16, torch.bfloat16) else torch.float16
        rk, rv = self._prefix(layer_idx, tk.shape[0] * tk.shape[1], tk.device)
        B, Hq, N, hd = query.shape
        n = tree_workspace_size(rk.n_heads, Hq // tk.shape[1], N, rk.n_tokens, tk.shape[2])
        if self._tree_work is None or self._tree_work.numel() < n or self._tree_work.device != tk.device:
            self._tree_work = torch.empty(n, dtype=torch.uint8, device=tk.device)
        out = torch.empty((B, N, Hq, hd), dtype=dt, device=tk.device)
        resident_tree_attention(rk, rv, query.to(dt), dk.to(dt), dv.to(dt), self._parents, tk.to(dt), tv.to(dt),
                                start=self._start, work=self._tree_work, out=out.transpose(1, 2))
        return out.to(query.dtype)

    def verify(self, tokens: torch.Tensor, logits: Optional[torch.Tensor] = None,
               choice: Optional[torch.Tensor] = None):
        """End the draft: the path of nodes that the model's choices confirm
        (accept_drafts: the argmax of logits (B, N, V), or choice (B, N)) goes into the
        cache, the other nodes are dropped.  tokens: (B, N), the forward's.  Sequences of a
        batch advance together, by the shortest accepted path.  Returns (accepted (B, A):
        the tokens now cached, node 0's first; next (B, 1): the token after them)."""
        if self._parents is None or len(self._drafts) != len(self.tail_k):
            raise ValueError("no drafted forward to verify")
        path, count, nxt = accept_drafts(tokens, self._parents, logits=logits, choice=choice)
        n = int(count.min())                       # the tails' length: the host has to know it
        if n == 0:
            raise ValueError("a sequence's node 0 is padding")
        taken = path[:, :n].long()
        accepted = tokens.gather(1, taken)
        if path.shape[1] > n:                      # a sequence cut short goes on with its next accepted node
            more = path[:, n].long()
            nxt = torch.where(more >= 0, tokens.gather(1, more.clamp_min(0)[:, None])[:, 0], nxt)
        self.accept(path[:, :n])
        return accepted, nxt[:, None]

    def accept(self, path: torch.Tensor) -> None:
        """End the draft with the nodes path (B, A), whole numbers (clamped to the nodes), in
        the cache."""
        if self._parents is None or len(self._drafts) != len(self.tail_k):
            raise ValueError("no drafted forward to accept")
        B, N = self._parents.shape
        if path.dim() != 2 or path.shape[0] != B or not 1 <= path.shape[1] <= N:
            raise ValueError("path must be (B, A), 1 <= A <= nodes")
        A, dev = path.shape[1], self._parents.device
        full = torch.full((B, N), -1, dtype=torch.int32, device=dev)
        full[:, :A] = path.clamp(0, N - 1)
        groups = {}                                # rows of one shape, type, device and tail length: K and V of all layers, as a rule
        for i in range(len(self.tail_k)):
            t = self.tail_k[i].shape[2]
            for buf, d in zip(self._buffers(i, t + A), self._drafts[i]):
                groups.setdefault((t, buf.shape, buf.dtype, buf.device), []).append((buf, d.to(buf.dtype)))
        for (t, *_), pairs in groups.items():
            count, at = (torch.full((B,), n, dtype=torch.int32, device=dev) for n in (A, t))
            append_accepted(*zip(*pairs), full, count, at)
        for i in range(len(self.tail_k)):          # (the tails end before the new rows until here)
            t = self.tail_k[i].shape[2]
            self.tail_k[i], self.tail_v[i] = (b[:, :, :t + A] for b in self._room[i])
        self.discard()
        for i in range(len(self.tail_k)):
            over = self.tail_k[i].shape[2] - self.tail_tokens
            if over >= RB:
                self._flush(i, over // RB * RB)

    def discard(self) -> None:
        """End the draft, the cache as it was."""
        self._parents = self._start = None
        self._drafts = {}

    def _buffers(self, layer_idx: int, need: int):
        """The layer's tails as the first tokens of buffers with room for `need`."""
        tk, tv = self.tail_k[layer_idx], self.tail_v[layer_idx]
        buf = self._room.get(layer_idx)
        if buf is None or buf[0].shape[2] < need:
            B, H, t, hd = tk.shape
            buf = tuple(torch.empty((B, H, need + 64, hd), dtype=x.dtype, device=x.device) for x in (tk, tv))
            for b, x in zip(buf, (tk, tv)):
                b[:, :, :t] = x
            self._room[layer_idx] = buf
        return buf

    # -- beams --------------------------------------------------------------
    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        """Sequence i becomes sequence beam_idx[i] as it was, in place (-1: the last one;
        what is out of range is clamped).  Whole prefixes move, what the sequences share
        too; the launches are a few whatever the number of chunks."""
        if not self.tail_k:
            return
        if beam_idx.dim() != 1 or beam_idx.numel() != self.tail_k[0].shape[0] or beam_idx.numel() > MAX_REORDER:
            return self.batch_select_indices(beam_idx)
        self._no_draft()
        idx = self._numbers(beam_idx)
        groups = {}                                # prefixes of one length, head count and device: all of them, as a rule
        for r in self.res_k + self.res_v:
            if r is not None:
                groups.setdefault((r.n_tokens, r.n_heads, r.a.device), []).append(r)
        tails = self._tails_of(idx)                # before anything moves: it may find no room
        for group in groups.values():
            reorder_sequences(group, idx)
        self._continue_as(idx, tails)

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        """Keep the sequences indices[r], in that order (a sequence may stand several
        times; -1 is the last one, what is out of range is clamped); the others' resident
        blocks and exceptions are freed.  A selection that finds no room for its result
        leaves the cache as it was; of fewer sequences than there are (or as many) each
        prefix is freed once its successor is there, and the cache is left empty if there is no
        room for one after the first.  At-rest chunks stay whole, with the
        bitstreams of all sequences they were flushed with (their .rows say whose are the
        cache's).  One host wait per prefix (K and V of each layer)."""
        if not self.tail_k:
            return
        self._no_draft()
        B = self.tail_k[0].shape[0]
        idx = torch.arange(B)[indices.cpu()] if indices.dtype == torch.bool else indices
        if idx.dim() != 1 or idx.numel() < 1:
            raise ValueError("indices must be a list of sequences")
        idx = self._numbers(idx)
        tails, old, new = self._tails_of(idx), self.res_k + self.res_v, []
        layers, fewer = len(self.res_k), idx.numel() <= B
        if fewer:
            self.res_k, self.res_v = [], []        # `old` alone holds them
        try:
            while len(new) < len(old):
                i = len(new)
                new.append(None if old[i] is None else old[i].select(idx, B, cap_tokens=old[i].cap_blocks * RB))
                if fewer:
                    old[i] = None
        except BaseException:
            if fewer and any(r is not None for r in new):
                self._empty()
            else:
                self.res_k, self.res_v = old[:layers], old[layers:]
            raise
        self.res_k, self.res_v = new[:layers], new[layers:]
        self._continue_as(idx, tails)

    def batch_repeat_interleave(self, repeats: int) -> None:
        """Every sequence `repeats` times in a row (a prompt's beams)."""
        if self.tail_k:
            self.batch_select_indices(torch.arange(self.tail_k[0].shape[0]).repeat_interleave(repeats))

    def _no_draft(self):
        if self._parents is not None:
            raise ValueError("a draft is pending: verify() or discard() it first")

    def _numbers(self, idx: torch.Tensor) -> torch.Tensor:
        """Sequence numbers as the prefixes, the tails and the chunks all read them."""
        if idx.dtype not in (torch.int32, torch.int64):
            raise ValueError("sequence numbers must be int32 or int64")
        B = self.tail_k[0].shape[0]
        idx = idx.to(self.tail_k[0].device)
        return torch.where(idx < 0, idx + B, idx).clamp(0, B - 1)

    def _tails_of(self, idx) -> list:
        """New tails of the sequences idx: K of all layers, then V."""
        tails = self.tail_k + self.tail_v
        groups = {}                                # tails of one shape, type and device
        for j, t in enumerate(tails):
            groups.setdefault((t.shape, t.dtype, t.device), []).append(j)
        for group in groups.values():
            for j, t in zip(group, gather_tails([tails[j] for j in group], idx)):
                tails[j] = t
        return tails

    def _continue_as(self, idx, tails) -> None:
        """The tails of the sequences idx, and their at-rest chunks."""
        layers = len(self.tail_k)
        self.tail_k, self.tail_v = tails[:layers], tails[layers:]
        self._room = {}
        self._epochs.select(idx)

    def get_seq_length(self, layer_idx=0):
        if layer_idx >= len(self.tail_k) or self.tail_k[layer_idx] is None:
            return 0
        r = self.res_k[layer_idx]
        return (r.n_tokens if r is not None else 0) + self.tail_k[layer_idx].shape[2]

    def get_mask_sizes(self, query_length: int, layer_idx: int = 0) -> tuple:
        """(kv_length, kv_offset): past tokens + the new query."""
        return self.get_seq_length(layer_idx) + query_length, 0

    def get_max_length(self, layer_idx=None) -> int:
        return -1

    def __len__(self):
        return len(self.tail_k)

    @property
    def is_compileable(self) -> bool:
        return False

    # -- at-rest chunks ---------------------------------------------------
    def offload_at_rest(self) -> int:
        """Move every at-rest chunk pair flushed so far to host memory in the
        wire form (codec.to_bytes: the reference's bitstream words, coset bits
        and fp16 scales plus tables, checkpoints and a CRC-32), releasing its
        device copy: decode steps read only the resident form and the tail, so
        the device then holds about the resident bytes and the tail.  Settles
        pending encodes (one host sync).  Returns the host bytes held."""
        for ch in self.chunks:
            for i, pair in enumerate(ch):
                ch[i] = tuple(e if isinstance(e, _HostAtRest) else _HostAtRest(e.batch, e.since) for e in pair)
        return self.at_rest_host_bytes()

    def restore_at_rest(self):
        """Bring offloaded chunk pairs back to the device (codec.from_bytes)."""
        for ch in self.chunks:
            for i, pair in enumerate(ch):
                ch[i] = tuple(_DeviceAtRest(e.batch, e.since) if isinstance(e, _HostAtRest) else e for e in pair)

    def at_rest_host_bytes(self) -> int:
        return sum(e.nbytes for ch in self.chunks for pair in ch for e in pair if isinstance(e, _HostAtRest))

    # -- reporting --------------------------------------------------------
    def compressed_bytes(self) -> int:
        """Bytes of the at-rest chunks as the reference counts them
        (bitstream + coset bits + fp16 scales, llm/compressed_kv_cache.py:113-119),
        wherever they are held; chunks are whole, also those of sequences that a selection
        has dropped since."""
        return sum(e.reference_bytes() for ch in self.chunks for pair in ch for e in pair)

    def resident_bytes(self) -> int:
        """Bytes of the resident decode form (records, meta, scales, exceptions)."""
        return sum(r.nbytes() for r in self.res_k + self.res_v if r is not None)

    def tail_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.tail_k + self.tail_v if t is not None)


class _Epochs:
    """Which of its sequences a chunk has for each sequence of the cache.  A chunk's
    bitstreams are its own whole, so reordering and selecting move only these numbers: one
    row of a table for all chunks flushed between two selections, (epochs, sequences) int64
    on the device, so that a selection is the same few launches however many chunks there
    are."""

    def __init__(self):
        self.table, self._open = None, False   # _open: chunks since the last selection, which have no row yet

    def now(self) -> tuple:
        """The epoch of a chunk that is flushed now."""
        self._open = True
        return self, 0 if self.table is None else self.table.shape[0]

    def rows(self, epoch: int) -> Optional[torch.Tensor]:
        """The chunk's sequence that each of the cache's is; None: the same one."""
        return None if self.table is None or epoch == self.table.shape[0] else self.table[epoch]

    def select(self, idx: torch.Tensor) -> None:
        idx = idx.long()
        held = [] if self.table is None else [self.table.index_select(1, idx)]
        if self._open:
            held.append(idx[None])
        if held:
            self.table, self._open = torch.cat(held), False


class _Half:
    """One K or V half of a flushed chunk pair; since: _Epochs.now() when it was flushed."""

    def __init__(self, since):
        self.since = since

    @property
    def rows(self) -> Optional[torch.Tensor]:
        """The chunk's sequence that each sequence of the cache is (None: the same one)."""
        epochs, at = self.since
        return epochs.rows(at)


class _AtRest(_Half):
    """A half as it was flushed, settled on first access."""

    def __init__(self, pend, index: int, since):
        super().__init__(since)
        self._pend, self._index = pend, index

    @property
    def batch(self):
        return self._pend.result().select(self._index)

    def reference_bytes(self) -> int:
        return int(self.batch.reference_bytes().sum())


class _DeviceAtRest(_Half):
    """A half held on the device as a settled batch."""

    def __init__(self, batch, since):
        super().__init__(since)
        self.batch = batch

    def reference_bytes(self) -> int:
        return int(self.batch.reference_bytes().sum())


class _HostAtRest(_Half):
    """A half held in host memory in the wire form; .batch restores it to the current
    device (a new device copy per access)."""

    def __init__(self, batch, since):
        super().__init__(since)
        self.blob = codec.to_bytes(batch)
        self.nbytes = len(self.blob)
        self._ref = int(batch.reference_bytes().sum())

    @property
    def batch(self):
        return codec.from_bytes(self.blob)

    def reference_bytes(self) -> int:
        return self._ref


def attn_workspace_size(n_heads: int, group: int, t_prefix: int, t_tail: int) -> int:
    from .. import _lib as L
    n = L.lib().lq_resident_attn_workspace(n_heads, group, t_prefix, t_tail)
    if n < 0:
        raise ValueError("bad attention geometry")
    return int(n)


def resident_attention(module, query, key, value, attention_mask, dropout: float = 0.0, scaling=None, **kwargs):
    """HF attention function "lq_resident": one-token decode steps over a
    ResidentKVCache run lq_resident_attention, drafted tokens
    lq_resident_tree_attention; everything else (prompts,
    plain tensors) goes to HF's SDPA over the materialised K / V."""
    from transformers.integrations.sdpa_attention import sdpa_attention_forward
    cache = getattr(key, "_lq_cache", None)
    if cache is not None and cache._parents is not None:
        # drafted nodes: the tree is the mask, whatever mask the model built for a chain
        if (kwargs.get("sliding_window") is not None or kwargs.get("softcap") is not None or
                (scaling is not None and abs(scaling - 128 ** -0.5) > 1e-12)):
            raise ValueError("drafted trees need plain attention: no sliding window or soft-capping, scale 1/sqrt(128)")
        return cache.attend_drafts(key._lq_layer, query), None
    if cache is None or query.shape[2] != 1:
        return sdpa_attention_forward(module, query, key, value, attention_mask, dropout=dropout, scaling=scaling,
                                      **kwargs)
    # The kernel attends to every prefix + tail token with scale 1/sqrt(128).
    # A decode step that needs anything else -- a mask (HF's SDPA mask builder
    # returns None for an unpadded causal step, a tensor e.g. for left-padded
    # batches), a sliding window, logit soft-capping or another scale -- runs
    # SDPA over the materialised K / V instead, as the reference's cache does.
    if (attention_mask is not None or kwargs.get("sliding_window") is not None or
            kwargs.get("softcap") is not None or
            (scaling is not None and abs(scaling - 128 ** -0.5) > 1e-12)):
        k, v = cache.materialise(key._lq_layer)
        return sdpa_attention_forward(module, query, k, v, attention_mask, dropout=dropout, scaling=scaling,
                                      **kwargs)
    out = cache.attend(key._lq_layer, query)            # (B, Hq, 1, hd)
    return out.transpose(1, 2).contiguous(), None        # HF layout (B, q_len, Hq, hd)


def register(name: str = ATTN_NAME) -> str:
    """Register the attention function (and SDPA's mask builder) under `name`."""
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask
    AttentionInterface.register(name, resident_attention)
    AttentionMaskInterface.register(name, sdpa_mask)
    return name
