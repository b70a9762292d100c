"""ResidentKVCache along several continuations: drafted trees verified by a model, and
beams (sequences reordered, selected and repeated)."""
import pytest
import torch

from tests.test_hf_resident_gpu import _model

gpu = pytest.mark.gpu


def _cache(model, ids, tail=32, **kw):
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    c = ResidentKVCache(bits_per_dim=4, tail_tokens=tail)
    with torch.no_grad():
        lo = model(ids, past_key_values=c, use_cache=True, **kw).logits[:, -1]
    return c, lo


def _step(model, c, tokens):
    with torch.no_grad():
        return model(tokens, past_key_values=c, use_cache=True).logits


def _tree_around(path, vocab, g):
    """A tree that holds the path's tokens among others: (tokens, parents, path nodes)."""
    tokens, parents, nodes = [int(path[0])], [-1], [0]
    for t in path[1:]:
        for _ in range(2):                                   # siblings that are wrong
            w = int(torch.randint(0, vocab, (1,), generator=g))
            if w != int(t):
                tokens.append(w)
                parents.append(nodes[-1])
        tokens.append(int(t))
        parents.append(nodes[-1])
        nodes.append(len(tokens) - 1)
        tokens.append(int(torch.randint(0, vocab, (1,), generator=g)))
        parents.append(len(tokens) - 2)
    return tokens, parents, nodes


@gpu
@pytest.mark.parametrize("prompt,tail,heads,kv", [(100, 32, 4, 2), (41, 0, 8, 2), (70, 128, 4, 4)])
def test_drafted_tree_matches_single_steps_gpu(prompt, tail, heads, kv):
    """A tree that holds the greedy continuation: its nodes' logits on that path are those
    of one-token steps (the attention's tolerance carried into the logits, as in
    test_hf_resident_gpu), verify() accepts the path, and the cache goes on as the
    stepped one does, drafts again (into the same buffers) and one-token steps.  Both
    caches keep what comes after the prompt in their tails until the end: a step that
    flushed 16 of them in between would leave the stepped one with other, quantised K / V
    than the drafts saw.  A last draft then flushes."""
    model, cfg = _model(heads=heads, kv_heads=kv)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, cfg.vocab_size, (1, prompt), generator=g).cuda()
    a, lo = _cache(model, ids, tail)
    b, _ = _cache(model, ids, tail)
    first = lo.argmax(-1)
    a.tail_tokens = b.tail_tokens = 1 << 20
    for _ in range(3):
        path, want = [int(first)], []
        for _ in range(5):
            lb = _step(model, b, torch.tensor([[path[-1]]], device="cuda"))[:, -1].float()
            want.append(lb)
            path.append(int(lb.argmax()))
        path = path[:5]                                      # b has cached exactly these
        tokens, parents, nodes = _tree_around(path, cfg.vocab_size, g)
        t = torch.tensor([tokens], device="cuda")
        before = a.get_seq_length()
        a.draft(parents)
        assert a.draft_positions().tolist() == [[before + d for d in _depths(parents)]]
        with torch.no_grad():
            logits = model(t, position_ids=a.draft_positions(), past_key_values=a, use_cache=True).logits
        assert a.get_seq_length() == before
        for i, w in zip(nodes, want):
            err = ((logits[:, i].float() - w).abs().max() / w.abs().max()).item()
            assert err < 5e-3, err
        choice = torch.zeros(1, len(tokens), dtype=torch.int64, device="cuda")   # b's choices: a near tie cannot decide
        choice[0, nodes] = torch.tensor([int(w.argmax()) for w in want], device="cuda")
        accepted, nxt = a.verify(t, choice=choice)
        assert accepted.tolist() == [path] and int(nxt) == int(want[-1].argmax())
        assert a.get_seq_length() == before + 5 == b.get_seq_length()
        la = _step(model, a, nxt)[:, -1].float()
        lb = _step(model, b, nxt)[:, -1].float()
        assert ((la - lb).abs().max() / lb.abs().max()).item() < 5e-3
        first = lb.argmax(-1)
    a.tail_tokens = tail
    before, flushed = a.get_seq_length(), a.res_k[0].n_tokens if a.res_k[0] is not None else 0
    last = [x.clone() for x in a.materialise(1)]
    t = torch.tensor([[int(first), 1, 2]], device="cuda")
    a.draft([-1, 0, 0])
    with torch.no_grad():
        model(t, position_ids=a.draft_positions(), past_key_values=a, use_cache=True)
    drafts = [x.clone() for x in a._drafts[1]]
    a.accept(torch.tensor([[0, 2]], device="cuda"))
    assert a.get_seq_length() == before + 2
    n = a.res_k[1].n_tokens
    assert n % 16 == 0 and before + 2 - n == a.tail_k[1].shape[2] and a.tail_k[1].shape[2] < tail + 16
    for now, old, d in zip(a.materialise(1), last, drafts):
        kept = max(n - flushed, 0) + flushed                  # the first n tokens are compressed by now, the rest as they were
        if kept < before:
            assert torch.equal(now[:, :, kept:before], old[:, :, kept:])
        if kept <= before:
            assert torch.equal(now[:, :, before:], d[:, :, [0, 2]])


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


@gpu
def test_verify_logits_batch_and_bookkeeping_gpu():
    """Two sequences whose accepted paths differ in length advance by the shorter; the
    longer one's next token is its next accepted draft.  discard() leaves the cache."""
    model, cfg = _model()
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, cfg.vocab_size, (2, 50), generator=g).cuda()
    c, lo = _cache(model, ids, 32)
    t = torch.tensor([[int(lo[0].argmax()), 7, 8, 9], [int(lo[1].argmax()), 3, 4, 5]], device="cuda")
    c.draft([-1, 0, 1, 0])
    kv = [x.clone() for x in c.materialise(1)]
    with torch.no_grad():
        model(t, position_ids=c.draft_positions(), past_key_values=c, use_cache=True)
    c.discard()
    assert c.get_seq_length() == 50 and all(torch.equal(x, y) for x, y in zip(c.materialise(1), kv))
    c.draft([-1, 0, 1, 0])
    with torch.no_grad():
        logits = model(t, position_ids=c.draft_positions(), past_key_values=c, use_cache=True).logits
    drafts = [(k.clone(), v.clone()) for k, v in (c._drafts[i] for i in range(2))]
    fake = torch.zeros_like(logits)
    fake[0, 0, 7] = fake[0, 1, 8] = fake[0, 2, 100] = 5.0    # accepts nodes 0, 1, 2
    fake[1, 0, 5] = fake[1, 3, 200] = 5.0                    # accepts nodes 0, 3
    accepted, nxt = c.verify(t, logits=fake)
    assert accepted.tolist() == [[int(t[0, 0]), 7], [int(t[1, 0]), 5]] and nxt.tolist() == [[8], [200]]
    assert c.get_seq_length() == 52
    for i in range(2):
        for half in range(2):
            full = c.materialise(i)[half]
            for b, nodes in enumerate(([0, 1], [0, 3])):
                assert torch.equal(full[b, :, 50:52], drafts[i][half][b][:, nodes])


@gpu
def test_left_padded_drafts_gpu():
    """Sequences of different lengths, left-padded: drafts with start= see no padding and
    agree with the same sequence drafted alone."""
    model, cfg = _model()
    g = torch.Generator().manual_seed(8)
    ids = torch.randint(0, cfg.vocab_size, (2, 60), generator=g).cuda()
    mask = torch.ones(2, 60, dtype=torch.long, device="cuda")
    mask[0, :13] = 0
    pos = (mask.cumsum(-1) - 1).clamp_min(0)
    c, _ = _cache(model, ids, 128, attention_mask=mask, position_ids=pos)
    alone, _ = _cache(model, ids[:1, 13:], 128)
    t = torch.randint(0, cfg.vocab_size, (2, 6), generator=g).cuda()
    par = [-1, 0, 0, 1, 3, 2]
    c.draft(par, start=[13, 0])
    alone.draft(par)
    assert torch.equal(c.draft_positions()[:1], alone.draft_positions())
    with torch.no_grad():
        both = model(t, position_ids=c.draft_positions(), past_key_values=c, use_cache=True).logits[0].float()
        one = model(t[:1], position_ids=alone.draft_positions(), past_key_values=alone, use_cache=True).logits[0].float()
    assert ((both - one).abs().max() / one.abs().max()).item() < 5e-3


def _filled(B, layers=3, tail=32, tokens=90, seed=1, dtype=torch.float16):
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    g = torch.Generator().manual_seed(seed)
    c = ResidentKVCache(bits_per_dim=4, tail_tokens=tail)
    for i in range(layers):
        k, v = (torch.randn(B, 2, tokens, 128, generator=g).to(dtype).cuda() for _ in range(2))
        k[..., 5] *= 12
        c.update(k, v, i)
    return c


@gpu
@pytest.mark.parametrize("tail", [0, 32, 128])
def test_reorder_select_and_repeat_gpu(tail):
    from latticequant_amd import codec
    c = _filled(4, tail=tail)
    q = torch.randn(4, 8, 1, 128, device="cuda").half()
    ref = [[x.clone() for x in c.materialise(i)] for i in range(3)]
    at = torch.arange(4)
    for how, idx in (("reorder", [2, 0, 2, 1]), ("reorder", [0, 1, 2, 3]), ("select", [3, 1, 0]), ("repeat", 2),
                     ("reorder", [5, 0, 1, 1, 4, 2])):
        if how == "reorder":
            c.reorder_cache(torch.tensor(idx, device="cuda"))
        elif how == "select":
            c.batch_select_indices(torch.tensor(idx))
        else:
            c.batch_repeat_interleave(idx)
            idx = torch.arange(at.numel()).repeat_interleave(idx).tolist()
        at = at[idx]
        for i in range(3):
            for x, y in zip(c.materialise(i), ref[i]):
                assert torch.equal(x, y[at.cuda()]), (how, i)
        assert c.get_seq_length() == 90
        if c.chunks[0]:
            half = c.chunks[1][0][0]
            rows = codec.decode_batch(half.batch).reshape(4, 2, -1, 128)
            now = torch.arange(4) if half.rows is None else half.rows.cpu()
            assert torch.equal(now, at) or how == "reorder" and idx == [0, 1, 2, 3]
            assert torch.equal(rows[now.cuda()], c.materialise(1)[0][:, :, :rows.shape[2]])
    held = c.compressed_bytes()
    c.offload_at_rest()
    c.restore_at_rest()
    assert c.compressed_bytes() == held and (not c.chunks[0] or torch.equal(c.chunks[0][0][0].rows.cpu(), at))
    # the cache is used on: a step whose tail flushes, attention over it
    new = torch.randn(6, 2, 16, 128, device="cuda").half()
    c.update(new, new, 0)
    out = c.attend(0, torch.randn(6, 8, 1, 128, device="cuda").half())
    assert torch.isfinite(out).all() and q is not None


@gpu
def test_reorder_leaves_callers_tensors_gpu():
    """The prompt's own K / V may be the tail (nothing flushed): reordering must not write them."""
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    c = ResidentKVCache(bits_per_dim=4, tail_tokens=128)
    k = torch.randn(3, 2, 20, 128, device="cuda").half()
    keep = k.clone()
    c.update(k, k, 0)
    c.reorder_cache(torch.tensor([1, 2, 0], device="cuda"))
    assert torch.equal(k, keep) and torch.equal(c.materialise(0)[0], keep[[1, 2, 0]])


@gpu
@pytest.mark.parametrize("tail", [0, 128])
def test_sequence_numbers_beyond_the_batch_gpu(tail):
    """Negative numbers count from the end and others are clamped, in the prefix, the tail
    and the chunks alike."""
    for how in ("reorder_cache", "batch_select_indices"):
        c = _filled(3, layers=1, tail=tail)
        ref = [x.clone() for x in c.materialise(0)]
        getattr(c, how)(torch.tensor([-1, 7, 0]))
        for x, y in zip(c.materialise(0), ref):
            assert torch.equal(x, y[[2, 2, 0]]), how
        assert all(e.rows.tolist() == [2, 2, 0] for pair in c.chunks[0] for e in pair)
        with pytest.raises(ValueError):
            getattr(c, how)(torch.tensor([0.0, 1.0, 2.0]))


@gpu
def test_accept_keeps_within_the_nodes_and_the_buffers_gpu():
    """A path's numbers are clamped to the nodes; the tails' buffers are the tails' own
    after a step or a flush in between."""
    c = _filled(2, layers=2, tail=64, tokens=20)
    want = [[x.clone() for x in c.materialise(i)] for i in range(2)]
    g = torch.Generator().manual_seed(5)
    for path, between in (([[0, 9], [-3, 1]], True), ([[0, 2], [0, 1]], True), ([[0, 1, 2], [0, 1, 2]], False)):
        c.draft([-1, 0, 1])
        d = [[torch.randn(2, 2, 3, 128, generator=g).half().cuda() for _ in range(2)] for _ in range(2)]
        for i in range(2):
            c.update(*d[i], i)
        c.accept(torch.tensor(path, device="cuda"))
        at = torch.tensor(path).clamp(0, 2).cuda()[:, None, :, None].expand(-1, 2, -1, 128)
        for i in range(2):
            want[i] = [torch.cat([w, x.gather(2, at)], 2) for w, x in zip(want[i], d[i])]
        if between:
            one = torch.randn(2, 2, 1, 128, generator=g).half().cuda()
            for i in range(2):
                c.update(one, one, i)
                want[i] = [torch.cat([w, one], 2) for w in want[i]]
        for i in range(2):
            assert all(torch.equal(x, w) for x, w in zip(c.materialise(i), want[i]))


@gpu
def test_drafts_behind_an_empty_tail_gpu():
    """Everything cached is compressed: the drafts follow the prefix at once."""
    from latticequant_amd.llm.tree import resident_tree_attention
    c = _filled(2, layers=2, tail=0, tokens=48)
    assert c.tail_k[0].shape[2] == 0
    g = torch.Generator().manual_seed(6)
    c.draft([-1, 0, 0])
    d = [[torch.randn(2, 2, 3, 128, generator=g).half().cuda() for _ in range(2)] for _ in range(2)]
    q = torch.randn(2, 8, 3, 128, generator=g).half().cuda()
    for i in range(2):
        c.update(*d[i], i)
        out = c.attend_drafts(i, q)
        want = resident_tree_attention(c.res_k[i], c.res_v[i], q, *d[i], torch.tensor([-1, 0, 0]))
        assert torch.equal(out.transpose(1, 2), want)
    before = [c.materialise(i)[0].clone() for i in range(2)]
    c.accept(torch.tensor([[0, 2], [0, 1]], device="cuda"))
    for i in range(2):
        new = torch.stack([d[i][0][0][:, [0, 2]], d[i][0][1][:, [0, 1]]])
        assert torch.equal(c.materialise(i)[0], torch.cat([before[i], new], 2))


@gpu
def test_generate_with_beams_gpu():
    """HF's beam search over the cache: with nothing flushed the cache holds the model's own
    fp16 K / V, and the beams found are as likely as DynamicCache's (the same up to a near
    tie); over a compressed prefix it runs."""
    from transformers.cache_utils import DynamicCache
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    model, cfg = _model()
    ids = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(2)).cuda()
    kw = dict(num_beams=3, max_new_tokens=12, do_sample=False, return_dict_in_generate=True, output_scores=True,
              pad_token_id=0, eos_token_id=None)
    a = model.generate(ids, past_key_values=ResidentKVCache(bits_per_dim=4, tail_tokens=256), **kw)
    b = model.generate(ids, past_key_values=DynamicCache(), **kw)
    assert (a.sequences_scores - b.sequences_scores).abs().max() < 2e-2
    c = model.generate(ids, past_key_values=ResidentKVCache(bits_per_dim=5, tail_tokens=16), **kw)
    assert c.sequences.shape == b.sequences.shape


def test_draft_refusals():
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    c = ResidentKVCache(bits_per_dim=4, tail_tokens=128)
    with pytest.raises(ValueError):
        c.draft([-1, 0])                                     # nothing cached
    k = torch.randn(2, 1, 4, 128).half()
    c.update(k, k, 0)
    for bad in ([[-1, 0]], [[-1.0], [-1.0]], [], [[[-1]], [[-1]]], [-1] * 257):
        with pytest.raises((ValueError, TypeError)):
            c.draft(bad)
    with pytest.raises(ValueError):
        c.draft([-1, 0], start=[1])
    with pytest.raises(ValueError):
        c.draft_positions()
    c.draft([-1, 0, 0])
    assert c.draft_positions().tolist() == [[4, 5, 5]] * 2
    for f in (lambda: c.draft([-1]), lambda: c.update(k, k, 0), lambda: c.reorder_cache(torch.tensor([0, 1])),
              lambda: c.batch_select_indices(torch.tensor([0])), lambda: c.verify(torch.zeros(2, 3, dtype=torch.int64)),
              lambda: c.accept(torch.zeros(2, 1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            f()
    c.discard()
    c.update(k, k, 0)
    assert c.get_seq_length() == 8


@gpu
def test_accept_of_keys_and_values_of_two_types_gpu():
    """K and V of different types (a model under autocast rotates K in float32)."""
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    c, g = ResidentKVCache(bits_per_dim=4, tail_tokens=64), torch.Generator().manual_seed(3)
    new = lambda n: (torch.randn(2, 2, n, 128, generator=g).cuda(),   # noqa: E731
                     torch.randn(2, 2, n, 128, generator=g).bfloat16().cuda())
    for i in range(2):
        c.update(*new(20), i)
    want = [[x.clone() for x in c.materialise(i)] for i in range(2)]
    c.draft([-1, 0, 0])
    d = [new(3) for _ in range(2)]
    for i in range(2):
        c.update(*d[i], i)
    c.accept(torch.tensor([[0, 2], [0, 1]], device="cuda"))
    for i in range(2):
        for x, w, y in zip(c.materialise(i), want[i], d[i]):
            assert x.dtype == y.dtype
            assert torch.equal(x, torch.cat([w, torch.stack([y[0][:, [0, 2]], y[1][:, [0, 1]]])], 2))


class _Stand:
    """What the cache asks of a prefix, without a GPU."""

    def __init__(self, n_heads, n_tokens, device, log):
        self.n_heads, self.n_tokens, self.cap_blocks, self.log = n_heads, n_tokens, n_tokens // 16, log
        self.a = torch.empty(0, device=device)

    def select(self, index, n_seq=None, blocks=None, cap_tokens=None):
        self.log.append(self.n_heads)
        return _Stand(index.numel() * self.n_heads // n_seq, self.n_tokens, self.a.device, self.log)


def _two_devices(monkeypatch, heads=(2, 2)):
    """A cache of two layers on two devices, the moves replaced by their checks (rows and
    prefixes of one device and shape) and a record."""
    from latticequant_amd.llm import resident_cache as rc
    c, log = rc.ResidentKVCache(bits_per_dim=4, tail_tokens=64), []
    for i, dev in enumerate(("cpu", "meta")):
        c.update(*(torch.zeros(2, heads[i], 20, 128, device=dev) for _ in range(2)), i)
        c.res_k[i], c.res_v[i] = (_Stand(2 * heads[i], 32, dev, log) for _ in range(2))

    def one(ts):
        if len({(t.device, t.shape, t.dtype) for t in ts}) != 1:
            raise ValueError("rows on one GPU, of one shape and type")

    def gather(tails, index):
        one(tails)
        return [t.new_empty((index.numel(),) + t.shape[1:]) for t in tails]

    def append(tails, drafts, path, count, tail_len):
        one(tails)
        one(drafts)
        log.append(len(tails))

    def reorder(res, index, t_from=0):
        if len({(r.a.device, r.n_heads, r.n_tokens) for r in res}) != 1:
            raise ValueError("the prefixes must have the same heads, tokens and device")
        log.append(len(res))
    for name, f in (("gather_tails", gather), ("append_accepted", append), ("reorder_sequences", reorder)):
        monkeypatch.setattr(rc, name, f)
    return c, log


def test_accept_of_layers_on_two_devices(monkeypatch):
    c, log = _two_devices(monkeypatch)
    c.draft([-1, 0, 0])
    for i, dev in enumerate(("cpu", "meta")):
        c.update(*(torch.zeros(2, 2, 3, 128, device=dev) for _ in range(2)), i)
    c.accept(torch.tensor([[0, 2], [0, 1]]))
    assert log == [2, 2] and [t.shape[2] for t in c.tail_k + c.tail_v] == [22] * 4


@pytest.mark.parametrize("heads", [(2, 2), (2, 1)])
def test_sequences_of_layers_on_two_devices(monkeypatch, heads):
    """Also where the layers have different numbers of heads."""
    c, log = _two_devices(monkeypatch, heads)
    c.reorder_cache(torch.tensor([1, 0]))
    assert log == [2, 2]
    c.batch_select_indices(torch.tensor([1, 0, 1]))
    assert [r.n_heads for r in c.res_k + c.res_v] == [3 * h for h in heads] * 2
    assert [tuple(t.shape[:3]) for t in c.tail_k + c.tail_v] == [(3, h, 20) for h in heads] * 2


@pytest.mark.parametrize("fails", ["gather_tails", "select"])
def test_a_selection_that_fails_changes_nothing(monkeypatch, fails):
    from latticequant_amd.llm import resident_cache as rc
    c, _ = _two_devices(monkeypatch)
    n = 0

    def no_room(*a, **kw):
        nonlocal n
        n += 1
        if n > 1:                                        # the second call: the first one's result is there already
            raise torch.OutOfMemoryError("no room")
        return done(*a, **kw)
    done = getattr(rc, fails) if fails == "gather_tails" else _Stand.select
    monkeypatch.setattr(*((rc, fails) if fails == "gather_tails" else (_Stand, fails)), no_room)
    before = list(map(id, c.res_k + c.res_v + c.tail_k + c.tail_v))
    with pytest.raises(torch.OutOfMemoryError):
        c.batch_select_indices(torch.tensor([1, 1, 0]))
    assert list(map(id, c.res_k + c.res_v + c.tail_k + c.tail_v)) == before
    if fails == "gather_tails":
        n, moved = 0, []
        monkeypatch.setattr(rc, "reorder_sequences", lambda *a, **kw: moved.append(a))
        with pytest.raises(torch.OutOfMemoryError):
            c.reorder_cache(torch.tensor([1, 0]))
        assert not moved and list(map(id, c.tail_k + c.tail_v)) == before[4:]


@gpu
@pytest.mark.parametrize("how", ["reorder_cache", "batch_select_indices"])
def test_launches_of_a_reorder_do_not_grow_with_the_chunks_gpu(how):
    """As many operations after 3 as after 24 flushes, chunks of many epochs, some of them
    held by the host; the maps are those of chunk by chunk."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from latticequant_amd import codec

    class Count(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.n += 1
            return func(*args, **(kwargs or {}))
    g = torch.Generator().manual_seed(7)
    c, ops, maps = _filled(3, layers=2, tail=16, tokens=40), [], [[], []]
    for turn in range(24):
        for i in range(2):
            k, v = (torch.randn(3, 2, 16, 128, generator=g).half().cuda() for _ in range(2))
            c.update(k, v, i)
            maps[i] += [list(range(3))] * (len(c.chunks[i]) - len(maps[i]))
        idx = torch.randint(0, 3, (3,), generator=g)
        with Count() as n:
            getattr(c, how)(idx.cuda())
        ops.append(n.n)
        maps = [[[m[j] for j in idx.tolist()] for m in x] for x in maps]
        if turn % 2 == 0:
            getattr(c, how)(torch.tensor([1, 1, 2]).cuda())   # no flush since the last one
            maps = [[[m[j] for j in (1, 1, 2)] for m in x] for x in maps]
        if turn == 9:
            c.offload_at_rest()
        elif turn == 14:
            c.restore_at_rest()
    for i in range(2):
        assert [[e.rows.tolist() for e in pair] for pair in c.chunks[i]] == [[m, m] for m in maps[i]]
    half = c.chunks[1][3][0]
    rows = codec.decode_batch(half.batch).reshape(3, 2, -1, 128)[half.rows]
    at = sum(pair[0].batch.shape[2] for pair in c.chunks[1][:3])
    assert torch.equal(rows, c.materialise(1)[0][:, :, at:at + rows.shape[2]])
    assert len(set(ops[2:])) == 1, ops


@gpu
def test_generate_with_beams_over_a_compressed_prefix_gpu():
    """Every reorder of a beam search over flushed tokens gives each layer the rows that plain
    indexing of the materialised cache gives, and the search goes as it does with selections
    that copy the sequences."""
    from latticequant_amd.llm.resident_cache import ResidentKVCache
    seen = []

    class Checked(ResidentKVCache):
        def reorder_cache(self, beam_idx):
            before = [[x.clone() for x in self.materialise(i)] for i in range(len(self))]
            super().reorder_cache(beam_idx)
            for i, old in enumerate(before):
                for x, y in zip(self.materialise(i), old):
                    assert torch.equal(x, y[beam_idx])
            seen.append((self.res_k[0].n_tokens, beam_idx.tolist() != list(range(beam_idx.numel()))))

    class Copied(ResidentKVCache):
        def reorder_cache(self, beam_idx):
            self.batch_select_indices(beam_idx)
    model, cfg = _model()
    ids = torch.randint(0, cfg.vocab_size, (2, 40), generator=torch.Generator().manual_seed(2)).cuda()
    kw = dict(num_beams=3, max_new_tokens=40, do_sample=False, return_dict_in_generate=True, output_scores=True,
              pad_token_id=0, eos_token_id=None)
    a = model.generate(ids, past_key_values=Checked(bits_per_dim=5, tail_tokens=16), **kw)
    b = model.generate(ids, past_key_values=Copied(bits_per_dim=5, tail_tokens=16), **kw)
    assert max(n for n, _ in seen) >= 48 and any(moved for _, moved in seen)
    assert torch.equal(a.sequences, b.sequences) and torch.equal(a.sequences_scores, b.sequences_scores)


@pytest.mark.parametrize("room", [0, 1, 3, 4])
def test_a_selection_of_fewer_frees_as_it_goes(monkeypatch, room):
    """Where sequences are dropped, a layer's prefix goes as soon as its successor is there, so
    that little room is needed; without room for the first one the cache stays as it was,
    and without room later on it is empty, never a mixture."""
    import gc
    import weakref
    c, _ = _two_devices(monkeypatch)
    old = [weakref.ref(r) for r in c.res_k + c.res_v]
    before = list(map(id, c.res_k + c.res_v + c.tail_k + c.tail_v))
    select, alive = _Stand.select, []

    def counted(self, *a, **kw):
        gc.collect()
        alive.append(sum(r() is not None for r in old))
        if len(alive) > room:
            raise torch.OutOfMemoryError("no room")
        return select(self, *a, **kw)
    monkeypatch.setattr(_Stand, "select", counted)
    if room < 4:
        with pytest.raises(torch.OutOfMemoryError):
            c.batch_select_indices(torch.tensor([1]))
        if room == 0:
            assert list(map(id, c.res_k + c.res_v + c.tail_k + c.tail_v)) == before
        else:
            assert len(c) == c.get_seq_length() == 0 and not c.res_k and not c.res_v and not c.chunks
    else:
        c.batch_select_indices(torch.tensor([1]))
        assert [r.n_heads for r in c.res_k + c.res_v] == [2] * 4
    assert alive == [4, 3, 2, 1][:room + 1]
