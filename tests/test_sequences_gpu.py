"""accept_drafts, append_accepted, gather_tails, reorder_sequences and ResidentKV.select
against plain indexing; whole numbers and copies, so equality throughout."""
import pytest
import torch

gpu = pytest.mark.gpu


def _walk(tokens, parents, choice):
    B, N = tokens.shape
    path, count, nxt = torch.full((B, N), -1, dtype=torch.int32), [], []
    for b in range(B):
        if parents[b][0] != -1:
            count.append(0)
            nxt.append(-1)
            continue
        walk = [0]
        while True:
            kids = [j for j in range(walk[-1] + 1, N)
                    if parents[b][j] == walk[-1] and tokens[b][j] == choice[b][walk[-1]]]
            if not kids:
                break
            walk.append(kids[0])
        path[b, :len(walk)] = torch.tensor(walk, dtype=torch.int32)
        count.append(len(walk))
        nxt.append(int(choice[b][walk[-1]]))
    return path, torch.tensor(count, dtype=torch.int32), torch.tensor(nxt)


def _argmax(x):
    """Lowest index of the largest; NaN above all."""
    out = torch.empty(x.shape[:-1], dtype=torch.int64)
    for i, row in enumerate(x.double().reshape(-1, x.shape[-1])):
        nan = row.isnan().nonzero()
        out.view(-1)[i] = nan[0, 0] if len(nan) else (row == row.max()).nonzero()[0, 0]
    return out


def _drafts(B, N, V, seed, agree=0.7):
    g = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, min(V, 50), (B, N), generator=g)
    parents = torch.full((B, N), -2, dtype=torch.int32)
    for b in range(B):
        for i in range(N if b % 3 != 2 else max(1, N // 2)):
            parents[b, i] = -1 if i == 0 else int(torch.randint(max(0, i - 3), i, (1,), generator=g))
    return tokens, parents, g


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,N,V", [(1, 1, 1), (2, 5, 7), (3, 9, 1001), (1, 64, 32003), (2, 256, 130), (5, 3, 128256),
                                   (3, 17, 15420), (2, 256, 1024), (1, 1, 262144), (2, 6, 43690), (1, 15, 4001)])
def test_accept_logits_gpu(B, N, V, dtype):
    from latticequant_amd.llm.tree import accept_drafts
    tokens, parents, g = _drafts(B, N, V, B * 100 + N)
    logits = torch.randn(B, N, V, generator=g).to(dtype)
    for b in range(B):                                   # the model confirms most drafts; ties between two places
        for j in range(1, N):
            p = int(parents[b, j])
            if p >= 0 and float(torch.rand(1, generator=g)) < 0.7:
                logits[b, p, tokens[b, j]] = 9.0
    want = _walk(tokens, parents, _argmax(logits))
    got = accept_drafts(tokens.cuda(), parents.cuda(), logits=logits.cuda())
    for a, w in zip(got, want):
        assert torch.equal(a.cpu(), w)


@gpu
def test_accept_special_values_gpu():
    """NaN above all and the first of several, -0 equal to 0, rows of -inf, equal values far
    apart, and a vocabulary whose rows start at every alignment."""
    from latticequant_amd.llm.tree import accept_drafts
    V = 4099
    x = torch.randn(1, 8, V, generator=torch.Generator().manual_seed(0))
    x[0, 0, [900, 3000]] = float("nan")
    x[0, 1] = float("-inf")
    x[0, 2] = -1.0
    x[0, 2, 70] = -0.0
    x[0, 2, 4000] = 0.0
    x[0, 3, [4098, 2048, 2047]] = 50.0
    x[0, 4, 4098] = 60.0
    x[0, 5, 0] = float("inf")
    x[0, 6] = float("-inf")
    x[0, 6, 4097] = -1e4
    x[0, 7, 5] = float("nan")
    x[0, 7, 4] = float("inf")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        y = x.to(dtype)
        want = _argmax(y)[0]
        tokens = torch.tensor([[0] + want[:-1].tolist()])
        par = torch.arange(-1, 7, dtype=torch.int32)
        path, count, nxt = accept_drafts(tokens.cuda(), par.cuda(), logits=y.cuda())
        assert int(count) == 8 and int(nxt) == int(want[7]) and path.cpu()[0].tolist() == list(range(8))


@gpu
def test_accept_choice_and_padding_gpu():
    from latticequant_amd.llm.tree import accept_drafts
    tokens, parents, g = _drafts(6, 17, 50, 4)
    parents[4, 0] = -2                                   # an idle sequence of the batch
    choice = torch.randint(0, 50, (6, 17), generator=g)
    choice[0] = tokens[0, 1]
    for b in (1, 3, 5):
        for j in range(16, 0, -1):
            if parents[b, j] >= 0:
                choice[b, parents[b, j]] = tokens[b, j]
    want = _walk(tokens, parents, choice)
    got = accept_drafts(tokens.cuda(), parents.cuda(), choice=choice.cuda())
    for a, w in zip(got, want):
        assert torch.equal(a.cpu(), w)
    assert int(got[1][4]) == 0 and int(got[2][4]) == -1 and int(got[1][1]) > 1
    # logits as a strided view (every second node of a longer tensor)
    logits = torch.nn.functional.one_hot(choice, 50).half()
    wide = torch.zeros(6, 34, 50, dtype=torch.float16)
    wide[:, ::2] = logits
    got = accept_drafts(tokens.cuda(), parents.cuda(), logits=wide.cuda()[:, ::2])
    for a, w in zip(got, want):
        assert torch.equal(a.cpu(), w)


@gpu
def test_accept_refusals_gpu():
    from latticequant_amd.llm.tree import accept_drafts
    tokens, parents, g = _drafts(2, 5, 20, 1)
    t, p, lo, ch = tokens.cuda(), parents.cuda(), torch.zeros(2, 5, 20).cuda(), tokens.cuda()
    accept_drafts(t, p, logits=lo)
    for a, kw in (((t, p), {}), ((t, p), dict(logits=lo, choice=ch)), ((t.int(), p), dict(logits=lo)),
                  ((t.cpu(), p), dict(logits=lo)), ((t, p[:, :4]), dict(logits=lo)), ((t, p.float()), dict(logits=lo)),
                  ((t, p), dict(logits=lo[:, :4])), ((t, p), dict(logits=lo.long())), ((t, p), dict(logits=lo.cpu())),
                  ((t, p), dict(choice=ch.int())), ((t, p), dict(choice=ch[:, :4])), ((t, p), dict(logits=lo[..., :0])),
                  ((t.repeat(1, 60), p.repeat(1, 60)), dict(choice=ch.repeat(1, 60))),
                  ((t, p), dict(logits=lo, work=torch.empty(1, dtype=torch.uint8, device="cuda")))):
        with pytest.raises(ValueError):
            accept_drafts(*a, **kw)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers,B,H,N,cap", [(1, 1, 1, 1, 4), (3, 4, 3, 11, 40), (70, 2, 2, 5, 9), (2, 1, 2, 256, 300)])
def test_append_accepted_gpu(layers, B, H, N, cap, dtype):
    from latticequant_amd.llm.tree import append_accepted
    g = torch.Generator().manual_seed(layers)
    tails = [torch.randn(B, H, cap, 128, generator=g).to(dtype).cuda() for _ in range(2 * layers)]
    drafts = [torch.randn(B, N, H, 128, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2 * layers)]
    drafts[-1] = drafts[-1].contiguous()                 # another layout: a launch of its own
    count = torch.randint(0, N + 1, (B,), generator=g, dtype=torch.int32)
    count[0] = N
    path = torch.stack([torch.randperm(N, generator=g) for _ in range(B)]).to(torch.int32)
    lens = torch.randint(0, cap - N + 1, (B,), generator=g, dtype=torch.int32)
    want = [t.clone() for t in tails]
    for t, d in zip(want, drafts):
        for b in range(B):
            for j in range(int(count[b])):
                t[b, :, int(lens[b]) + j] = d[b, :, int(path[b, j])]
    new = append_accepted(tails, drafts, path.cuda(), count.cuda(), lens.cuda())
    assert torch.equal(new.cpu(), lens + count)
    for t, w in zip(tails, want):
        assert torch.equal(t, w)


@gpu
def test_append_accepted_bounds_gpu():
    """Rows past a tail's end, and path entries that are no nodes, are left out; the rows
    behind a view's end stay as they were."""
    from latticequant_amd.llm.tree import append_accepted
    buf = torch.zeros(2, 1, 12, 128, dtype=torch.float16, device="cuda")
    tail = buf[:, :, :8]
    draft = torch.arange(1, 7, device="cuda").half().reshape(1, 1, 6, 1).expand(2, 1, 6, 128).contiguous()
    path = torch.tensor([[0, 2, 3, 5, 1, 4], [-1, 3, 9, 2, 0, 0]], dtype=torch.int32, device="cuda")
    new = append_accepted([tail], [draft], path, torch.tensor([6, 4], device="cuda"), torch.tensor([5, 1], device="cuda"))
    assert new.tolist() == [8, 5]
    assert buf[0, 0, :, 0].tolist() == [0, 0, 0, 0, 0, 1, 3, 4, 0, 0, 0, 0]
    assert buf[1, 0, :, 0].tolist() == [0, 0, 4, 0, 3, 0, 0, 0, 0, 0, 0, 0]


@gpu
@pytest.mark.parametrize("B,R,T", [(1, 4, 3), (5, 5, 130), (4, 1, 17)])
def test_gather_tails_gpu(B, R, T):
    from latticequant_amd.llm.tree import gather_tails
    g = torch.Generator().manual_seed(B)
    tails = [torch.randn(B, 3, T, 128, generator=g).half().cuda() for _ in range(4)]
    tails.append(torch.randn(B, T, 3, 128, generator=g).half().cuda().transpose(1, 2))
    idx = torch.randint(0, B, (R,), generator=g)
    for a, t in zip(gather_tails(tails, idx.cuda()), tails):
        assert a.is_contiguous() and torch.equal(a, t[idx.cuda()])
    assert gather_tails([], idx) == []


@gpu
def test_row_moves_refusals_gpu():
    from latticequant_amd.llm.tree import append_accepted, gather_tails
    t = torch.zeros(2, 1, 8, 128, dtype=torch.float16, device="cuda")
    d, n = t[:, :, :3].contiguous(), torch.zeros(2, dtype=torch.int32, device="cuda")
    p = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    append_accepted([t], [d], p, n, n)
    for a in (([], [], p, n, n), ([t], [d, d], p, n, n), ([t], [d.float()], p, n, n), ([t, t[:, :, :4]], [d, d], p, n, n),
              ([t], [d[:1]], p, n, n), ([t], [d], p[:, :2], n, n), ([t], [d], p, n[:1], n), ([t], [d], p, n.float(), n),
              ([t[:1].expand(2, 1, 8, 128)], [d], p, n, n), ([t[..., :100]], [d[..., :100]], p, n, n),
              ([t.cpu()], [d.cpu()], p, n, n)):
        with pytest.raises(ValueError):
            append_accepted(*a)
    for a in (([t], n[:0]), ([t[0]], n), ([t], n.float()), ([t, t.float()], n)):
        with pytest.raises(ValueError):
            gather_tails(*a)


@gpu
def test_a_tail_twice_is_refused_gpu():
    """Two drafts of one tail would be written in no order."""
    from latticequant_amd.llm.tree import append_accepted
    t = torch.zeros(1, 1, 8, 128, dtype=torch.float16, device="cuda")
    d, n = t[:, :, :2].contiguous(), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        append_accepted([t, t], [d, d + 1], torch.zeros(1, 2, dtype=torch.int32, device="cuda"), n, n)
    assert not t.any()


def _prefix(B, H, T, seed):
    from latticequant_amd import codec
    from latticequant_amd.llm.resident import ResidentKV
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, 128, generator=g)
    x[..., torch.randperm(128, generator=g)[:4]] *= 12.0
    x = x.half().cuda()
    enc, _ = codec.encode_batch(x[None], 4)
    r = ResidentKV(B * H, T + 48, device="cuda")
    r.append(x, enc.scale32.view(-1)[:B * H], enc.scale16.view(-1)[:B * H])
    return r


PLANES = ("a", "b", "mask", "meta", "scale")


@gpu
@pytest.mark.parametrize("B,H,T,t_from,n", [(2, 3, 48, 0, 1), (4, 2, 160, 64, 6), (7, 1, 320, 304, 3), (16, 2, 64, 16, 2),
                                            (17, 1, 48, 16, 2), (128, 1, 32, 0, 1), (3, 2, 64, 64, 2), (5, 1, 32, 0, 66)])
def test_reorder_sequences_gpu(B, H, T, t_from, n):
    from latticequant_amd.llm.resident import reorder_sequences
    g = torch.Generator().manual_seed(B)
    few = [_prefix(B, H, T, 10 * B + i) for i in range(min(n, 3))]
    res = few + [_prefix(B, H, T, 7) for _ in range(n - len(few))]
    index = torch.randint(0, B, (B,), generator=g, dtype=torch.int32)
    before = [{p: getattr(r, p).clone() for p in PLANES} for r in res]
    rows = [r.dequant().reshape(B, H, T, 128) for r in res]
    reorder_sequences(res, index.cuda(), t_from=t_from)
    ix = index.long().cuda()
    for r, old, x in zip(res, before, rows):
        for p in PLANES:
            w = old[p].reshape(B, H, r.cap_blocks, -1).clone()
            w[:, :, t_from // 16:T // 16] = w[ix][:, :, t_from // 16:T // 16]
            assert torch.equal(getattr(r, p), w.reshape(-1)), p
        y = x.clone()
        y[:, :, t_from:] = x[ix][:, :, t_from:]
        assert torch.equal(r.dequant().reshape(B, H, T, 128), y)   # exceptions follow their blocks


@gpu
def test_reorder_out_of_range_and_cycle_gpu():
    """A cycle, and indices that name no sequence (their sequences stay); appends after it."""
    from latticequant_amd import codec
    r = _prefix(4, 2, 64, 3)
    x = r.dequant().reshape(4, 2, 64, 128)
    r.reorder(torch.tensor([1, 2, 0, 3], device="cuda"))
    assert torch.equal(r.dequant().reshape(4, 2, 64, 128), x[[1, 2, 0, 3]])
    r.reorder(torch.tensor([9, 0, -1, 4], device="cuda"))
    y = r.dequant().reshape(4, 2, 64, 128)
    assert torch.equal(y, x[[1, 1, 0, 3]])
    new = (torch.randn(4, 2, 16, 128, generator=torch.Generator().manual_seed(1)) * 8).half().cuda()
    enc, _ = codec.encode_batch(new[None], 4)
    r.append(new, enc.scale32.view(-1)[:8], enc.scale16.view(-1)[:8])
    z = r.dequant().reshape(4, 2, 80, 128)
    assert torch.equal(z[:, :, :64], y)
    assert torch.equal(z[:, :, 64:].reshape(-1), codec.decode_batch(enc)[0].reshape(-1))


@gpu
@pytest.mark.parametrize("B,H,T,R,keep", [(1, 2, 48, 1, None), (1, 2, 160, 4, None), (4, 3, 320, 2, 7), (3, 1, 2064, 5, 100),
                                          (2, 2, 16, 3, 1), (2, 1, 64, 2, 0), (4, 8, 2048, 4, 90)])
def test_select_gpu(B, H, T, R, keep):
    g = torch.Generator().manual_seed(R)
    r = _prefix(B, H, T, R)
    x = r.dequant().reshape(B, H, T // 16, 16, 128)
    index = torch.randint(0, B, (R,), generator=g)
    blocks = None if keep is None else torch.randint(0, T // 16, (R, keep), generator=g)
    want = x[index.cuda()]
    if blocks is not None:
        want = torch.stack([want[i][:, blocks[i].cuda()] for i in range(R)])
    n = r.select(index.cuda(), B, blocks=None if blocks is None else blocks.cuda(), cap_tokens=T + 32)
    got = n.dequant().reshape(R, H, -1, 16, 128)
    assert torch.equal(got, want) and n.n_tokens == want.shape[2] * 16 and int(n.status.item()) == 0
    assert torch.equal(r.dequant().reshape(x.shape), x)
    nb = want.shape[2]
    if nb:
        counts = n.meta.view(R * H, n.cap_blocks, 4)[:, :nb, 3].reshape(-1)
        base = n.meta.view(R * H, n.cap_blocks, 4)[:, :nb, 2].reshape(-1)
        assert torch.equal(base, (counts.cumsum(0) - counts).to(torch.int32))
        assert n.exceptions().shape[0] == int(counts.sum()) == int(n.n_exc.item())
    # the new prefix is appended to like any other
    from latticequant_amd import codec
    new = (torch.randn(R, H, 32, 128, generator=g) * 6).half().cuda()
    enc, _ = codec.encode_batch(new[None], 4)
    n.append(new, enc.scale32.view(-1)[:R * H], enc.scale16.view(-1)[:R * H])
    z = n.dequant().reshape(R, H, -1, 128)
    assert torch.equal(z[:, :, :nb * 16].reshape(-1), want.reshape(-1))
    assert torch.equal(z[:, :, nb * 16:].reshape(-1), codec.decode_batch(enc)[0].reshape(-1))


@gpu
def test_select_not_while_captured_gpu():
    r, x = _prefix(2, 1, 64, 5), torch.zeros(4, device="cuda")
    want = r.select(torch.tensor([1, 0]), 2)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError):
            r.select(torch.tensor([1, 0]), 2)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert (x == 3).all() and torch.equal(r.select(torch.tensor([1, 0]), 2).a, want.a)


@gpu
def test_select_after_a_failed_allocation_gpu(monkeypatch):
    """A selection whose planes cannot be allocated gives its read back; the next one works."""
    from latticequant_amd.llm.resident import ResidentKV
    r = _prefix(2, 1, 64, 4)
    want = r.select(torch.tensor([1, 1, 0]), 2)
    bare = ResidentKV._bare

    def fails(*a):
        raise torch.OutOfMemoryError("no room")
    for _ in range(40):                                  # more than the reads that are kept
        monkeypatch.setattr(ResidentKV, "_bare", fails)
        with pytest.raises(torch.OutOfMemoryError):
            r.select(torch.tensor([1, 1, 0]), 2)
        monkeypatch.setattr(ResidentKV, "_bare", bare)
    s = r.select(torch.tensor([1, 1, 0]), 2)
    assert all(torch.equal(getattr(s, p), getattr(want, p)) for p in PLANES)
    assert torch.equal(s.exceptions(), want.exceptions())


@gpu
def test_select_reports_dropped_exceptions_gpu():
    """A prefix whose exception list was too short stays marked when it is selected from."""
    r = _prefix(2, 1, 64, 3)
    n = r.exceptions().shape[0]
    assert n > 8
    s = r.select(torch.tensor([1, 0]), 2)
    assert int(s.status.item()) == 0 and s.exceptions().shape[0] == n
    r.exc, r._st = r.exc[:8 * 8].clone(), None           # the first eight alone are left
    s = r.select(torch.tensor([1, 0]), 2)
    assert int(s.status.item()) == 1                     # LQ_RES_ST_EXC_OVERFLOW
    assert s.exceptions().shape[0] == n and int((s.exceptions() != 0).any(1).sum()) <= 8


@gpu
def test_reorder_and_select_refusals_gpu():
    from latticequant_amd.llm.resident import ResidentKV, reorder_sequences
    r, s = _prefix(4, 1, 32, 1), _prefix(4, 1, 48, 2)
    i = torch.arange(4, device="cuda")
    for a in (([r, s], i), ([r, r], i), ([r], i.float()), ([r], i[:3]), ([r], i[None]), ([r], i[:0])):
        with pytest.raises(ValueError):
            reorder_sequences(*a)
    for t in (-16, 8, 48):
        with pytest.raises(ValueError):
            r.reorder(i, t_from=t)
    with pytest.raises(ValueError):
        ResidentKV(129, 16, device="cuda").reorder(torch.arange(129))
    reorder_sequences([], i)
    for a, kw in (((i, 3), {}), ((i, 0), {}), ((i.float(), 4), {}), ((i[None], 4), {}), ((i[:0], 4), {}),
                  ((i, 4), dict(blocks=i)), ((i, 4), dict(blocks=i[None])), ((i, 4), dict(blocks=i[:, None].float()))):
        with pytest.raises(ValueError):
            r.select(*a, **kw)
    with pytest.raises(ValueError):
        ResidentKV(4, 16, device="cuda").select(i, 4, blocks=i[:, None])
    assert ResidentKV(4, 16, device="cuda").select(i, 4).n_tokens == 0


@gpu
def test_moves_streams_and_graph_gpu():
    """On a stream of their own, and captured and replayed with changed inputs between."""
    from latticequant_amd.llm.tree import accept_drafts, append_accepted
    from latticequant_amd.llm.resident import reorder_sequences
    tokens, parents, g = _drafts(3, 9, 40, 2)
    choice = torch.randint(0, 40, (3, 9), generator=g)
    t, p = tokens.cuda(), parents.cuda()
    logits = torch.nn.functional.one_hot(choice, 1000).half().cuda()
    tail = torch.zeros(3, 2, 20, 128, dtype=torch.float16, device="cuda")
    draft = torch.randn(3, 2, 9, 128, generator=g).half().cuda()
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    res = _prefix(3, 2, 64, 5)
    ix = torch.tensor([1, 2, 0], dtype=torch.int32, device="cuda")

    def step():
        path, count, nxt = accept_drafts(t, p, logits=logits)
        new = append_accepted([tail], [draft], path, count, lens)
        reorder_sequences([res], ix, t_from=16)
        return path, count, nxt, new
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = step()
    s.synchronize()
    for a, w in zip(out, _walk(tokens, parents, choice)):
        assert torch.equal(a.cpu(), w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = step()
    for i in range(4):
        choice = torch.randint(0, 40, (3, 9), generator=g)
        choice[0, 0] = tokens[0, 1]
        logits.copy_(torch.nn.functional.one_hot(choice, 1000).half())
        lens.fill_(i)
        tail.zero_()
        before = res.dequant().reshape(3, 2, 64, 128)
        graph.replay()
        torch.cuda.synchronize()
        want = _walk(tokens, parents, choice)
        for a, w in zip(cap, want):
            assert torch.equal(a.cpu(), w)
        assert torch.equal(cap[3].cpu(), want[1] + i)
        for b in range(3):
            n = int(want[1][b])
            assert torch.equal(tail[b, :, i:i + n], draft[b][:, want[0][b, :n].long().cuda()])
            assert not tail[b, :, i + n:].any()
        after = res.dequant().reshape(3, 2, 64, 128)
        assert torch.equal(after[:, :, 16:], before[[1, 2, 0]][:, :, 16:]) and torch.equal(after[:, :, :16], before[:, :, :16])


def test_select_total_of_no_read():
    from latticequant_amd import _lib as L
    assert L.load().lq_select_total(None, None) == L.LQ_ERR_ARG


def test_workspaces_geometry():
    from latticequant_amd import _lib as L
    lib = L.load()
    assert lib.lq_accept_workspace(8, 64, 128256) > 0 and lib.lq_select_workspace(32, 2048) > 0
    for bad in ((0, 5, 10), (1, 0, 10), (1, 257, 10), (1, 5, 0), (70000, 1, 10), (1, 5, 1 << 31)):
        assert lib.lq_accept_workspace(*bad) == -1
    for bad in ((0, 5), (5, 0), (1 << 20, 1 << 20)):
        assert lib.lq_select_workspace(*bad) == -1


def test_select_needs_to_know_the_sequences():
    """Without n_seq, and none known of the prefix (or rows appended in two groupings),
    there is nothing to select from."""
    from latticequant_amd.llm.resident import ResidentKV
    i = torch.arange(2)
    r = ResidentKV(4, 16, device="cpu")
    with pytest.raises(ValueError):
        r.select(i)
    for n in (0, -1, 3):
        with pytest.raises(ValueError):
            ResidentKV(4, 16, device="cpu", n_seq=n)
    r = ResidentKV(4, 16, device="cpu", n_seq=2)
    with pytest.raises(ValueError):                      # rows of four sequences, by a prefix of two
        r.append(torch.zeros(4, 1, 16, 128), torch.ones(4), torch.ones(4).half())


@gpu
def test_select_of_known_sequences_gpu():
    """n_seq is the prefix's own by default: that of the rows appended, of its construction,
    or of the selection that made it."""
    from latticequant_amd.llm.resident import ResidentKV
    r = _prefix(3, 2, 64, 9)
    index, blocks = torch.tensor([2, 0, 2, 1], device="cuda"), torch.randint(0, 4, (4, 3), device="cuda")
    planes = ResidentKV(6, 112, device="cuda", n_seq=3)   # planes made elsewhere
    for p in PLANES + ("exc", "n_exc"):
        setattr(planes, p, getattr(r, p))
    planes.n_tokens = 64
    for b in (None, blocks):
        want = r.select(index, 3, blocks=b)
        for src in (r, planes):
            got = src.select(index, blocks=b)
            assert got.n_seq == 4 and torch.equal(got.dequant(), want.dequant())
            assert torch.equal(got.select(index[:2]).dequant(), want.select(index[:2], 4).dequant())
    assert ResidentKV(6, 16, device="cuda", n_seq=3).select(index).n_seq == 4
    flat = ResidentKV(6, 64, device="cuda")
    x, s = torch.randn(3, 2, 16, 128, device="cuda").half(), torch.full((6,), 0.25, device="cuda")
    flat.append(x, s, s.half())
    flat.append(x.reshape(1, 6, 16, 128), s, s.half())    # two groupings: which one is meant?
    with pytest.raises(ValueError):
        flat.select(index)
    assert torch.equal(flat.select(torch.tensor([1]), 3).dequant(), flat.dequant()[2:4])


@gpu
def test_row_moves_of_unaligned_sources_gpu():
    """Sources that are contiguous but start between 16-byte boundaries are copied, as those of
    odd strides are."""
    from latticequant_amd.llm.tree import append_accepted, gather_tails
    flat = torch.randn(2 * 3 * 5 * 128 + 8, device="cuda").half()
    tail = torch.zeros(2, 3, 8, 128, dtype=torch.float16, device="cuda")
    path = torch.arange(5, dtype=torch.int32, device="cuda").expand(2, 5).contiguous()
    for off in (1, 3, 4):
        d = flat[off:off + 2 * 3 * 5 * 128].view(2, 3, 5, 128)
        assert d.data_ptr() % 16
        new = append_accepted([tail], [d], path, torch.tensor([5, 2], device="cuda"), torch.tensor([0, 1], device="cuda"))
        assert new.tolist() == [5, 3] and torch.equal(tail[0, :, :5], d[0]) and torch.equal(tail[1, :, 1:3], d[1, :, :2])
        assert torch.equal(gather_tails([d], torch.tensor([1, 1, 0]))[0], d[[1, 1, 0]])
    d = torch.randn(3, 5, 128, 1, device="cuda").half().movedim(3, 0)   # a length of one whose stride is 1
    assert d.stride(0) == 1
    assert torch.equal(gather_tails([d], torch.tensor([0, 0]))[0], d[[0, 0]])
