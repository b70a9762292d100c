"""resident_tree_attention against the formula in 64 bits.

The reference takes the prefix as the resident form's own dequantised values
(bit-exact with the oracle, test_resident_gpu.py) and walks each node's parents.

Tolerance, from the arithmetic.  w_t are the softmax weights, eps(t) half a step of
type t (fp16 2^-11, bf16 2^-8): the output is rounded once, eps(out) |o|; each weight
is rounded to fp16 once, 2^-11 sum w_t |v_t|; the scores are fp32 sums of 128 products
and the exponential and the sums are fp32, together below 2^-13 sum w_t |v_t| at these
sizes; a weight below 2^-24 of the largest is fp16-subnormal, at most 2^-35 each; the
smallest outputs are subnormal, 2^-25."""
import math

import pytest
import torch


def _tree(kind, B, N, seed):
    g = torch.Generator().manual_seed(seed)
    par = torch.full((B, N), -2, dtype=torch.int32)
    for b in range(B):
        m = N if b == 0 else int(torch.randint(1, N + 1, (1,), generator=g))
        for i in range(m):
            if i == 0 or kind == "roots":
                par[b, i] = -1
            elif kind == "chain":
                par[b, i] = i - 1
            else:
                par[b, i] = int(torch.randint(0, i, (1,), generator=g))
    return par


def _sees(par):
    """(B, N, N): node j is i or an ancestor of it; rows of padding are empty."""
    B, N = par.shape
    out = torch.zeros(B, N, N, dtype=torch.bool)
    for b, row in enumerate(par.tolist()):
        for i in range(N):
            chain, j = [], i
            while 0 <= j < N:
                chain.append(j)
                p = row[j]
                j = p if p < j else -2
            if j == -1:
                out[b, i, chain] = True
    return out


def _prefix(B, H, T, seed, outliers=True):
    from latticequant_amd import codec
    from latticequant_amd.llm.resident import ResidentKV, from_chunk
    if T == 0:
        return ResidentKV(B * H, 16, device="cuda")
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, 128, generator=g)
    if outliers:
        x[..., torch.randperm(128, generator=g)[:3]] *= 10.0   # exceptions: coordinates outside the 5-bit code
    x = x.half().cuda()
    enc, _ = codec.encode_batch(x[None], 4)
    return from_chunk(x, enc)


def _case(B, H, G, N, T, cap, seed, kind="tree", dtype=torch.float16, ragged=False, start=False):
    g = torch.Generator().manual_seed(seed)
    c = {"k": _prefix(B, H, T, seed + 1), "v": _prefix(B, H, T, seed + 2), "par": _tree(kind, B, N, seed),
         "q": torch.randn(B, H * G, N, 128, generator=g).to(dtype).cuda(), "len": None, "start": None}
    for n in ("dk", "dv"):
        c[n] = torch.randn(B, H, N, 128, generator=g).to(dtype).cuda()
    for n in ("tk", "tv"):
        c[n] = torch.randn(B, H, cap, 128, generator=g).to(dtype).cuda() if cap else None
    if ragged:
        c["len"] = torch.randint(0, cap + 1, (B,), generator=g, dtype=torch.int32)
    if start:
        c["start"] = torch.randint(0, T + cap + 1, (B,), generator=g, dtype=torch.int32)
        c["start"][0] = 0
    return c


def _run(c, **kw):
    from latticequant_amd.llm.tree import resident_tree_attention
    dev = lambda t: None if t is None else t.cuda()   # noqa: E731
    return resident_tree_attention(c["k"], c["v"], c["q"], c["dk"], c["dv"], c["par"].cuda(), c["tk"], c["tv"],
                                   tail_len=dev(c["len"]), start=dev(c["start"]), **kw)


def _reference(c):
    """(o, sum of w |v|, most tokens) in 64 bits."""
    B, Hq, N, _ = c["q"].shape
    T = c["k"].n_tokens
    H = c["k"].n_heads // B
    G = Hq // H
    sees = _sees(c["par"])
    o = torch.zeros(B, Hq, N, 128, dtype=torch.float64)
    wv = torch.zeros_like(o)
    pk, pv = (c[n].dequant().reshape(B, H, T, 128).double().cpu() for n in "kv")
    for b in range(B):
        n = 0 if c["tk"] is None else c["tk"].shape[2] if c["len"] is None else int(c["len"][b])
        s0 = 0 if c["start"] is None else int(c["start"][b])
        tail = lambda t: pk[b, :, :0] if t is None else t[b, :, :n].double().cpu()   # noqa: E731
        past_k = torch.cat([pk[b], tail(c["tk"])], 1)[:, s0:]
        past_v = torch.cat([pv[b], tail(c["tv"])], 1)[:, s0:]
        for i in range(N):
            see = sees[b, i]
            if not see.any():
                continue
            K = torch.cat([past_k, c["dk"][b].double().cpu()[:, see]], 1)
            V = torch.cat([past_v, c["dv"][b].double().cpu()[:, see]], 1)
            qq = c["q"][b, :, i].double().cpu().reshape(H, G, 128)
            w = torch.softmax(torch.matmul(qq, K.transpose(1, 2)) / math.sqrt(128), -1)
            o[b, :, i] = torch.matmul(w, V).reshape(Hq, 128)
            wv[b, :, i] = torch.matmul(w, V.abs()).reshape(Hq, 128)
    return o, wv, T + (0 if c["tk"] is None else c["tk"].shape[2]) + N


def _check(out, c):
    o, wv, n = _reference(c)
    eps = torch.finfo(out.dtype).eps / 2
    lim = eps * o.abs() + (2.0 ** -11 + 2.0 ** -13) * wv + n * 2.0 ** -35 * 8 + 2.0 ** -25
    err = (out.double().cpu() - o).abs()
    assert torch.isfinite(out).all()
    worst = (err / lim).max().item()
    print(f"tree attention: {worst:.3f} of the bound")
    assert worst <= 1.0
    gone = ~_sees(c["par"]).any(-1)
    assert (out.cpu().transpose(1, 2)[gone] == 0).all()


pytestmark = []
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("B,H,G,N,T,cap,kind", [
    (1, 2, 4, 1, 16, 0, "chain"),        # one token, one block (half a tile), no tail
    (1, 2, 4, 5, 0, 0, "tree"),          # nothing but the drafts
    (1, 1, 1, 33, 0, 7, "chain"),        # no prefix; drafts cross a tile
    (1, 2, 3, 7, 48, 33, "tree"),        # odd group, half tile, ragged tail tile
    (2, 2, 4, 16, 272, 64, "tree"),      # 64 rows: teams of two waves
    (1, 2, 7, 27, 1040, 101, "tree"),    # 189 rows: teams of four, two row blocks
    (1, 1, 16, 100, 512, 5, "tree"),     # 1600 rows, four draft words
    (1, 1, 1, 256, 96, 0, "chain"),      # the longest chain: eight draft words, the longest chain of parents
    (1, 1, 2, 256, 32, 40, "roots"),     # 256 roots: each sees the cache and itself
    (3, 1, 4, 6, 4096, 143, "chain"),    # several splits, sequences of the batch with padding nodes
])
def test_tree_attention_gpu(B, H, G, N, T, cap, kind):
    c = _case(B, H, G, N, T, cap, seed=B * 1000 + N, kind=kind)
    _check(_run(c), c)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,T", [(3, 64), (20, 800)])
def test_tree_attention_ragged_gpu(dtype, N, T):
    """Tails of different lengths (an empty one too), left padding that reaches into
    the tail, bf16."""
    c = _case(4, 2, 4, N, T, 50, seed=7 + N, dtype=dtype, ragged=True, start=True)
    c["len"][1] = 0
    c["start"][2] = T + 13
    _check(_run(c), c)


@gpu
def test_tree_attention_strides_and_out_gpu():
    """The layouts a model has: (B, N, heads, 128) transposed, a tail inside a longer
    buffer, out transposed; rows around out stay as they were; unaligned rows are copied."""
    c = _case(2, 2, 4, 9, 160, 40, seed=3)
    want = _run(c)
    d = dict(c)
    for n in ("q", "dk", "dv"):
        d[n] = c[n].transpose(1, 2).contiguous().transpose(1, 2)
    for n in ("tk", "tv"):
        big = torch.full((2, 2, 64, 128), float("nan"), dtype=torch.float16, device="cuda")
        big[:, :, :40] = c[n]
        d[n] = big[:, :, :40]
    buf = torch.full((2, 9, 8 + 1, 128), 5.0, dtype=torch.float16, device="cuda")
    out = buf[:, :, :8].transpose(1, 2)
    got = _run(d, out=out)
    assert got is out and torch.equal(got, want) and (buf[:, :, 8] == 5.0).all()
    wide = torch.zeros(2, 8, 9, 129, dtype=torch.float16, device="cuda")
    wide[..., 1:] = c["q"]
    assert torch.equal(_run(dict(c, q=wide[..., 1:])), want)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("N", [6, 40])
def test_tree_attention_masked_values_gpu(bad, N):
    """Infinities and NaN where a row does not see them leave it alone: behind a
    tail's end, before its start, in drafts that are no ancestors, in padding."""
    c = _case(2, 1, 4, N, 32, 48, seed=11, kind="chain", ragged=True, start=True)
    c["len"][:] = torch.tensor([20, 33])
    c["start"][:] = torch.tensor([0, 40])
    c["par"][0] = -1
    c["par"][0, N - 1] = 0                               # sees nodes 0 and N - 1 only
    c["par"][1, N // 2:] = -2
    clean = _run(c)
    for n in ("tk", "tv"):
        c[n][0, :, 20:] = bad
        c[n][1, :, 33:] = bad
        c[n][1, :, :8] = bad                             # tokens 32 .. 39
    for n in ("dk", "dv"):
        c[n][1, :, N // 2:] = bad
        c[n][0, :, 2, 5:77:3] = bad
    c["q"][1, :, N // 2:] = bad
    out = _run(c)
    seen = torch.ones(2, N, dtype=torch.bool)
    seen[0, 2] = False                                   # node 2 sees itself
    _, ok = out, seen.cuda()
    a, b = out.transpose(1, 2)[ok], clean.transpose(1, 2)[ok]
    assert torch.isfinite(a).all()
    # the products are taken token by token where a draft's V is not finite: other roundings
    assert (a.float() - b.float()).abs().max() <= 4 * 2.0 ** -11 * c["dv"].nan_to_num(0, 0, 0).abs().max().float()
    assert not torch.isfinite(out[0, :, 2]).all()


@gpu
def test_tree_attention_infinite_draft_seen_gpu():
    """An infinity in V reaches the rows that see it with the right sign."""
    c = _case(1, 1, 2, 5, 32, 0, seed=5, kind="chain")
    c["dv"][0, 0, 1, 3] = float("-inf")
    out = _run(c)
    assert torch.isfinite(out[0, :, 0]).all()
    assert (out[0, :, 1:, 3] == float("-inf")).all()
    assert torch.isfinite(out[0, :, 1:, 4:]).all() and torch.isfinite(out[0, :, 1:, :3]).all()


@gpu
@pytest.mark.parametrize("B,H,G,N,T,cap,dtype", [
    (4, 8, 16, 5, 4096, 70, torch.float16),      # 80 rows, much to read: teams of four
    (4, 8, 13, 11, 4112, 40, torch.bfloat16),    # 143 rows: teams of eight, half a tile at the end
    (3, 6, 16, 14, 8192, 0, torch.float16),      # 224 rows, no tail
])
def test_tree_attention_wide_teams_gpu(B, H, G, N, T, cap, dtype):
    c = _case(B, H, G, N, T, cap, seed=21, dtype=dtype, ragged=cap > 0, start=True)
    _check(_run(c), c)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_tree_attention_wide_teams_masked_values_gpu(bad):
    """As test_tree_attention_masked_values_gpu, in the kernel's widest form; rows that see
    nothing that is not finite keep their bits."""
    c = _case(4, 8, 16, 10, 4096, 48, seed=23, kind="roots", ragged=True, start=True)
    c["len"][:] = torch.tensor([20, 33, 0, 48])
    c["start"][:] = torch.tensor([0, 4100, 17, 4096])
    clean = _run(c)
    for n in ("tk", "tv"):
        c[n][0, :, 20:] = bad
        c[n][1, :, 33:] = bad
        c[n][2] = bad
        c[n][1, :, :4] = bad
    out = _run(c)
    assert torch.equal(out, clean)
    for n in ("dk", "dv"):
        c[n][1, :, 3, 7] = bad                           # its own row alone sees it
    out = _run(c)
    others = torch.arange(10, device="cuda") != 3
    assert torch.isfinite(out[:, :, others]).all() and torch.equal(out[[0, 2, 3]], clean[[0, 2, 3]])
    assert torch.equal(out[1][:, others], clean[1][:, others])


@gpu
@pytest.mark.parametrize("rows", [16, 32, 64])
def test_tree_attention_exception_counts_gpu(rows):
    """0 to 64 exceptions a block of 16 tokens, spread at random (the header names seven, a
    round takes 32): vectors with a coordinate outside the 5-bit range."""
    from latticequant_amd.llm.resident import ResidentKV
    B, H, T = 1, 2, 16 * 66
    c = _case(B, H, 4, rows // 4, 0, 20, seed=27, dtype=torch.float16)
    g = torch.Generator().manual_seed(28)
    for n in "kv":
        x = torch.randn(B * H, T // 16, 256, 8, generator=g).clamp(-3, 3)   # vectors of blocks
        for h in range(B * H):
            for i in range(T // 16):
                at = torch.randperm(256, generator=g)[:(i if h == 0 else [0, 1, 7, 8, 9, 31, 32, 33, 64, 2][i % 10])]
                x[h, i, at, i % 8] = 9.0                 # 36 steps of 0.25
        x = x.reshape(B, H, T, 128).half().cuda()
        s = torch.full((B * H,), 0.25, device="cuda")
        r = ResidentKV(B * H, T, device="cuda")
        r.append(x, s, s.half())
        counts = r.meta.view(B * H, -1, 4)[0, :T // 16, 3].cpu()
        assert counts.min() == 0 and (counts == 7).any() and (counts == 8).any() and counts.max() > 60
        c[n] = r
    _check(_run(c), c)


@gpu
def test_tree_attention_large_scores_gpu():
    """A far maximum, found late, and weights that underflow: the running maximum's rescaling."""
    c = _case(1, 2, 4, 4, 512, 40, seed=9)
    c["tk"] *= 6
    c["q"] *= 4
    _check(_run(c), c)


@gpu
def test_tree_attention_matches_decode_gpu():
    """One node over the same cache is a decode step whose tail ends with the node."""
    from latticequant_amd.llm.resident import resident_decode_attention
    c = _case(2, 4, 4, 1, 2048, 100, seed=21)
    a = _run(c)
    b = resident_decode_attention(c["k"], c["v"], c["q"], torch.cat([c["tk"], c["dk"]], 2),
                                  torch.cat([c["tv"], c["dv"]], 2))
    _check(a, c)
    _check(b, c)


@gpu
def test_tree_attention_prefix_part_stream_and_graph_gpu():
    """t_prefix, a stream of its own with a kept workspace, and a captured call replayed
    on changed inputs, each time against an eager call."""
    from latticequant_amd.llm.tree import tree_attn_workspace
    c = _case(1, 2, 4, 12, 1024, 30, seed=33, ragged=True)
    part = dict(c, k=_prefix(1, 2, 1024, 34), v=_prefix(1, 2, 1024, 35))
    work = tree_attn_workspace(2, 4, 12, 1024, 30, device="cuda")
    want = _run(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(c, work=work)
    s.synchronize()
    assert torch.equal(got, want)
    short = _run(part, t_prefix=512)
    assert not torch.equal(short, _run(part))
    par, ln = c["par"].cuda(), c["len"].cuda()
    out = torch.zeros_like(c["q"])
    from latticequant_amd.llm.tree import resident_tree_attention
    call = lambda: resident_tree_attention(c["k"], c["v"], c["q"], c["dk"], c["dv"], par, c["tk"], c["tv"],   # noqa: E731
                                           tail_len=ln, work=work, out=out)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for i in range(4):
        c["q"].copy_(torch.randn_like(c["q"]))
        ln.fill_(7 * i)
        par[0, 3] = -1 - i % 2
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, resident_tree_attention(c["k"], c["v"], c["q"], c["dk"], c["dv"], par, c["tk"],
                                                        c["tv"], tail_len=ln))


@gpu
def test_tree_workspace_shared_by_geometries_gpu():
    """One workspace for calls of other rows, heads and lengths, eager and replayed in turn:
    the results are those of a workspace of each call's own, whatever it held before."""
    from latticequant_amd.llm.tree import tree_workspace_size
    cases = [_case(*a, seed=31) for a in ((1, 2, 4, 1, 1024, 30), (2, 8, 4, 8, 2048, 0), (1, 1, 3, 1, 4096, 5),
                                          (1, 2, 8, 20, 512, 40), (3, 4, 1, 7, 1040, 9), (1, 1, 1, 1, 8192, 0))]
    size = [tree_workspace_size(c["k"].n_heads, c["q"].shape[1] * c["q"].shape[0] // c["k"].n_heads, c["q"].shape[2],
                                c["k"].n_tokens, 0 if c["tk"] is None else c["tk"].shape[2]) for c in cases]
    work = torch.empty(max(size), dtype=torch.uint8, device="cuda").fill_(0x7f)
    for c in cases:
        c["par"] = c["par"].cuda()
    want = [_run(c) for c in cases]
    for c, w in zip(cases, want):
        _check(w, c)
    graph, held = torch.cuda.CUDAGraph(), []
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = [_run(c, work=work) for c in cases]
    for turn in range(4):
        for h in held:
            h.fill_(float("nan"))
        graph.replay()
        eager = [_run(c, work=work) for c in cases[::-1]][::-1]
        torch.cuda.synchronize()
        for h, e, w in zip(held, eager, want):
            assert torch.equal(h, w) and torch.equal(e, w), turn


@gpu
def test_tree_attention_refusals_gpu():
    from latticequant_amd.llm.tree import resident_tree_attention, tree_attn_workspace
    c = _case(1, 2, 4, 5, 32, 10, seed=1)
    par = c["par"].cuda()

    def call(**kw):
        a = dict(k=c["k"], v=c["v"], q=c["q"], draft_k=c["dk"], draft_v=c["dv"], parents=par, tail_k=c["tk"],
                 tail_v=c["tv"])
        a.update(kw)
        return resident_tree_attention(**a)
    call()
    for kw in (dict(q=c["q"].float()), dict(q=c["q"][..., :64]), dict(draft_k=c["dk"][:, :, :4]),
               dict(draft_v=c["dv"].bfloat16()), dict(parents=par[:, :4]), dict(parents=par.float()), dict(tail_k=None),
               dict(tail_v=c["tv"][:, :, :9]), dict(t_prefix=24), dict(t_prefix=48), dict(t_prefix=-16),
               dict(tail_len=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(start=torch.zeros(1, device="cuda")), dict(out=c["q"].float()),
               dict(out=c["q"][:, :1].expand(-1, 8, -1, -1)), dict(q=c["q"][:, :7]), dict(q=c["q"][:0]),
               dict(q=c["q"].cpu()), dict(tail_k=None, tail_v=None, tail_len=torch.zeros(1, dtype=torch.int32)),
               dict(work=torch.empty(8, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError):
        tree_attn_workspace(2, 17, 5, 32, 10)


def test_tree_workspace_geometry():
    """Workspace sizes come from the host alone; geometries that are refused."""
    from latticequant_amd import _lib as L
    f = L.load().lq_tree_attn_workspace
    assert f(1, 8, 64, 4, 32768, 128) > 0 and f(1, 8, 1, 1, 0, 0) > 0 and f(4, 8, 256, 16, 1 << 20, 4096) > 0
    for bad in ((0, 8, 5, 4, 32, 0), (1, 0, 5, 4, 32, 0), (1, 8, 0, 4, 32, 0), (1, 8, 257, 4, 32, 0),
                (1, 8, 5, 0, 32, 0), (1, 8, 5, 17, 32, 0), (1, 8, 5, 4, 33, 0), (1, 8, 5, 4, -16, 0),
                (1, 8, 5, 4, 32, -1)):
        assert f(*bad) == -1, bad


FORMS = [(1, 2, 4, 4, 512, 20),                          # k_tree_few: 16 rows,
         (1, 2, 4, 8, 512, 20),                          # 32 rows
         (1, 2, 4, 16, 512, 20),                         # k_tree_many: two waves,
         (4, 8, 10, 10, 4096, 20),                       # four,
         (4, 8, 16, 10, 4096, 20)]                       # eight


@gpu
@pytest.mark.parametrize("B,H,G,N,T,cap", FORMS)
def test_tree_attention_rows_apart_gpu(B, H, G, N, T, cap):
    """A node that no other sees changes nobody's bits, however large its finite q, K and V."""
    c = _case(B, H, G, N, T, cap, seed=41, kind="roots")
    c["par"][:] = -1
    clean = _run(c)
    others = torch.arange(N, device="cuda") != 2
    for n, f in (("q", 30.0), ("dk", 50.0), ("dv", 1000.0)):
        c[n][:, :, 2] *= f
        out = _run(c)
        assert torch.equal(out[:, :, others], clean[:, :, others]), n
    assert torch.isfinite(out).all() and not torch.equal(out, clean)


@gpu
@pytest.mark.parametrize("B,H,G,N,T,cap", FORMS)
def test_tree_attention_dropped_exceptions_gpu(B, H, G, N, T, cap):
    """Vectors that a too short exception list dropped are zero, as dequant() has them."""
    c = _case(B, H, G, N, T, cap, seed=43)
    for n in "kv":
        r = c[n]
        counts = r.meta.view(B * H, -1, 4)[:, :T // 16, 3]
        total = int(counts.sum())
        assert total > 200
        r.exc, r._st = r.exc[:(total // 2 + 3) * 8].clone(), None
    _check(_run(c), c)


@gpu
def test_decode_attention_dropped_exceptions_gpu():
    """The one-token step has them as zero too."""
    from latticequant_amd.llm.resident import resident_decode_attention
    c = _case(2, 4, 4, 1, 1040, 30, seed=45)
    for n in "kv":
        r = c[n]
        r.exc, r._st = r.exc[:(int(r.n_exc.item()) // 2 + 3) * 8].clone(), None
    _check(resident_decode_attention(c["k"], c["v"], c["q"], torch.cat([c["tk"], c["dk"]], 2),
                                     torch.cat([c["tv"], c["dv"]], 2)), c)


@gpu
def test_tree_attention_unaligned_rows_gpu():
    """Rows that are contiguous but start between 16-byte boundaries, or have an odd stride
    over a length of one, are copied like those of other odd strides."""
    c = _case(1, 2, 4, 9, 160, 40, seed=3)
    want = _run(c)
    for off in (1, 4):
        d = dict(c)
        for n in ("q", "dk", "dv", "tk", "tv"):
            flat = torch.empty(c[n].numel() + 8, dtype=torch.float16, device="cuda")
            d[n] = flat[off:off + c[n].numel()].view(c[n].shape)
            d[n].copy_(c[n])
            assert d[n].data_ptr() % 16
        assert torch.equal(_run(d), want)
    d = dict(c, q=c["q"][0].unsqueeze(-1).movedim(3, 0))
    assert d["q"].stride(0) == 1 and torch.equal(_run(d), want)


@gpu
@pytest.mark.parametrize("kind", ["chain", "tree"])
@pytest.mark.parametrize("G,N,cap,dtype", [
    (2, 50, 40, torch.float16),          # 100 rows: teams of four, drafts over two subtiles
    (4, 40, 0, torch.bfloat16),          # 160 rows: teams of eight, a draft tile with empty subtiles
    (4, 100, 70, torch.float16),         # 400 rows: two row blocks, drafts cut within the tile
])
def test_tree_attention_wide_teams_deep_trees_gpu(G, N, cap, dtype, kind):
    """Drafts of several words of nodes where a tile holds two or four subtiles."""
    c = _case(4, 8, G, N, 4096, cap, seed=47, kind=kind, dtype=dtype, ragged=cap > 0)
    _check(_run(c), c)


@gpu
@pytest.mark.parametrize("G,N", [(2, 50), (4, 40), (4, 100)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_tree_attention_wide_teams_late_node_not_finite_gpu(G, N, bad):
    """An infinity or NaN in V of a node behind the first 32: its descendants have it, the
    others keep their bits."""
    c = _case(4, 8, G, N, 4096, 0, seed=49, kind="tree")
    for b in range(4):
        c["par"][b] = torch.tensor([-1] + [i // 2 for i in range(N - 1)])   # a full tree: all nodes valid
    clean = _run(c)
    c["dv"][1, :, 35, 3] = bad
    out = _run(c)
    hit = _sees(c["par"])[1, :, 35].cuda()
    assert 1 <= int(hit.sum()) < N - 30
    assert torch.equal(out[[0, 2, 3]], clean[[0, 2, 3]]) and torch.equal(out[1][:, ~hit], clean[1][:, ~hit])
    assert not torch.isfinite(out[1, :, hit, 3]).any()
    rest = torch.arange(128, device="cuda") != 3
    assert torch.isfinite(out[1][:, hit][..., rest]).all()
