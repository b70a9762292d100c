"""Steps of a server over one pool of pages: attention with page weights, log probabilities of
the sampled tokens, full pages written, the least weighted ones dropped and used again. Each
part of every step against a plain computation in 64 bits on what the step found."""
import numpy as np
import pytest
import torch

from latticequant_amd.llm.logprobs import token_logprobs
from latticequant_amd.llm.paged import PAGE, PagedKV, evict_pages, paged_attn_workspace, paged_decode_attention
from tests.test_paged_gpu import _evicted, _reference

pytestmark = pytest.mark.gpu
HD = 128
VOCAB = 517


class _Server:
    """B sequences of H kv heads and groups of G, `budget` pages each."""

    def __init__(self, B, H, G, budget, dtype, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.B, self.H, self.G, self.budget, self.dtype = B, H, G, budget, dtype
        self.k, self.v = PagedKV(H, B * (budget + 2), device="cuda"), PagedKV(H, B * (budget + 2), device="cuda")
        self.free = list(range(B * (budget + 2)))
        self.width = budget + 2
        self.tab = torch.full((B, self.width), -1, dtype=torch.int32, device="cuda")
        self.cnt = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.w = torch.zeros(B, self.width, device="cuda")
        self.tk, self.tv = (torch.zeros(B, H, PAGE, HD, dtype=dtype, device="cuda") for _ in range(2))
        self.tl = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.head = self.rand(H * G * HD, VOCAB) / 40
        self.work = paged_attn_workspace(B, H, G, self.width, PAGE, weights=True, device="cuda")

    def rand(self, *shape):
        return torch.randn(*shape, generator=self.g, device="cuda")

    def append(self, n):
        """n new rows behind each sequence; a tail that is full goes into a page first."""
        for i in range(n):
            full = [b for b in range(self.B) if int(self.tl[b]) == PAGE]
            if full:
                at = torch.tensor([[self.free.pop(0)] for _ in full], device="cuda")
                self.k.write(self.tk[full], at)
                self.v.write(self.tv[full], at)
                for b, p in zip(full, at[:, 0].tolist()):
                    self.tab[b, int(self.cnt[b])] = p
                    self.w[b, int(self.cnt[b])] = 0.0
                    self.cnt[b] += 1
                    self.tl[b] = 0
            for b in range(self.B):
                if i < n - b:                      # lengths differ
                    t = int(self.tl[b])
                    self.tk[b, :, t], self.tv[b, :, t] = (self.rand(self.H, HD).to(self.dtype) for _ in range(2))
                    self.tl[b] = t + 1

    def attend(self, q):
        return paged_decode_attention(self.k, self.v, q, self.tab, self.cnt, self.tk, self.tv, tail_len=self.tl,
                                      weights=self.w, decay=0.5, work=self.work)

    def drop(self):
        e = evict_pages(self.tab, self.cnt, self.w, self.budget, 1, 2)
        for b in range(self.B):
            gone = int(self.cnt[b]) - int(e.n_pages[b])
            self.free += e.freed[b, :gone].tolist()
        self.tab, self.cnt, self.w = e.pages, e.n_pages, e.weights
        return e


@pytest.mark.parametrize("B,H,G,budget,dtype", [(1, 2, 4, 5, torch.float16), (3, 2, 3, 4, torch.bfloat16),
                                                (2, 4, 8, 60, torch.float16)])
def test_steps(B, H, G, budget, dtype):
    s = _Server(B, H, G, budget, dtype, B)
    s.append((budget - 2) * PAGE)
    for step in range(6):
        s.append(11)
        q = s.rand(B, H * G, 1, HD).to(dtype)
        counts, tails = s.cnt.tolist(), s.tl.tolist()
        want, tol, w, wtol = _reference(s.k, s.v, q, s.tab, counts, s.tk, s.tv, tails, rounded=True)
        before = s.w.double()
        o = s.attend(q)
        assert bool(((o.double() - want).abs() <= tol).all())
        on = torch.arange(s.width, device="cuda") < s.cnt[:, None]
        exp = 0.5 * before + w
        # the sum over the heads and one fma: (rows + 2) roundings of 2^-24
        assert bool(((s.w.double() - exp).abs() <= w * (wtol + (H * G + 2) * 2.0 ** -24) + exp * 2.0 ** -23 + 1e-30)[on].all())

        logits = o.reshape(B, -1).float() @ s.head
        token = logits.argmax(1)
        lp = token_logprobs(logits, token, top=3)
        ref = torch.log_softmax(logits.double(), 1)
        assert torch.equal(lp.top_ids[:, 0], token) and torch.equal(lp.top_logprobs[:, 0], lp.logprob)
        # |logits| below 2^4: the row's sum off by 2^-14 relatively at most, the difference by two roundings of 2^-20
        assert bool((lp.logprob.double() - ref.gather(1, token[:, None])[:, 0]).abs().max() < 2.0 ** -13)

        given = [x.cpu().numpy() for x in (s.tab, s.cnt, s.w)]
        got = s.drop()
        for a, b in zip(got, _evicted(*given, s.budget, 1, 2)):
            assert np.array_equal(a.cpu().numpy(), b)
        held = [p for b in range(B) for p in s.tab[b, :int(s.cnt[b])].tolist()]
        assert sorted(held + s.free) == list(range(s.k.n_pages))
    assert s.cnt.tolist()[0] == budget                     # pages were dropped, and written again


def test_replayed_steps():
    """Attention, log probabilities and eviction of a step in one graph, the table replaced by
    the kept pages within it, against the same calls made eagerly."""
    s = _Server(2, 2, 4, 40, torch.float16, 9)
    s.append(41 * PAGE + 3)
    q = s.rand(2, 8, 1, HD).half()
    first = [x.clone() for x in (s.tab, s.cnt, s.w)]

    def step(out):
        o = paged_decode_attention(s.k, s.v, q, s.tab, s.cnt, s.tk, s.tv, tail_len=s.tl, weights=s.w, decay=0.5, work=s.work)
        lp = token_logprobs(o.reshape(2, -1), None, top=2)
        evict_pages(s.tab, s.cnt, s.w, 40, 1, 2, out=out)
        s.tab.copy_(out.pages)
        s.cnt.copy_(out.n_pages)
        s.w.copy_(out.weights)
        return o, lp

    out = evict_pages(s.tab, s.cnt, s.w, 40, 1, 2)
    step(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lp = step(out)
    seen = []
    for replayed in (False, True):
        for x, y in zip((s.tab, s.cnt, s.w), first):
            x.copy_(y)
        r = torch.Generator(device="cuda").manual_seed(3)
        for i in range(4):
            q.copy_(torch.randn(q.shape, generator=r, device="cuda"))
            if replayed:
                g.replay()
                got = (o, *lp)
            else:
                a, b = step(out)
                got = (a, *b)
            torch.cuda.synchronize()
            seen.append([x.clone() for x in (*got, s.tab, s.cnt, s.w) if x is not None])
    for a, b in zip(seen[:4], seen[4:]):
        assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))
