"""One pool of resident pages for many sequences: writes and reads by page, attention of one
new token with page weights, eviction by them, against plain computations in 64 bits."""
import math

import numpy as np
import pytest
import torch

from latticequant_amd.llm.paged import (PAGE, Eviction, PagedKV, evict_pages, paged_attn_workspace,
                                        paged_decode_attention)
from latticequant_amd.llm.resident import ResidentKV

pytestmark = pytest.mark.gpu
HD = 128
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # half a step


def _rows(n, h, t, seed, loud=2, dtype=torch.float16):
    """Rows with `loud` outlier channels (exceptions), and scales of 4 bits a dimension."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, h, t, HD, generator=g, device="cuda")
    x[..., :loud] *= 5.0
    s = 0.2 + 0.1 * torch.rand(n, h, generator=g, device="cuda")
    return x.to(dtype), s


def _pool(h, n, seed, loud=2):
    p = PagedKV(h, n, device="cuda")
    x, s = _rows(n, h, PAGE, seed, loud)
    p.write(x, torch.arange(n, device="cuda")[:, None], s, s.half())
    return p


def _table(counts, n, width, seed, fill=-1):
    rng = np.random.RandomState(seed)
    order = rng.permutation(n)
    tab = np.full((len(counts), width), fill, np.int32)
    at = 0
    for b, c in enumerate(counts):
        tab[b, :c] = order[np.arange(at, at + c) % n]
        at += c
    return torch.from_numpy(tab).cuda()


def _scales(p, at, h):
    """Scales of the tokens of pages `at` of head h."""
    return p.pool.scale.view(p.n_heads, p.n_pages, PAGE)[h, at].double().reshape(-1)


def _reference(k, v, q, tab, counts, tk, tv, tails, rounded=False):
    """(out, tolerance of it, page weights, relative tolerance of those): 64 bits, from the
    lattice points times their scales (K's rounded to fp16 with page weights).

    P is rounded to fp16 (half a step, 2^-11), and so are V's coordinates beyond 1008 (2 c + 32
    beyond 2048): a row is off by at most 2 x 2^-11 times its sum of p |v| (rows of the tail
    have the sum of the rounded P instead of V's rounding).  A score is a sum of 128
    products of q and c + 16 in fp32, less 16 sum q: off by at most 130 x 2^-24 of the sum of their
    sizes, by 2^-11 of those with such a coordinate, and, where bf16 values below 2^-14 lose
    bits, by 2^-25 of the other's sizes; a weight relatively by that much twice (its own
    and the row's sum), once more for exp2 and the rounding of its argument (z below
    2^7: 2^-17).  The sums of P (c + 16) over 32 tiles: 34 roundings of at most 32 times the
    largest scale, twice.  Weights below 2^-34 of the row's largest may vanish."""
    B, Hq = q.shape[:2]
    H, G, W = k.n_heads, Hq // k.n_heads, tab.shape[1]
    every = torch.arange(k.n_pages, device="cuda")[:, None]
    rk, rv = k.read(every, torch.float16 if rounded else torch.float32).double(), v.read(every, torch.float32).double()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    w = torch.zeros(B, W, dtype=torch.float64, device="cuda")
    wtol = 0.0
    half = HALF[q.dtype]
    for b in range(B):
        c, t = counts[b], tails[b]
        if c * PAGE + t == 0:
            continue
        at = tab[b, :c].long()
        at = torch.where((at < 0) | (at >= k.n_pages), k.n_pages - 1, at)
        for h in range(H):
            kk = rk[at, h].reshape(-1, HD)
            vv = rv[at, h].reshape(-1, HD)
            sk, sv = _scales(k, at, h)[:, None], _scales(v, at, h)
            big = torch.where((2 * kk / sk).abs() > 2016, kk.abs(), 0.0)
            bias = 16 * float(sk.max()) if c else 0.0
            vmax = (float(vv.abs().max()) + 32 * float(sv.max())) if c else 0.0
            if t:
                kk = torch.cat([kk, tk[b, h, :t].double()])
                vv = torch.cat([vv, tv[b, h, :t].double()])
            qq = q[b, h * G:(h + 1) * G, 0].double()
            size = (qq.abs() @ kk.abs().t().contiguous()).amax(1) + bias * qq.abs().sum(1)
            es = 130 * 2.0 ** -24 * size + 2.0 ** -25 * (qq.abs().sum(1) + kk.abs().sum(1).max())
            if c:
                es = es + 2.0 ** -11 * (qq.abs() @ big.t().contiguous()).amax(1)
            es = es / math.sqrt(HD)
            p = torch.softmax(qq @ kk.t().contiguous() / math.sqrt(HD), 1)
            rel = 2 * es + 2.0 ** -16
            out[b, h * G:(h + 1) * G, 0] = p @ vv
            a = p @ vv.abs()
            tol[b, h * G:(h + 1) * G, 0] = (a * (2.0 ** -10 + rel[:, None]) + half * (p @ vv).abs() * (1 + 2.0 ** -9) +
                                            len(vv) * 2.0 ** -34 * max(vmax, float(vv.abs().max())) +
                                            34 * 2.0 ** -23 * vmax + 2.0 ** -24)
            if c:
                w[b, :c] += p[:, :c * PAGE].reshape(G, c, PAGE).sum((0, 2))
            wtol = max(wtol, float(rel.max()))
    return out, tol, w, wtol


def _case(B, H, G, counts, tails, dtype, seed, cap=None, width=None, loud=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = max(1, sum(counts)) + 3
    k, v = _pool(H, n, seed, loud), _pool(H, n, seed + 1, 1 if loud else 0)
    width = max(counts) if width is None else width
    tab = _table(counts, n, width, seed)
    cap = max(tails) if cap is None else cap
    q = torch.randn(B, H * G, 1, HD, generator=g, device="cuda").to(dtype)
    tk, tv = (torch.randn(B, H, cap, HD, generator=g, device="cuda").to(dtype) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return k, v, q, tab, i32(counts), tk, tv, i32(tails)


SHAPES = [
    # B, H, G, pages, tail rows
    (1, 1, 1, [0], [1]),
    (1, 1, 1, [1], [0]),
    (1, 8, 4, [31], [5]),
    (1, 2, 16, [3], [33]),
    (2, 4, 7, [5, 0], [0, 64]),
    (3, 1, 3, [1, 2, 3], [16, 1, 0]),
    (4, 2, 2, [130, 1, 0, 65], [7, 0, 0, 16]),
    (5, 8, 1, [64, 63, 62, 1, 0], [1, 31, 32, 33, 0]),
    (300, 1, 2, [i % 3 for i in range(300)], [(i * 7) % 5 for i in range(300)]),
    (2, 8, 4, [600, 257], [16, 3]),
    (1, 1, 8, [2100], [1]),
    (33, 4, 5, [(11 * i) % 40 for i in range(33)], [(5 * i) % 17 for i in range(33)]),
    (2, 2, 4, [0, 3], [1000, 700]),
    (1500, 1, 2, [(i * i) % 4 if i % 5 else 0 for i in range(1500)], [i % 3 for i in range(1500)]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}x{s[2]}-{max(s[3])}")
def test_attention_and_weights(shape, dtype):
    B, H, G, counts, tails = shape
    k, v, q, tab, cnt, tk, tv, tl = _case(B, H, G, counts, tails, dtype, 100 + B + H)
    want, tol, w, wtol = _reference(k, v, q, tab, counts, tk, tv, tails)
    got = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    assert got.dtype is dtype and got.shape == q.shape
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((got.double() - want).abs().max())}"
    if not tab.shape[1]:
        return
    want, tol, w, wtol = _reference(k, v, q, tab, counts, tk, tv, tails, rounded=True)
    old = torch.rand(tab.shape, device="cuda")
    acc = old.clone()
    again = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl, weights=acc, decay=0.75)
    assert torch.equal(again.isnan(), got.isnan())
    assert bool(((again.double() - want).abs() <= tol).all())
    on = torch.arange(tab.shape[1], device="cuda") < cnt[:, None]
    assert torch.equal(acc[~on], old[~on]), "places past the count changed"
    exp = 0.75 * old.double() + w
    # the sum over the heads and one fma: (rows + 2) roundings of 2^-24
    assert bool(((acc.double() - exp).abs() <= w * (wtol + (H * G + 2) * 2.0 ** -24) + exp * 2.0 ** -23 + 1e-30)[on].all())
    acc.fill_(float("nan"))
    paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl, weights=acc, decay=0.0)
    assert bool(((acc.double() - w).abs() <= w * (wtol + (H * G + 2) * 2.0 ** -24) + 1e-30)[on].all())
    assert bool(acc[~on].isnan().all())


@pytest.mark.parametrize("width", [0, 1, 64])
@pytest.mark.parametrize("shape", SHAPES[:9] + [(128, 4, 2, [i % 5 for i in range(128)], [i % 4 for i in range(128)]),
                                                (129, 4, 2, [i % 5 for i in range(129)], [i % 4 for i in range(129)])],
                         ids=lambda s: f"{s[0]}x{s[1]}x{s[2]}-{max(s[3])}")
def test_tables_wider_than_the_lengths(shape, width):
    """Short sequences whose table and tail would hold more: a workgroup's equal share of
    the list instead of a whole (sequence, head)."""
    B, H, G, counts, tails = shape
    k, v, q, tab, cnt, tk, tv, tl = _case(B, H, G, counts, tails, torch.float16, 7 + B + H, max(tails) + 9 * width,
                                          max(counts) + width)
    want, tol, w, wtol = _reference(k, v, q, tab, counts, tk, tv, tails)
    got = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    assert bool(((got.double() - want).abs() <= tol).all())
    want, tol, w, wtol = _reference(k, v, q, tab, counts, tk, tv, tails, rounded=True)
    acc = torch.zeros(tab.shape, device="cuda")
    got = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl, weights=acc)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert bool(((acc.double() - w).abs() <= w * (wtol + (H * G + 2) * 2.0 ** -24) + 1e-30).all())


def test_weights_sum_to_the_heads():
    k, v, q, tab, cnt, *_ = _case(3, 4, 4, [40, 7, 129], [0, 0, 0], torch.float16, 3, cap=0)
    acc = torch.zeros(tab.shape, device="cuda")
    for _ in range(3):
        paged_decode_attention(k, v, q, tab, cnt, weights=acc)
    # 3 steps x 16 heads; every weight off relatively by 2^-15 at most (see _reference, |q||k| below 2^10)
    assert torch.allclose(acc.double().sum(1), torch.full((3,), 48.0, dtype=torch.float64, device="cuda"), rtol=2 ** -10)


def test_no_pages_at_all_and_no_tail():
    k, v, q, tab, cnt, tk, tv, tl = _case(2, 2, 2, [0, 0], [3, 0], torch.float16, 5, width=0)
    got = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    want, tol, *_ = _reference(k, v, q, tab, [0, 0], tk, tv, [3, 0])
    assert bool(((got.double() - want).abs() <= tol).all()) and not bool(got[1].any())
    got = paged_decode_attention(k, v, q, tab, cnt, weights=torch.zeros(2, 0, device="cuda"))
    assert not bool(got.any())


def test_counts_and_numbers_are_clamped():
    counts, tails = [4, 3], [2, 5]
    k, v, q, tab, cnt, tk, tv, tl = _case(2, 2, 4, counts, tails, torch.float16, 6, width=4)
    wild = tab.clone()
    wild[1, 1] = 10 ** 9
    wild[1, 2] = -7
    want, tol, *_ = _reference(k, v, q, wild, counts, tk, tv, tails)
    got = paged_decode_attention(k, v, q, wild, cnt, tk, tv, tail_len=tl)
    assert bool(((got.double() - want).abs() <= tol).all())
    over = torch.tensor([99, -3], dtype=torch.int32, device="cuda")
    got = paged_decode_attention(k, v, q, tab, over, tk, tv, tail_len=torch.tensor([10 ** 6, -1], device="cuda"))
    want, tol, *_ = _reference(k, v, q, tab, [4, 0], tk, tv, [5, 0])
    assert bool(((got.double() - want).abs() <= tol).all()) and not bool(got[1].any())


def test_what_is_not_read_does_not_matter():
    counts, tails = [5, 2], [3, 1]
    k, v, q, tab, cnt, tk, tv, tl = _case(2, 2, 4, counts, tails, torch.bfloat16, 7, cap=40, width=9)
    a = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    for t in (tk, tv):
        t[0, :, 3:], t[1, :, 1:] = float("nan"), float("inf")
    used = set(tab[0, :5].tolist() + tab[1, :2].tolist())
    free = torch.tensor([i for i in range(k.n_pages) if i not in used], device="cuda")
    for p in (k, v):
        s = torch.full((len(free), 2), 3.0e4, device="cuda")
        p.write(torch.full((len(free), 2, PAGE, HD), 6.0e4, device="cuda"), free[:, None], s, s.half())
    tab[0, 5:], tab[1, 2:] = 2 ** 31 - 1, -2 ** 31
    b = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    assert torch.equal(a, b)


def test_tail_values_that_are_not_finite_reach_their_sequence_only():
    k, v, q, tab, cnt, tk, tv, tl = _case(3, 2, 2, [3, 3, 3], [4, 4, 4], torch.float16, 8)
    a = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    tk[1, 0, 2, 5] = float("nan")
    b = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2]) and torch.equal(a[1, 2:], b[1, 2:])
    assert bool(b[1, :2].isnan().all())


@pytest.mark.parametrize("layout", ["heads_last", "odd_stride", "unaligned", "expanded"])
def test_strides(layout):
    counts, tails = [9, 4], [6, 20]
    k, v, q, tab, cnt, tk, tv, tl = _case(2, 4, 4, counts, tails, torch.float16, 9)
    want = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl)
    if layout == "heads_last":
        f = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    elif layout == "odd_stride":
        f = lambda t: torch.zeros(*t.shape[:3], HD + 3, dtype=t.dtype, device="cuda")[..., :HD].copy_(t)
    elif layout == "unaligned":
        f = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    else:
        q = q[:1].expand(2, -1, -1, -1)
        tk, tv = (t[:1].expand(2, -1, -1, -1) for t in (tk, tv))
        want = paged_decode_attention(k, v, q.contiguous(), tab, cnt, tk.contiguous(), tv.contiguous(), tail_len=tl)
        f = lambda t: t
    out = torch.empty(2, 1, 16, HD, dtype=torch.float16, device="cuda").transpose(1, 2)
    got = paged_decode_attention(k, v, f(q), tab.long(), cnt.long(), f(tk), f(tv), tail_len=tl.long(), out=out)
    assert got is out and torch.equal(got, want)


def test_shared_pages_and_a_table_of_one_sequence():
    k, v, q, tab, cnt, *_ = _case(2, 2, 4, [40, 40], [0, 0], torch.float16, 10, cap=0)
    tab[1] = tab[0]
    q[1] = q[0]
    got = paged_decode_attention(k, v, q, tab, cnt)
    one = paged_decode_attention(k, v, q[:1], tab[:1], cnt[:1])
    # another division of the work, another order of the joins: both within a step of the same value
    assert bool(((got[0].float() - one[0].float()).abs() <= 2.0 ** -9 * one[0].float().abs() + 2.0 ** -10).all())
    assert torch.equal(got[0], paged_decode_attention(k, v, q, tab, cnt)[0])


def test_against_the_contiguous_prefix():
    """The same points at the same scales as a ResidentKV's, bit for bit."""
    x, s = _rows(1, 4, 96, 11)
    r = ResidentKV(4, 96, device="cuda")
    r.append(x, s, s.half())
    p = PagedKV(4, 9, device="cuda")
    at = torch.tensor([[7, 2, 0, 8, 3, 5]], device="cuda")
    p.write(x, at, s, s.half())
    for dt in (torch.float16, torch.float32, torch.bfloat16):
        assert torch.equal(p.read(at, dt)[0], r.dequant(dt))
    assert not bool(p.read(torch.tensor([[1]], device="cuda")).any())     # never written
    assert not bool(p.read(torch.tensor([[9, -1]], device="cuda")).any())  # outside
    p.write(x, at, bits=4)                                                # scales of its own
    err = (p.read(at)[0].float() - x[0].float()).square().mean() / x.float().square().mean()
    assert float(err) < 0.02


def test_pages_written_again_keep_their_room():
    p = PagedKV(2, 8, device="cuda")
    at = torch.arange(8, device="cuda")[:, None]
    seen = []
    for i in range(12):
        x, s = _rows(8, 2, PAGE, 20 + i, loud=1 + i % 4)
        p.write(x, at, s, s.half())
        r = ResidentKV(16, PAGE, device="cuda")
        r.append(x.reshape(1, 16, PAGE, HD), s.view(-1), s.view(-1).half())
        assert torch.equal(p.read(at).reshape(16, PAGE, HD), r.dequant())
        seen.append(int(p.pool.n_exc))
    before = p.read(at)
    for _ in range(3):                                     # as many exceptions again: no more room
        p.write(x, at, s, s.half())
    assert int(p.pool.n_exc) == seen[-1] and torch.equal(p.read(at), before)
    assert seen[-1] <= 2 * 16 * int(p.pool.room.max()) and int(p.pool.status) == 0
    assert int(p.pool.room.max()) <= 256


@pytest.mark.parametrize("loud", [(1, 9), (3, 3), (40, 2)])
def test_a_page_that_stands_twice_leaves_the_others(loud):
    p = _pool(2, 12, 60, loud=3)
    every = torch.arange(12, device="cuda")[:, None]
    x, s = _rows(12, 2, PAGE, 61, loud=loud[0])
    p.write(x, every, s, s.half())
    before = p.read(every)
    for i in range(3):
        x, s = _rows(4, 2, PAGE, 62 + i, loud=loud[1])
        x[1:, :, i::2] /= 8                                # exceptions in other places
        p.write(x, torch.tensor([[7], [7], [7], [2]], device="cuda"), s, s.half())
        after = p.read(every)
        others = [j for j in range(12) if j != 7 and j != 2]
        assert torch.equal(after[others], before[others])
        fresh = PagedKV(2, 1, device="cuda")
        fresh.write(x[3:], torch.zeros(1, 1, dtype=torch.int64, device="cuda"), s[3:], s[3:].half())
        assert torch.equal(after[2], fresh.read(torch.zeros(1, 1, dtype=torch.int64, device="cuda"))[0])
    p.write(x[:1], torch.tensor([[7]], device="cuda"), s[:1], s[:1].half())
    fresh.write(x[:1], torch.zeros(1, 1, dtype=torch.int64, device="cuda"), s[:1], s[:1].half())
    assert torch.equal(p.read(every)[7], fresh.read(torch.zeros(1, 1, dtype=torch.int64, device="cuda"))[0])


def test_many_exceptions_lengthen_the_list():
    """Every vector an exception, more of them than the list has room for; neighbours keep
    theirs."""
    p = PagedKV(1, 40, device="cuda", exc_cap=4)
    x, s = _rows(2, 1, PAGE, 30)
    p.write(x, torch.tensor([[0], [39]], device="cuda"), s, s.half())
    first = p.read(torch.tensor([[0], [39]], device="cuda"))
    y = torch.randn(38, 1, PAGE, HD, device="cuda") * 100
    t = torch.full((38, 1), 0.25, device="cuda")
    p.write(y, torch.arange(1, 39, device="cuda")[:, None], t, t.half())
    assert int(p.pool.n_exc) >= 38 * 250 and p.exc_cap >= int(p.pool.n_exc) and int(p.pool.status) == 0
    assert torch.equal(p.read(torch.tensor([[0], [39]], device="cuda")), first)
    r = ResidentKV(38, PAGE, device="cuda")
    r.append(y.reshape(1, 38, PAGE, HD), t.view(-1), t.view(-1).half())
    assert torch.equal(p.read(torch.arange(1, 39, device="cuda")[:, None]).reshape(38, PAGE, HD), r.dequant())
    # attention over pages that are nothing but exceptions
    q = torch.randn(1, 3, 1, HD, device="cuda").half() * 0.01
    tab = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    cnt = torch.tensor([40], dtype=torch.int32, device="cuda")
    want, tol, *_ = _reference(p, p, q, tab, [40], None, None, [0])
    assert bool(((paged_decode_attention(p, p, q, tab, cnt).double() - want).abs() <= tol).all())


def test_dropped_entries_are_zero():
    """A list shortened behind the pool's back: entries past it count as zero vectors."""
    p = _pool(2, 12, 40)
    tab, cnt = _table([12], 12, 12, 1), torch.tensor([12], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 1, HD, device="cuda").half()
    p.pool.exc = p.pool.exc[:8 * 20].clone()
    p.pool._st = None
    want, tol, *_ = _reference(p, p, q, tab, [12], None, None, [0])    # read() has them as zeros too
    assert bool(((paged_decode_attention(p, p, q, tab, cnt).double() - want).abs() <= tol).all())


def test_pool_beyond_four_gibibytes():
    """Byte offsets past 32 bits: a pool of 4.3 million pages, the last ones in use."""
    n = (1 << 22) + 70
    k, v = PagedKV(1, n, device="cuda", exc_cap=65536), PagedKV(1, n, device="cuda", exc_cap=65536)
    at = torch.tensor([[0, n - 1, 1 << 21, n - 3, (1 << 22) - 1, 1 << 22, 5]], device="cuda")
    rows = {}
    for name, p, seed in (("k", k, 1), ("v", v, 2)):
        x, s = _rows(1, 1, 7 * PAGE, 50 + seed)
        p.write(x, at, s, s.half())
        small = PagedKV(1, 7, device="cuda")
        small.write(x, torch.arange(7, device="cuda")[None], s, s.half())
        rows[name] = small
        assert torch.equal(p.read(at), small.read(torch.arange(7, device="cuda")[None]))
    q = torch.randn(1, 5, 1, HD, device="cuda").bfloat16()
    cnt = torch.tensor([7], dtype=torch.int32, device="cuda")
    order = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    a, b = torch.zeros(1, 7, device="cuda"), torch.zeros(1, 7, device="cuda")
    assert torch.equal(paged_decode_attention(k, v, q, at, cnt), paged_decode_attention(rows["k"], rows["v"], q, order, cnt))
    paged_decode_attention(k, v, q, at, cnt, weights=a)
    paged_decode_attention(rows["k"], rows["v"], q, order, cnt, weights=b)
    assert torch.equal(a, b)


def test_one_workspace_calls_of_other_sizes_and_other_streams():
    cases = [_case(2, 4, 4, [50, 3], [6, 1], torch.float16, 60), _case(5, 4, 4, [1, 0, 9, 200, 4], [1] * 5, torch.float16, 61)]
    work = torch.empty(max(paged_attn_workspace(c[2].shape[0], 4, 4, c[3].shape[1], c[5].shape[2], True).numel()
                           for c in cases), dtype=torch.uint8, device="cuda").fill_(255)
    want = [paged_decode_attention(*c[:7], tail_len=c[7]) for c in cases]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in (0, 1, 1, 0):
        acc = torch.zeros(cases[i][3].shape, device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = paged_decode_attention(*cases[i][:7], tail_len=cases[i][7], work=work, weights=acc)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.allclose(got.float(), want[i].float(), rtol=2.0 ** -9, atol=2.0 ** -10)


def test_captured_step():
    """Attention with weights, eviction and lengths that change between replays, in one graph,
    beside eager work; two graphs share the workspace."""
    counts = [30, 12, 0]
    k, v, q, tab, cnt, tk, tv, tl = _case(3, 4, 4, counts, [5, 1, 9], torch.float16, 70, cap=16, width=32)
    work = paged_attn_workspace(3, 4, 4, 32, 16, weights=True, device="cuda")
    acc, out = torch.zeros(3, 32, device="cuda"), torch.empty_like(q)
    ev = evict_pages(tab, cnt, acc, 8, 1, 2)
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl, weights=acc, decay=0.5, work=work, out=out)
            evict_pages(tab, cnt, acc, 8, 1, 2, out=ev)
        graphs.append(g)
    acc.zero_()
    exp = acc.clone()
    for step in range(6):
        q.copy_(torch.randn(q.shape, device="cuda"))
        cnt.copy_(torch.tensor([30 - step, 12, step], device="cuda"))
        if step:
            tab[2, step - 1] = tab[0, step]
        want = paged_decode_attention(k, v, q, tab, cnt, tk, tv, tail_len=tl, weights=exp, decay=0.5)
        chosen = evict_pages(tab, cnt, exp, 8, 1, 2)
        out.fill_(7.0)
        graphs[step % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(acc, exp)
        for a, b in zip(ev, chosen):
            assert torch.equal(a, b)


def test_refusals_on_the_device():
    k, v, q, tab, cnt, tk, tv, tl = _case(2, 2, 4, [4, 3], [2, 5], torch.float16, 80)
    with pytest.raises(ValueError, match="workspace too small"):
        paged_decode_attention(k, v, q, tab, cnt, tk, tv, work=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="out must be like q"):
        paged_decode_attention(k, v, q, tab, cnt, tk, tv, out=torch.empty(2, 8, 1, HD, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_decode_attention(k, v, q.float().requires_grad_().half(), tab, cnt, tk, tv)
    ev = evict_pages(tab, cnt, torch.zeros(2, 4, device="cuda"), 2)
    with pytest.raises(ValueError, match="apart"):
        evict_pages(ev.pages, ev.n_pages, ev.weights, 1, out=ev)
    raw = torch.zeros(20, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="apart"):         # one after the other, overlapping
        evict_pages(raw[2:10].view(2, 4), cnt, torch.zeros(2, 4, device="cuda"), 2,
                    out=ev._replace(pages=raw[:8].view(2, 4)))
    with pytest.raises(ValueError, match="stands twice"):
        k.write(torch.zeros(1, 2, 32, HD, device="cuda"), torch.tensor([[1, 1]]))
    x = torch.zeros(1, 2, 16, HD, device="cuda", dtype=torch.float16)
    at = torch.tensor([[1]], device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            k.write(x, at)
    torch.cuda.synchronize()


# ------------------------------------------------------------------ eviction --

def _evicted(pages, count, weight, keep, sink, recent):
    B, W = pages.shape
    out = Eviction(np.full((B, W), -1, np.int32), np.zeros(B, np.int32), np.zeros((B, W), np.float32),
                   np.full((B, W), -1, np.int32))
    for b in range(B):
        n = int(count[b])
        lo = min(sink, n)
        hi = max(lo, n - recent)
        w = weight[b, lo:hi].astype(np.float64)
        w = np.where(np.isnan(w), np.inf, np.where(np.isposinf(w), 1e300, w))
        some = lo + np.lexsort((np.arange(hi - lo), -w))[:max(0, keep - lo - (n - hi))]
        kept = np.arange(n) if n <= keep else np.sort(np.concatenate([np.arange(lo), some, np.arange(hi, n)])).astype(int)
        gone = np.setdiff1d(np.arange(n), kept)
        out.n_pages[b] = len(kept)
        out.pages[b, :len(kept)], out.weights[b, :len(kept)] = pages[b, kept], weight[b, kept]
        out.freed[b, :len(gone)] = pages[b, gone]
    return out


@pytest.mark.parametrize("W", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4097, 20011, 70001])
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_eviction(W, kind):
    rng = np.random.RandomState(W)
    B = 5 if W < 5000 else 2
    count = rng.randint(0, W + 1, B).astype(np.int32)
    count[0] = W
    pages = rng.randint(0, 2 ** 31 - 1, (B, W)).astype(np.int32)
    if kind == "spread":
        weight = np.exp(3 * rng.randn(B, W)).astype(np.float32)
    elif kind == "ties":
        weight = rng.randint(0, 3, (B, W)).astype(np.float32) * np.float32(0.1)
    else:
        weight = rng.choice(np.array([0.0, -0.0, np.nan, np.inf, 1e-42, -1.0, 5.0, -np.inf], np.float32), (B, W))
    dev = [torch.from_numpy(x).cuda() for x in (pages, count, weight)]
    for keep, sink, recent in [(0, 0, 0), (1, 0, 0), (W // 2, 0, 0), (W // 3 + 8, 3, 5), (W - 1, 0, 0), (W, 0, 0),
                               (W + 5, 2, 3), (W // 4 + 2 * W, W, W), (2, 1, 1)]:
        if keep < sink + recent:
            continue
        got = evict_pages(*dev, keep, sink, recent)
        want = _evicted(pages, count, weight, keep, sink, recent)
        for name, a, b in zip(Eviction._fields, got, want):
            assert np.array_equal(a.cpu().numpy(), b, equal_nan=name == "weights"), (name, keep, sink, recent)


def test_eviction_of_strided_inputs_and_counts_out_of_range():
    w = torch.rand(4, 64, device="cuda")
    pages = torch.arange(256, device="cuda").reshape(4, 64)
    cnt = torch.tensor([70, -2, 64, 10], device="cuda")
    got = evict_pages(pages[:, ::2], cnt, w[:, ::2], 7, 1, 1)
    want = _evicted(pages[:, ::2].cpu().numpy(), cnt.clamp(0, 32).cpu().numpy(), w[:, ::2].cpu().numpy(), 7, 1, 1)
    for a, b in zip(got, want):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("W,B", [(16384, 2), (16385, 3), (40001, 4), (70001, 1), (20000, 130)])
def test_eviction_of_long_tables(W, B):
    """Tables that one or several workgroups a sequence work on, with counts from none to all,
    ties across the workgroups' parts and protected ends longer than a part."""
    rng = np.random.RandomState(B)
    count = rng.randint(0, W + 1, B).astype(np.int32)
    count[0] = W
    if B > 2:
        count[1:3] = 0, 65
    pages = rng.randint(0, 2 ** 31 - 1, (B, W)).astype(np.int32)
    weight = rng.randint(0, 4, (B, W)).astype(np.float32)
    weight[B // 2] = np.exp(rng.randn(W))
    dev = [torch.from_numpy(x).cuda() for x in (pages, count, weight)]
    for keep, sink, recent in [(0, 0, 0), (W // 2, 4, 16), (W // 2, W // 3, 9), (W // 2, 9, W // 3), (W - 1, 0, 1)]:
        got = evict_pages(*dev, keep, sink, recent)
        for a, b in zip(got, _evicted(pages, count, weight, keep, sink, recent)):
            assert np.array_equal(a.cpu().numpy(), b), (keep, sink, recent)


# ------------------------------------------------------------------ numbers --

BEYOND = [2 ** 32, 2 ** 32 + 5, -2 ** 32 + 1, 2 ** 63 - 1, -2 ** 63, 2 ** 31]


def test_page_numbers_beyond_32_bits_are_outside_the_pool():
    p = _pool(2, 8, 90)
    every = torch.arange(8, device="cuda")[:, None]
    before = p.read(every)
    x, s = _rows(6, 2, PAGE, 91, loud=5)
    p.write(x, torch.tensor(BEYOND, device="cuda")[:, None], s, s.half())
    assert torch.equal(p.read(every), before)
    assert not bool(p.read(torch.tensor([BEYOND], device="cuda")).any())


def test_counts_and_numbers_beyond_32_bits_are_clamped():
    k, v, q, tab, cnt, tk, tv, tl = _case(2, 2, 4, [6, 6], [3, 3], torch.float16, 92, cap=5)
    wild = tab.long()
    wild[0, :len(BEYOND)] = torch.tensor(BEYOND, device="cuda")
    clamped = wild.clone()
    clamped[0, :len(BEYOND)] = k.n_pages - 1
    got = paged_decode_attention(k, v, q, wild, torch.tensor([2 ** 32 + 1, -2 ** 32 + 3], device="cuda"), tk, tv,
                                 tail_len=torch.tensor([2 ** 40, -2 ** 40 + 2], device="cuda"))
    want = paged_decode_attention(k, v, q, clamped, torch.tensor([6, 0], device="cuda"), tk, tv,
                                  tail_len=torch.tensor([5, 0], device="cuda"))
    assert torch.equal(got, want) and not bool(got[1].any()) and bool(got[0].any())
    w = torch.rand(2, 6, device="cuda")
    for a, b in zip(evict_pages(tab, torch.tensor([2 ** 33 + 2, -2 ** 33 + 2], device="cuda"), w, 3),
                    evict_pages(tab, torch.tensor([6, 0], device="cuda"), w, 3)):
        assert torch.equal(a, b)


# ------------------------------------------------------------------- scales --

def _scaled(h, n, seed, scales, loud=0):
    """A pool whose page j has rows of about three times scales[j], head by head a little apart."""
    p = PagedKV(h, n, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = torch.tensor([scales[j % len(scales)] for j in range(n)], device="cuda")[:, None].repeat(1, h)
    s[:, 1::2] *= 0.75
    s = s.half().float()
    x = torch.randn(n, h, PAGE, HD, generator=g, device="cuda") * 3 * s[:, :, None, None]
    x[..., :loud] *= 9.0
    p.write(x, torch.arange(n, device="cuda")[:, None], s, s.half())
    return p


SCALES = {"rising": [2.0 ** (i / 4 - 10) for i in range(68)], "falling": [2.0 ** (7 - i / 4) for i in range(68)],
          "mixed": [0.25, 100.0, 2.0 ** -10, 1.0, 2.0, 0.5, 1.0009765625, 2.0 ** -14, 64.0],
          "late": [0.25] * 37 + [1.5] + [0.3] * 41 + [2.0] + [0.3] * 50 + [40.0]}


@pytest.mark.parametrize("group", [4, 7, 16])
@pytest.mark.parametrize("kind", list(SCALES))
@pytest.mark.parametrize("counts,tails", [([50, 33], [5, 0]), ([300, 131, 2], [0, 17, 3])])
def test_scales_that_differ_by_page(kind, group, counts, tails):
    """V's scales from below 2^-10 to above 100 within a sequence, in the order of its pages, so that
    the weights' range is moved in the first tile, in later ones and behind a correction of the sums;
    K's scales in another order (with q small enough that a score has no more than about 30)."""
    H, n = 2, max(counts) + 3
    k, v = _scaled(H, n, 200, SCALES[kind][::-1]), _scaled(H, n, 201, SCALES[kind], loud=1)
    g = torch.Generator(device="cuda").manual_seed(202)
    B, cap = len(counts), max(tails)
    tab = torch.arange(max(counts), dtype=torch.int32, device="cuda").repeat(B, 1)
    for dtype in (torch.float16, torch.bfloat16):
        q = (torch.randn(B, H * group, 1, HD, generator=g, device="cuda") / max(SCALES[kind])).to(dtype)
        tk, tv = (torch.randn(B, H, cap, HD, generator=g, device="cuda").to(dtype) for _ in range(2))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        for w in (None, torch.zeros(B, max(counts), device="cuda")):
            want, tol, exp, wtol = _reference(k, v, q, tab, counts, tk, tv, tails, rounded=w is not None)
            got = paged_decode_attention(k, v, q, tab, i32(counts), tk, tv, tail_len=i32(tails), weights=w, decay=0.0)
            assert bool(((got.double() - want).abs() <= tol).all())
            if w is not None:
                on = torch.arange(max(counts), device="cuda") < i32(counts)[:, None]
                assert bool(((w.double() - exp).abs() <= exp * (wtol + (H * group + 2) * 2.0 ** -24) + 1e-30)[on].all())


@pytest.mark.parametrize("group", [1, 5, 16])
@pytest.mark.parametrize("scale", [2.0 ** -8, 2.0 ** -12, 2.0 ** -14])
@pytest.mark.parametrize("weights", [False, True])
def test_light_tokens_of_small_scales(scale, group, weights):
    """Tokens of 2^-17.5 of the weight of one that every wave meets, with small scales of V: what
    they give keeps its bits, as with a scale of one.  2 x 8 x 131072 tokens by pages that stand many
    times; every 32nd page's first token is the heavy one, with V = 0."""
    H, W, every = 8, 8192, 32
    k, v = PagedKV(H, 2, device="cuda"), PagedKV(H, 2, device="cuda")
    one = torch.ones(2, H, device="cuda")
    x = torch.zeros(2, H, PAGE, HD, device="cuda")
    x[1, :, 0] = 1.0                                       # the heavy token's K
    k.write(x, torch.arange(2, device="cuda")[:, None], one / 4, one.half() / 4)
    x = torch.full_like(x, 15.0) * scale
    x[1, :, 0] = 0.0
    v.write(x, torch.arange(2, device="cuda")[:, None], one * scale, one.half() * scale)
    a = 17.55 * math.log(2.0) / math.sqrt(HD)              # q k / sqrt(128) for the heavy token: 128 a / sqrt(128)
    q = torch.full((2, H * group, 1, HD), a, device="cuda").bfloat16()
    tab = (torch.arange(W, device="cuda") % every == 0).int().repeat(2, 1)
    cnt = torch.tensor([W, W], dtype=torch.int32, device="cuda")
    acc = torch.zeros(2, W, device="cuda") if weights else None
    got = paged_decode_attention(k, v, q, tab, cnt, weights=acc)
    z = float(q[0, 0, 0, 0].double()) * math.sqrt(HD)
    heavy, light = W // every, W * PAGE - W // every
    want = 15.0 * scale * light / (light + heavy * math.exp(z))
    # P rounded once (2^-11) or its sum; a score's 130 x 2^-24 of |q||k| and the bias 4 |q|, twice; exp2
    # (2^-16); the sums: 34 x 2^-23 of (15 + 32) scales; the output's rounding 2^-8
    size = 128 * abs(a) * 5 / math.sqrt(HD)
    tol = want * (2.0 ** -11 + 2 * 130 * 2.0 ** -24 * size + 2.0 ** -16 + 2.0 ** -8) + 34 * 2.0 ** -23 * 47 * scale
    err = float((got.double() - want).abs().max())
    assert err <= tol, (err / want, tol / want)


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("B,H", [(64, 8), (65, 8), (130, 8), (700, 1)])
def test_no_pages_and_no_tail_of_many_units(B, H, weights):
    """More units than are taken whole, none of which can have a token."""
    k = _pool(H, 2, 95)
    q = torch.randn(B, 2 * H, 1, HD, device="cuda").half()
    none = torch.zeros(B, 0, dtype=torch.int32, device="cuda")
    cnt = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    w = torch.zeros(B, 0, device="cuda") if weights else None
    empty = torch.zeros(B, H, 0, HD, device="cuda").half()
    for tails in ((None, None), (empty, empty)):
        out = torch.full_like(q, 7.0)
        paged_decode_attention(k, k, q, none, cnt, *tails, weights=w, out=out)
        assert not bool(out.any())
    cap, wide = torch.zeros(B, H, 9, HD, device="cuda").half(), torch.zeros(B, 3, dtype=torch.int32, device="cuda")
    w = torch.ones(B, 3, device="cuda") if weights else None
    out = torch.full_like(q, 7.0)
    paged_decode_attention(k, k, q, wide, torch.zeros_like(cnt), cap, cap, tail_len=torch.zeros_like(cnt), weights=w, out=out)
    assert not bool(out.any()) and (w is None or bool((w == 1).all()))


# ----------------------------------------------------------- exception lists --

def test_a_list_that_suffices_does_not_move():
    """Many small writes in a row, each of which might be nothing but exceptions: the list has room
    for those there are, so a graph captured over it stays right."""
    H, n = 8, 96
    k, v = (PagedKV(H, n, device="cuda", exc_cap=4096) for _ in range(2))
    x, s = _rows(n, H, PAGE, 110, loud=0)
    x /= 2                                                 # within the range: six deviations
    x[:, :, 3, 40] = 9.0                                   # an exception a page and head
    every = torch.arange(n, device="cuda")[:, None]
    k.write(x, every, s, s.half())
    v.write(x, every, s, s.half())
    tab, cnt = every.t().int().contiguous(), torch.tensor([n], dtype=torch.int32, device="cuda")
    q, out = torch.randn(1, 2 * H, 1, HD, device="cuda").half(), torch.empty(1, 2 * H, 1, HD, device="cuda").half()
    work = paged_attn_workspace(1, H, 2, n, 0, device="cuda")
    paged_decode_attention(k, v, q, tab, cnt, work=work, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_decode_attention(k, v, q, tab, cnt, work=work, out=out)
    torch.cuda.synchronize()
    at = [(p.pool.exc.data_ptr(), p.pool.rec.data_ptr()) for p in (k, v)]
    for i in range(3):
        x, s = _rows(n, H, PAGE, 111 + i, loud=0)
        x /= 2
        x[:, :, 3 + i, 40] = 9.0
        for j in range(n):
            for p in (k, v):
                p.write(x[j:j + 1], every[j:j + 1], s[j:j + 1], s[j:j + 1].half())
        assert [(p.pool.exc.data_ptr(), p.pool.rec.data_ptr()) for p in (k, v)] == at and k.exc_cap == 4096
        assert n * H <= int(k.pool.n_exc) <= 4096 - 256 * H and int(k.pool.status) == 0
        fresh = ResidentKV(n * H, PAGE, device="cuda")
        fresh.append(x.reshape(1, n * H, PAGE, HD), s.reshape(-1), s.reshape(-1).half())
        assert torch.equal(k.read(every).reshape(n * H, PAGE, HD), fresh.dequant())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged_decode_attention(k, v, q, tab, cnt))
    x = torch.randn(1, H, PAGE, HD, device="cuda") * 100   # nothing but exceptions: it has to move now
    t = torch.full((1, H), 0.25, device="cuda")
    while k.exc_cap == 4096:
        k.write(x, every[int(k.pool.n_exc) // 2048:][:1], t, t.half())
        assert int(k.pool.n_exc) <= k.exc_cap and int(k.pool.status) == 0


@pytest.mark.parametrize("cap", [1, 700, 5000])
def test_a_large_write_that_overflows_the_list(cap):
    """More than 16384 vectors at once and a list too short for their exceptions, twice, on top of
    pages that own entries: it is lengthened and the call repeated, with the rooms already taken."""
    H, n = 8, 40
    p = PagedKV(H, n, device="cuda", exc_cap=cap)
    rows, scales = _rows(n, H, PAGE, 120, loud=3)
    every = torch.arange(n, device="cuda")[:, None]

    def check():
        r = ResidentKV(n * H, PAGE, device="cuda")
        r.append(rows.reshape(1, n * H, PAGE, HD), scales.reshape(-1), scales.reshape(-1).half())
        assert int(r.status) == 0
        assert torch.equal(p.read(every).reshape(n * H, PAGE, HD), r.dequant())
        assert int(p.pool.status) == 0 and int(p.pool.n_exc) <= p.exc_cap == p.pool.rec.numel()

    p.write(rows[:4], every[:4], scales[:4], scales[:4].half())          # within the bound of small writes
    p.write(rows[4:], every[4:], scales[4:], scales[4:].half())
    grown = p.exc_cap
    assert grown > cap
    check()
    x, s = _rows(30, H, PAGE, 121, loud=100)                             # nearly all are exceptions now
    rows[5:35], scales[5:35] = x, s
    p.write(x, every[5:35], s, s.half())
    assert p.exc_cap > grown
    check()
    q = torch.randn(2, 4 * H, 1, HD, device="cuda").half() / 16
    tab = torch.stack([every[:, 0], every[:, 0].flip(0)]).int()
    cnt = torch.tensor([n, 17], dtype=torch.int32, device="cuda")
    for w in (None, torch.zeros(2, n, device="cuda")):
        want, tol, exp, wtol = _reference(p, p, q, tab, [n, 17], None, None, [0, 0], rounded=w is not None)
        got = paged_decode_attention(p, p, q, tab, cnt, weights=w)
        assert bool(((got.double() - want).abs() <= tol).all())
        if w is not None:
            assert bool(((w.double() - exp).abs() <= exp * (wtol + (4 * H + 2) * 2.0 ** -24) + 1e-30).all())


@pytest.mark.parametrize("big", [2 ** 29 - 1, 2 ** 29, 2 ** 30, 2 ** 31 - 1, 2 ** 40])
def test_eviction_that_protects_more_than_there_is(big):
    w, n = torch.rand(2, 5, device="cuda"), torch.tensor([5, 3], device="cuda")
    pages = torch.arange(10, device="cuda").reshape(2, 5)
    for keep, sink, recent in ((big, big, 0), (big, 0, big), (2 * big, big, big), (big + 1, 1, big), (big, 0, 0)):
        got = evict_pages(pages, n, w, keep, sink, recent)
        assert got.n_pages.tolist() == [5, 3] and got.pages.tolist() == [[0, 1, 2, 3, 4], [5, 6, 7, -1, -1]]
        assert bool((got.freed == -1).all())


def test_more_blocks_than_a_grid_has():
    """2^24 + 7 blocks in one write and one read: more than 2^32 threads hold, at a workgroup a block.
    All but a few numbers are outside the pool."""
    n = 2 ** 24 + 7
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("rows of 69 GB")
    p = _pool(1, 12, 130)
    num = torch.full((1, n), -1, dtype=torch.int32, device="cuda")
    places = [0, 5, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 1, n - 2, n - 1]
    for i, j in enumerate(places):
        num[0, j] = i
    before = p.read(torch.arange(7, 12, device="cuda")[None])
    x = torch.zeros(1, 1, n * PAGE, HD, dtype=torch.float16, device="cuda")
    rows, s = _rows(1, 1, len(places) * PAGE, 131, loud=3)
    for i, j in enumerate(places):
        x[:, :, j * PAGE:(j + 1) * PAGE] = rows[:, :, i * PAGE:(i + 1) * PAGE]
    p.write(x, num, s, s.half())
    del x
    fresh = ResidentKV(1, len(places) * PAGE, device="cuda")
    fresh.append(rows, s, s.half())
    want = fresh.dequant()
    assert torch.equal(p.read(torch.arange(7, device="cuda")[None])[0], want)
    assert torch.equal(p.read(torch.arange(7, 12, device="cuda")[None]), before) and int(p.pool.status) == 0
    got = p.read(num)[0, 0].view(n, PAGE, HD)
    assert torch.equal(got[places].reshape(1, -1, HD), want)
    got[places] = 0.0
    assert not bool(torch.stack([got[i:i + 2 ** 20].any() for i in range(0, n, 2 ** 20)]).any())


def test_numbers_of_entries_end_at_32_bits():
    """Rooms that would lie past 2^31 entries are in no list: the write fails, what is there stays."""
    p = _pool(8, 12, 140)
    every = torch.arange(12, device="cuda")[:, None]
    before = p.read(every[:2])
    p.pool.n_exc.fill_(2 ** 31 - 100)
    y, t = torch.randn(10, 8, PAGE, HD, device="cuda") * 100, torch.full((10, 8), 0.25, device="cuda")
    cap = p.exc_cap
    with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
        p.write(y, every[2:], t, t.half())
    assert int(p.pool.n_exc) == 2 ** 31 - 1 and p.exc_cap == cap
    assert torch.equal(p.read(every[:2]), before)
    assert not bool(p.read(every[2:]).isnan().any())


# -------------------------------------------------------------- light tokens --

@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [1, 4, 7, 16])
@pytest.mark.parametrize("pages", [1, 2, 31, 300])
def test_light_tokens_beside_a_heavy_one(pages, group, dtype, weights):
    """A first token that takes nearly all of the weight and has V = 0 (as an attention sink has), so
    that the output is what the others give: as exact relatively to that as without it.

    P is rounded once and its sum is not (2^-11), V's coordinates are exact. Sums in fp32 of
    32 tokens of a product, of up to 64 tiles a wave, of waves and workgroups: 2^-23 of the sum of
    p |v| each, 128 in all (a product of 32 tokens may drop what lies 2^-24 below its largest
    term, and each of the 32 does). Scores: 130 x 2^-24 of |q| (|k| + 16 scales), twice, 2^-16 for exp2."""
    H, n = 2, pages * PAGE
    g = torch.Generator(device="cuda").manual_seed(300 + pages)
    k, v = PagedKV(H, pages, device="cuda"), PagedKV(H, pages, device="cuda")
    one = torch.ones(pages, H, device="cuda")
    x = torch.randn(pages, H, PAGE, HD, generator=g, device="cuda") * 0.25
    x[0, :, 0] = 4.0                                       # z = 128 a 4 / sqrt(128) for the first, sum of few q k for others
    k.write(x, torch.arange(pages, device="cuda")[:, None], one / 4, one.half() / 4)
    x = torch.randn(pages, H, PAGE, HD, generator=g, device="cuda") * 3
    x[0, :, 0] = 0.0
    v.write(x, torch.arange(pages, device="cuda")[:, None], one, one.half())
    a = (math.log(100.0) + math.log(n)) / (4 * math.sqrt(HD))   # a share of 1 % for the others together
    q = torch.full((1, H * group, 1, HD), a, device="cuda") * (1 + 0.1 * torch.randn(1, H * group, 1, HD, generator=g, device="cuda"))
    q = q.to(dtype)
    tab = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cnt = torch.tensor([pages], dtype=torch.int32, device="cuda")
    got = paged_decode_attention(k, v, q, tab, cnt, weights=torch.zeros(1, pages, device="cuda") if weights else None)
    every = tab.long().t()
    for h in range(H):
        kk, vv = (p.read(every, torch.float32).double()[:, h].reshape(n, HD) for p in (k, v))
        qq = q[0, h * group:(h + 1) * group, 0].double()
        p = torch.softmax(qq @ kk.t().contiguous() / math.sqrt(HD), 1)
        want, size = p @ vv, p @ vv.abs()
        es = 130 * 2.0 ** -24 * ((qq.abs() @ kk.abs().t().contiguous()).amax(1) + 4 * qq.abs().sum(1)) / math.sqrt(HD)
        tol = (size * (2.0 ** -11 + 128 * 2.0 ** -23 + 2 * es[:, None] + 2.0 ** -16) + want.abs() * HALF[dtype] * (1 + 2.0 ** -9) +
               (2.0 ** -25 if dtype is torch.float16 else 0.0))
        err = (got[0, h * group:(h + 1) * group, 0].double() - want).abs()
        assert bool((err <= tol).all()), (float((err / tol).max()), float(p[:, 0].min()), float(err.max()), float(size.max()))


def test_a_small_write_after_one_that_found_no_room():
    """A large write whose entries have no room leaves their number known: a small one then fails
    too, where it would drop its own, instead of taking the list for long enough."""
    p = _pool(8, 12, 150)
    every = torch.arange(12, device="cuda")[:, None]
    p.pool.n_exc.fill_(2 ** 31 - 100)
    y, t = torch.randn(10, 8, PAGE, HD, device="cuda") * 100, torch.full((10, 8), 0.25, device="cuda")
    for n in (10, 1, 2):
        with pytest.raises(RuntimeError, match="fewer than 2\\^31"):
            p.write(y[:n], every[:n], t[:n], t[:n].half())
