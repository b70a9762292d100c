"""Log probabilities of given tokens, entropies and top alternatives, against 64 bits."""
import pytest
import torch

from latticequant_amd.llm.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]


def _check(x, tok, top, got):
    """Tolerances.  z = c x - r is one rounding (2^-24 |z|) of a constant off by 2^-25: with
    the logits that count within 40 of the largest, 2^-18 in all; exp2 and log2 2^-22; a lane's
    and the lanes' sums V / 2048 + 32 additions.  The entropy multiplies these by the range of
    the logits that count, at most 1 + ln V + 40 exp(-40) V, taken as 2 (1 + ln V)."""
    V = x.shape[-1]
    d = x.double().reshape(-1, V)
    lp = torch.log_softmax(d, 1)
    tol = 2.0 ** -18 + 2.0 ** -22 + (V / 2048 + 32) * 2.0 ** -23
    if tok is not None:
        want = lp.gather(1, tok.reshape(-1, 1).clamp(0, V - 1))[:, 0]
        err = (got.logprob.double().reshape(-1) - want).abs()
        far = 2.0 ** -22 * want.abs()
        ok = (err <= tol + far) | (want == got.logprob.double().reshape(-1)) | (want.isnan() & got.logprob.reshape(-1).isnan())
        assert bool(ok.all()), float(err.max())
    p = lp.exp()
    want = -torch.where(p > 0, p * lp, 0.0 * p).sum(1)
    err = (got.entropy.double().reshape(-1) - want).abs()
    ok = (err <= tol * 2 * (1 + torch.log(torch.tensor(float(V))).item())) | (want.isnan() & got.entropy.reshape(-1).isnan())
    assert bool(ok.all()), float(err.max())
    if top:
        f = x.float().reshape(-1, V)
        order = torch.where(f.isnan(), float("inf"), f)
        # NaN above +inf: two stable sorts, the lower place first of equal ones
        at = order.sort(dim=1, descending=True, stable=True).indices
        at = at.gather(1, (~f.isnan()).gather(1, at).to(torch.uint8).sort(dim=1, stable=True).indices)[:, :top]
        assert torch.equal(got.top_ids.reshape(-1, top), at)
        want = lp.gather(1, at)
        mine = got.top_logprobs.double().reshape(-1, top)
        ok = ((mine - want).abs() <= tol + 2.0 ** -22 * want.abs()) | (mine == want) | (want.isnan() & mine.isnan())
        assert bool(ok.all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (3, 7, 7), (2, 64, 64), (5, 65, 20), (1, 8191, 5),
                                            (4, 8193, 1), (1, 32000, 5), (37, 50021, 3), (1, 200003, 64), (7, 4096, 33),
                                            (300, 1000, 10), (1030, 513, 2), (2, 131072, 0), (256, 16400, 7), (257, 16400, 3),
                                            (300, 20000, 0), (1025, 16387, 0)])
def test_rows(rows, vocab, top, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + vocab)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 4).to(dtype)
    tok = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    _check(x, tok, top, token_logprobs(x, tok, top))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("order", ["up", "down", "equal", "steps"])
def test_orders(order, dtype):
    """Every logit a new largest; none; all equal; long runs of equal ones."""
    x = torch.linspace(-8, 8, 20000, device="cuda")
    x = {"up": x, "down": x.flip(0), "equal": torch.full_like(x, 3.0), "steps": (x * 2).floor()}[order]
    x = x.to(dtype)[None].repeat(2, 1)
    tok = torch.tensor([0, 19999], device="cuda")
    _check(x, tok, 64, token_logprobs(x, tok, 64))


@pytest.mark.parametrize("vocab", [3001, 40009])
@pytest.mark.parametrize("dtype", DT)
def test_masks_and_values_that_are_not_finite(dtype, vocab):
    low = torch.finfo(dtype).min
    x = torch.randn(9, vocab, device="cuda").to(dtype)
    x[0, 10:] = -float("inf")
    x[1] = -float("inf")
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4, 100:] = low
    x[5] = low
    x[6] = -low
    x[7, 3] = -low
    x[8, :-1] = -float("inf")
    tok = torch.tensor([3, 3, 3, 3, 200, 5, 5, 3, vocab - 1], device="cuda")
    got = token_logprobs(x, tok, 12)
    for r in (0, 1, 2, 5, 6, 8):
        _check(x[r:r + 1], tok[r:r + 1], 12, type(got)(*(t[r:r + 1] for t in got)))
    assert bool(got.logprob[3].isnan()) and int(got.top_ids[3, 0]) == 7
    # in 32 bits, as 64 bits have a wider range: the lowest value less the largest
    _check(x[4:5, :100], None, 12, type(got)(*(t[4:5] for t in got)))
    assert float(got.logprob[4]) <= float(low) * 0.99
    # p = 1: z and log2 l are off alike by the rounding of c m, what is left is that of log2 and of two differences
    for r in (7, 8):
        assert -2.0 ** -22 <= float(got.logprob[r]) <= 0.0 <= float(got.entropy[r]) <= 2.0 ** -22


def test_tokens_that_name_none():
    x = torch.randn(4, 100, device="cuda")
    got = token_logprobs(x, torch.tensor([-100, -1, 100, 99], device="cuda"))
    assert got.logprob[:2].tolist() == [0.0, 0.0] and bool(got.logprob[2].isnan())
    assert abs(float(got.logprob[3]) - float(torch.log_softmax(x[3].double(), 0)[99])) < 1e-5
    got = token_logprobs(x, top=2)
    assert not bool(got.logprob.any())
    _check(x, None, 2, got)


@pytest.mark.parametrize("layout", ["padded", "odd", "transposed", "expanded", "leading", "last_position"])
def test_layouts(layout):
    x = torch.randn(6, 5003, device="cuda").bfloat16()
    tok = torch.randint(0, 5003, (6,), device="cuda")
    if layout == "padded":
        y = torch.zeros(6, 5056, device="cuda").bfloat16()[:, :5003].copy_(x)
    elif layout == "odd":
        y = torch.zeros(6 * 5005 + 1, device="cuda").bfloat16()[1:].view(6, 5005)[:, :5003].copy_(x)
    elif layout == "transposed":
        y = x.t().contiguous().t()
    elif layout == "expanded":
        x = x[:1].repeat(6, 1)
        y = x[:1].expand(6, -1)
    elif layout == "leading":
        y, tok = x.view(2, 3, -1), tok.view(2, 3)
    else:
        big = torch.randn(6, 4, 5003, device="cuda").bfloat16()
        big[:, -1] = x
        y = big[:, -1]
    got = token_logprobs(y, tok, 4)
    assert got.logprob.shape == tok.shape and got.top_ids.shape == tok.shape + (4,)
    _check(x, tok, 4, got)


def test_many_rows_and_none():
    x = torch.randn(70001, 33, device="cuda").half()
    tok = torch.randint(0, 33, (70001,), device="cuda")
    _check(x, tok, 1, token_logprobs(x, tok, 1))
    got = token_logprobs(x[:0], tok[:0], 3)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 3)


def test_offsets_past_32_bits():
    """Rows that start more than 2^32 bytes behind the first."""
    n, V = 17, 1 << 28
    big = torch.empty(n * V, dtype=torch.bfloat16, device="cuda")
    x = big.view(n, V)[:, 5:40008]
    x.copy_(torch.randn(n, 40003, device="cuda"))
    tok = torch.randint(0, 40003, (n,), device="cuda")
    _check(x.contiguous(), tok, 5, token_logprobs(x, tok, 5))


def test_captured_and_other_streams():
    x = torch.randn(3, 60000, device="cuda").bfloat16()
    tok = torch.randint(0, 60000, (3,), device="cuda")
    want = token_logprobs(x, tok, 7)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = token_logprobs(x, tok, 7)
    for i in range(4):
        x.copy_(torch.randn(3, 60000, device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        want = token_logprobs(x, tok, 7)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = token_logprobs(x, tok, 7)
    torch.cuda.synchronize()
    for a, b in zip(other, want):
        assert torch.equal(a, b)


def test_refusals():
    x = torch.randn(2, 50, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        token_logprobs(x.clone().requires_grad_())


@pytest.mark.parametrize("vocab", [3001, 40009])
@pytest.mark.parametrize("value", [1e5, 1e6, 3e6, 1e7, 1e8, 1e9, 1e10, 1e12, 1e20, 1e30, 1e36, 2e38])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_of_any_finite_value(dtype, value, vocab):
    """Logits masked with -value: a run of the row, all but a few, all of them, all but lesser ones
    of like size; and logits of the size itself. (A reference of that size is off by more
    than the logits differ where c x is rounded.)"""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    low = torch.tensor(-value, device="cuda").to(dtype)
    x = (torch.randn(7, vocab, generator=g, device="cuda") * 3).to(dtype)
    x[0, vocab // 3:] = low
    x[1, 10:] = low
    x[2] = low
    x[3] = low
    x[3, ::7] = low * 1.5
    x[4, :-1] = low
    x[5] = -low
    x[5, 5:] = x[6, 5:]
    x[6] = (value + value / 64 * torch.randn(vocab, generator=g, device="cuda").clamp(-8, 8)).to(dtype)
    tok = torch.tensor([3, 3, 3, 3, vocab - 1, 2, 11], device="cuda")
    _check(x, tok, 12, token_logprobs(x, tok, 12))
    _check(x, None, 0, token_logprobs(x))
    masked = torch.full((7,), vocab // 2, device="cuda")
    got = token_logprobs(x, masked).logprob.double()
    want = torch.log_softmax(x.double(), 1).gather(1, masked[:, None])[:, 0]
    # c x, c m and ln 2 z: four roundings of the result's size
    assert bool(((got - want).abs() <= 2.0 ** -22 * want.abs() + 2.0 ** -17).all())


@pytest.mark.parametrize("vocab", [3001, 40009])
@pytest.mark.parametrize("centre", [2.0 ** 20, -2.0 ** 20, 2.0 ** 17, -2.0 ** 22])
def test_logits_of_large_size_and_small_differences(centre, vocab):
    """fp32 logits that differ by a few units far from zero: of every lane its own reference."""
    x = torch.randn(4, vocab, device="cuda") * 4 + centre
    tok = torch.randint(0, vocab, (4,), device="cuda")
    _check(x, tok, 20, token_logprobs(x, tok, 20))


@pytest.mark.parametrize("top", [0, 2])
def test_more_rows_than_a_grid_has(top):
    """2^24 + 3 rows: more than 2^32 threads hold, at a row a workgroup."""
    n, V = 2 ** 24 + 3, 5
    x = torch.randn(n, V, device="cuda").half()
    tok = torch.randint(-1, V, (n,), device="cuda")
    got = token_logprobs(x, tok, top)
    for i in (slice(0, 999), slice(2 ** 22 - 500, 2 ** 22 + 500), slice(2 ** 23 - 9, 2 ** 23 + 9), slice(n - 999, n)):
        part = [None if t is None else t[i] for t in got]
        assert not bool(part[0][tok[i] < 0].any())
        part[0] = torch.where(tok[i] < 0, torch.log_softmax(x[i].double(), 1)[:, 0].float(), part[0])
        _check(x[i], tok[i], top, type(got)(*part))
    # a sum over all of them says that none was left out
    p = torch.log_softmax(x.float(), 1)
    want = torch.where(tok < 0, 0.0, p.gather(1, tok.clamp_min(0)[:, None])[:, 0])
    assert bool(((got.logprob - want).abs() < 1e-4).all()) and bool((got.entropy > 0).all())
