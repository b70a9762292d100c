"""CPU tier: what paged attention, eviction and log probabilities refuse, before any GPU work."""
import ctypes

import pytest
import torch

from latticequant_amd import _lib as L
from latticequant_amd._dev import int32_on
from latticequant_amd.llm.logprobs import token_logprobs
from latticequant_amd.llm.paged import PagedKV, _apart, evict_pages, paged_decode_attention, paged_workspace_size
from latticequant_amd.llm.resident import reorder_sequences
from latticequant_amd.llm.tree import _ints


def _args(B=2, H=2, G=4, W=3, cap=5, dtype=torch.float16):
    k, v = PagedKV(H, 4, device="cpu"), PagedKV(H, 4, device="cpu")
    return dict(k=k, v=v, q=torch.zeros(B, H * G, 1, 128, dtype=dtype), pages=torch.zeros(B, W, dtype=torch.int32),
                n_pages=torch.zeros(B, dtype=torch.int32), tail_k=torch.zeros(B, H, cap, 128, dtype=dtype),
                tail_v=torch.zeros(B, H, cap, 128, dtype=dtype))


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(2, 8, 2, 128).half()), "q must be"),
    (dict(q=torch.zeros(2, 8, 1, 64).half()), "q must be"),
    (dict(q=torch.zeros(2, 8, 1, 128)), "q must be"),
    (dict(q=torch.zeros(2, 7, 1, 128).half()), "times the pools' heads"),
    (dict(q=torch.zeros(2, 34, 1, 128).half()), "times the pools' heads"),
    (dict(v=PagedKV(2, 5, device="cpu")), "same heads, pages"),
    (dict(v=PagedKV(1, 4, device="cpu")), "same heads, pages"),
    (dict(pages=torch.zeros(3, 3, dtype=torch.int32)), "pages must be"),
    (dict(pages=torch.zeros(6, dtype=torch.int32)), "pages must be"),
    (dict(tail_v=None), "go together"),
    (dict(tail_k=None, tail_v=None, tail_len=torch.zeros(2, dtype=torch.int32)), "without a tail"),
    (dict(tail_v=torch.zeros(2, 2, 4, 128).half()), "tail K / V"),
    (dict(tail_k=torch.zeros(2, 2, 5, 128).bfloat16()), "one type"),
    (dict(weights=torch.zeros(2, 4)), "weights must be"),
    (dict(weights=torch.zeros(2, 3).half()), "weights must be"),
    (dict(weights=torch.zeros(3, 2).t()), "weights must be"),
    (dict(out=torch.zeros(2, 8, 1, 128)), "out must be"),
    (dict(out=torch.zeros(1, 8, 1, 128).half().expand(2, -1, -1, -1)), "out must be"),
])
def test_attention(change, message):
    with pytest.raises(ValueError, match=message):
        paged_decode_attention(**{**_args(), **change})


def test_attention_has_no_gradient():
    a = _args()
    a["q"].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_decode_attention(**a)


def test_pools():
    for h, n in ((0, 4), (4, 0), (65536, 65536)):
        with pytest.raises(ValueError):
            PagedKV(h, n, device="cpu")
    p = PagedKV(2, 4, device="cpu")
    x = torch.zeros(1, 2, 32, 128)
    for bad, pages in ((x[:, :1], [[0, 1]]), (x[..., :64], [[0, 1]]), (x[:, :, :20], [[0]]), (x, [[0]]), (x, [[0, 4]]),
                       (x, [[-1, 0]]), (x, [[2, 2]]), (x.double(), [[0, 1]])):
        with pytest.raises(ValueError):
            p.write(bad, torch.tensor(pages))
    with pytest.raises(ValueError, match="int32 or int64"):
        p.write(x, torch.tensor([[0.0, 1.0]]))
    with pytest.raises(ValueError, match="go together"):
        p.write(x, torch.tensor([[0, 1]]), scale32=torch.ones(2))
    with pytest.raises(ValueError):
        p.read(torch.tensor([0, 1]))


def test_geometry():
    assert paged_workspace_size(4, 8, 4, 100, 16) % 16 == 0
    assert paged_workspace_size(4, 8, 4, 100, 16, True) > paged_workspace_size(4, 8, 4, 100, 16)
    for bad in ((0, 8, 4, 1, 1), (1, 0, 4, 1, 1), (1, 8, 0, 1, 1), (1, 8, 17, 1, 1), (1, 8, 4, -1, 1), (1, 8, 4, 1, -1),
                (60000, 64, 4, 1 << 20, 0)):
        with pytest.raises(ValueError):
            paged_workspace_size(*bad)


def test_c_entries_refuse_null_and_bad_sizes():
    lib = L.load()
    res = L.Resident(a=16, b=16, mask=16, meta=16, exc=16, scale=16, n_exc=16, status=16, n_heads=2, cap_blocks=4, exc_cap=1)
    rows = L.Rows(p=16, stride_b=128, stride_h=128, stride_t=128)
    odd = L.Rows(p=16, stride_b=129, stride_h=128, stride_t=128)
    pool = L.Pages(r=res, room=16, rec=16)
    r, q = ctypes.addressof(pool), ctypes.addressof(rows)

    def attend(k=r, v=r, qq=q, n=2, g=4, pages=16, width=3, counts=16, tk=q, tv=q, cap=4, work=16, nbytes=1 << 40, out=q, dt=0):
        return lib.lq_paged_attention(k, v, qq, n, g, pages, width, counts, tk, tv, cap, None, None, 1.0, dt, work, nbytes,
                                      out, None)
    for bad in (dict(k=None), dict(v=None), dict(qq=None), dict(qq=ctypes.addressof(odd)), dict(n=0), dict(g=0), dict(g=17),
                dict(pages=None), dict(counts=None), dict(tk=None), dict(cap=-1), dict(work=None), dict(work=24),
                dict(nbytes=0), dict(out=None), dict(dt=2), dict(width=-1)):
        assert attend(**bad) == L.LQ_ERR_ARG, bad
    assert lib.lq_page_quantize(None, 0, 1, 16, 16, 16, r, 16, None) == L.LQ_ERR_ARG
    assert lib.lq_page_quantize(16, 0, 1, 17, 16, 16, r, 16, None) == L.LQ_ERR_ARG
    assert lib.lq_page_dequant(r, None, 1, 1, 16, 0, None) == L.LQ_ERR_ARG
    ev = [16, 16, 16, 1, 4, 2, 1, 1, 16, 16, 16, 16, None]
    for i, x in ((0, None), (3, 0), (4, 0), (5, 1), (6, -1), (7, -1), (11, None)):
        bad = list(ev)
        bad[i] = x
        assert lib.lq_evict_pages(*bad) == L.LQ_ERR_ARG
    lp = [16, 0, 10, 1, 10, None, 0, 16, 16, None, None, None]
    for i, x in ((0, None), (1, 3), (2, -1), (3, 0), (3, 2 ** 31), (4, 0), (4, 2 ** 31), (6, -1), (6, 11), (6, 65), (7, None),
                 (8, None), (6, 2)):
        bad = list(lp)
        bad[i] = x
        assert lib.lq_token_logprobs(*bad) == L.LQ_ERR_ARG


def test_eviction_and_logprobs_need_the_gpu_and_sound_arguments():
    w, p, n = torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for a, kw in (((p, n, w, 1), {}), ((p, n, w.half(), 1), {}), ((p, n, w[0], 1), {}), ((p, n, w, 1), dict(sink=1, recent=1)),
                  ((p, n, w, -1), {}), ((p, n, w, 2), dict(sink=-1))):
        with pytest.raises(ValueError):
            evict_pages(*a, **kw)
    x = torch.zeros(2, 5)
    for a, kw in (((x,), {}), ((x.double(),), {}), ((x, torch.zeros(3, dtype=torch.int64)), {}), ((x,), dict(top=6)),
                  ((x,), dict(top=-1)), ((x[:, :0],), {})):
        with pytest.raises(ValueError):
            token_logprobs(*a, **kw)


def test_numbers_beyond_32_bits_stay_out_of_range():
    """Tables, counts and indices of 64 bits become 32-bit ones without wrapping into a range."""
    t = torch.tensor([2 ** 32, 2 ** 32 + 5, -2 ** 32 + 1, 2 ** 63 - 1, -2 ** 63, 2 ** 31, 7, -7])
    want = [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 7, -7]
    assert int32_on(t, "cpu").tolist() == want and _ints(t, (8,), "t", t.device).tolist() == want
    assert int32_on(t.int(), "cpu").tolist() == t.int().tolist()


def test_a_pool_checks_page_numbers_of_64_bits(monkeypatch):
    monkeypatch.setenv("LQ_DEBUG_CHECKS", "1")
    p = PagedKV(1, 4, device="cpu")
    for bad in (2 ** 32, -2 ** 32, 2 ** 63 - 1):
        with pytest.raises(ValueError, match="outside the pool"):
            p._numbers(torch.tensor([[bad]]), None, False)


@pytest.mark.parametrize("weights", [False, True])
def test_geometry_without_pages_and_tail(weights):
    """A table of no width and no tail is a call like any other, however many units it has."""
    for b, h in ((1, 1), (2, 2), (64, 8), (65, 8), (128, 8), (65535, 3)):
        assert paged_workspace_size(b, h, 4, 0, 0, weights) > 0


def test_the_view_of_a_pool_follows_its_buffers():
    """A longer exception list is in the next view of the pool, whatever took the resident
    form's own view in between."""
    p = PagedKV(2, 4, device="cpu", exc_cap=16)
    assert p.struct().r.exc_cap == 16 and p.struct() is p.struct()
    for cap, between in ((40, lambda: None), (90, p.pool.struct)):
        p.pool._grow_exc(cap, 16)
        between()
        st = p.struct()
        assert (st.r.exc_cap, st.r.exc, st.rec) == (cap, p.pool.exc.data_ptr(), p.pool.rec.data_ptr())
        assert p.exc_cap == cap and p.pool.rec.numel() == cap


@pytest.mark.parametrize("fails", [torch.int16, torch.uint8])
def test_a_list_that_cannot_be_lengthened_stays_whole(fails, monkeypatch):
    """Where there is no memory for a longer list, entries and their records stay as long as each other."""
    p = PagedKV(2, 4, device="cpu", exc_cap=16)
    zeros = torch.zeros

    def full(*a, **kw):
        if kw.get("dtype") is fails:
            raise torch.OutOfMemoryError("no room")
        return zeros(*a, **kw)
    monkeypatch.setattr(torch, "zeros", full)
    with pytest.raises(torch.OutOfMemoryError):
        p.pool._grow_exc(40, 16)
    assert p.struct().r.exc_cap == p.exc_cap == 16 and p.pool.rec.numel() == 16


def test_a_pool_keeps_its_size_and_its_blocks():
    """What the resident form behind a pool would do without the pages' rooms (their array is as
    long as the pool, and a moved block would write over another's entries)."""
    p = PagedKV(4, 8, device="cpu")
    p.pool.reserve(8 * 16)
    with pytest.raises(ValueError, match="keeps its size"):
        p.pool.reserve(9 * 16)
    assert p.struct().r.cap_blocks == 8 and p.pool.room.numel() == 32
    for move in (lambda: p.pool.reorder(torch.tensor([1, 0])),
                 lambda: reorder_sequences([p.pool], torch.tensor([1, 0]), 16)):
        with pytest.raises(ValueError, match="keep their places"):
            move()


def test_eviction_of_more_sequences_than_a_grid_has():
    """2^32 threads of 1024 a sequence."""
    lib = L.load()
    for n in (2 ** 22, 2 ** 31 - 1):
        assert lib.lq_evict_pages(16, 16, 16, n, 4, 2, 1, 1, 16, 16, 16, 16, None) == L.LQ_ERR_ARG
    n = 2 ** 22
    with pytest.raises(ValueError, match="fewer than 2\\^22"):
        evict_pages(torch.zeros(1, 2, dtype=torch.int32).expand(n, 2), torch.zeros(1, dtype=torch.int32).expand(n),
                    torch.zeros(1, 2).expand(n, 2), 1)


def test_nothing_that_wants_a_gradient_is_written_or_passed_by():
    a = _args()
    for name, t in (("weights", torch.zeros(2, 3)), ("tail_v", a["tail_v"].clone()), ("out", torch.zeros(2, 8, 1, 128).half())):
        with pytest.raises(RuntimeError, match="no gradient"):
            paged_decode_attention(**{**_args(), name: t.requires_grad_()})
    p, x, at = PagedKV(2, 4, device="cpu"), torch.zeros(1, 2, 16, 128), torch.tensor([[0]])
    for s32, s16 in ((torch.ones(2, requires_grad=True), torch.ones(2)), (torch.ones(2), torch.ones(2, requires_grad=True))):
        with pytest.raises(RuntimeError, match="no gradient"):
            p.write(x, at, s32, s16)
    with pytest.raises(RuntimeError, match="no gradient"):
        evict_pages(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, requires_grad=True), 1)


def test_rows_of_out_are_apart():
    """Against a count of every element's place, over strides that rows share elements by and that they do not."""
    for B in (1, 2, 3):
        for Hq in (1, 2, 4):
            for sb in (0, 64, 120, 128, 136, 256, 504, 512, 640):
                for sh in (0, 8, 128, 136, 256, 384, 1536):
                    out = torch.zeros(8000).as_strided((B, Hq, 1, 128), (sb, sh, 128, 1))
                    places = torch.arange(8000).as_strided((B, Hq, 1, 128), (sb, sh, 128, 1))
                    alone = places.unique().numel() == places.numel()
                    # (rows that lie between each other's are refused with those that overlap)
                    assert alone or not _apart(out), (B, Hq, sb, sh)
                    if _apart(out) != alone:
                        assert B > 1 and Hq > 1 and min(sb, sh) >= 128, (B, Hq, sb, sh)
    with pytest.raises(ValueError, match="out must be"):
        paged_decode_attention(**{**_args(), "out": torch.zeros(6000).half().as_strided((2, 8, 1, 128), (512, 64, 128, 1))})
