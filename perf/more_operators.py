"""Operators for serving many sequences over one pool of compressed KV pages.

A case is a dict of plain values.  `kind` names the operator:

  attend    paged_decode_attention: one new token of each sequence attends to its pages
            of the pool and to its fp16 / bf16 tail; with `weights` also the softmax weight
            that each page received
  evict     evict_pages: each sequence keeps the pages of most accumulated weight
  logprobs  token_logprobs: log probabilities of given tokens, entropies, top alternatives

With `own` false, run() computes them in elementary torch operations on fp16 rows.
"""
import math
import random

import numpy as np
import torch

own = False

HD = 128
PAGE = 16                                                # tokens of a page
PAGE_BYTES = 1024 + 256 + 32 + 16 + 32                   # of one kv head, K or V
_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the smallest step: one sequence a page into its answer (latency)
        {"name": "attend_token", "kind": "attend", "batch": 1, "heads": 8, "group": 4, "tokens": 500, "ragged": False,
         "dtype": "fp16", "weights": False},
        # an ordinary serving batch of a bf16 model, every length from a few tokens to 2048
        {"name": "attend_batch", "kind": "attend", "batch": 32, "heads": 8, "group": 4, "tokens": 2048, "ragged": True,
         "dtype": "bf16", "weights": False},
        # odd counts: seven sequences, groups of seven query heads, page weights wanted
        {"name": "attend_odd_weights", "kind": "attend", "batch": 7, "heads": 4, "group": 7, "tokens": 9001,
         "ragged": True, "dtype": "fp16", "weights": True},
        # two long documents
        {"name": "attend_long", "kind": "attend", "batch": 2, "heads": 8, "group": 4, "tokens": 131072, "ragged": False,
         "dtype": "fp16", "weights": False},
        # a full server that also keeps account of its pages, 64 sequences up to 8192 tokens
        {"name": "attend_full_weights", "kind": "attend", "batch": 64, "heads": 8, "group": 4, "tokens": 8192,
         "ragged": True, "dtype": "bf16", "weights": True},
        # one sequence of 16384 tokens drops a third of its pages (latency)
        {"name": "evict_one", "kind": "evict", "batch": 1, "pages": 1024, "keep": 683, "sink": 1, "recent": 8},
        # all sequences of a batch down to a budget that some are below
        {"name": "evict_batch", "kind": "evict", "batch": 64, "pages": 2048, "keep": 700, "sink": 4, "recent": 32},
        # four sequences of a million tokens
        {"name": "evict_long", "kind": "evict", "batch": 4, "pages": 65536, "keep": 16384, "sink": 4, "recent": 64},
        # the sampled token of one sequence with five alternatives (latency)
        {"name": "logprobs_token", "kind": "logprobs", "rows": 1, "vocab": 32000, "pad": 0, "top": 5, "dtype": "bf16"},
        # an odd vocabulary of a padded output layer, fp32 logits
        {"name": "logprobs_odd", "kind": "logprobs", "rows": 37, "vocab": 50021, "pad": 27, "top": 3, "dtype": "fp32"},
        # a serving batch with twenty alternatives, the vocabulary of the repository's model benchmark
        {"name": "logprobs_batch", "kind": "logprobs", "rows": 256, "vocab": 128256, "pad": 0, "top": 20,
         "dtype": "bf16"},
        # evaluation: the log likelihood of 2048 tokens of a text
        {"name": "logprobs_text", "kind": "logprobs", "rows": 2048, "vocab": 128256, "pad": 0, "top": 0,
         "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "evict", "logprobs", "logprobs"])
    if kind == "attend":
        batch, heads, group = _log(rng, 1, 64), rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 4, 7, 8, 16])
        most = min(131072, 2 * 8 * 131072 // (batch * heads), 2 * 8 * 4 * 131072 // (batch * heads * group))
        return {"kind": kind, "batch": batch, "heads": heads, "group": group, "tokens": _log(rng, 1, most),
                "ragged": batch > 1 and rng.random() < 0.7, "dtype": rng.choice(["fp16", "bf16"]),
                "weights": rng.random() < 0.5}
    if kind == "evict":
        batch = _log(rng, 1, 64)
        pages = _log(rng, 1, 4 * 65536 // batch if batch > 4 else 65536)
        sink, recent = rng.randint(0, 4), rng.randint(0, 64)
        return {"kind": kind, "batch": batch, "pages": pages, "sink": sink, "recent": recent,
                "keep": sink + recent + rng.randint(0, pages)}
    top = rng.choice([0, 0, 1, 5, 20, 64])
    vocab = _log(rng, 500, 128256)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    rows = 2048 if top == 0 else 256
    rows = max(1, min(rows, rows * 128256 // (vocab * (2 if dtype == "fp32" else 1))))
    return {"kind": kind, "rows": _log(rng, 1, rows), "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 63)]),
            "top": top, "dtype": dtype}


# ------------------------------------------------------------------ inputs --

def _gen(seed, k=0):
    return torch.Generator(device="cuda").manual_seed(seed * 16 + k)


def _rand(shape, seed, k, dtype, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed, k), device="cuda") * scale).to(dtype)


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _d8(x):
    r = x.round()
    e = x - r
    j = e.abs().argmax(-1, keepdim=True)
    step = torch.where(e.gather(-1, j) < 0, -1.0, 1.0)
    return r.scatter_add(-1, j, step * (r.sum(-1) % 2)[..., None])


def _e8(x):
    a, b = _d8(x), _d8(x - 0.5) + 0.5
    near = (x - a).square().sum(-1) <= (x - b).square().sum(-1)
    return torch.where(near[..., None], a, b)


def _lens(case):
    """Cached tokens of each sequence, the new one among them: (pages, tail tokens).
    A page is written once sixteen tokens stand before the newest."""
    rng, n = random.Random(case["batch"] * 1000003 + case["tokens"]), case["tokens"]
    t = [n] + [rng.randint(1, n) if case["ragged"] else n for _ in range(case["batch"] - 1)]
    return [(x - 1) // PAGE for x in t], [(x - 1) % PAGE + 1 for x in t]


def _pool(case, seed, k, n):
    """Rows (pages, heads, 16, 128) that n pages of a 4-bit pool hold (lattice points
    times an fp16 scale per page and head, a few outlier channels in K as rotary keys
    show them), and the scales."""
    h, g = case["heads"], _gen(seed, k)
    s = (0.2 + 0.1 * torch.rand(n, h, 1, 1, generator=g, device="cuda")).half().float()
    loud = torch.rand(h, 1, HD, generator=g, device="cuda").argsort(-1) < (2 if k == 0 else 0)
    loud = torch.where(loud, 5.0, 1.0)
    out = torch.empty(n, h, PAGE, HD, dtype=torch.float16, device="cuda")
    for i in range(0, n, 2048):                          # few fp32 copies at a time
        x = torch.randn(out[i:i + 2048].shape, generator=g, device="cuda") * loud
        x = _e8((x / s[i:i + 2048]).reshape(-1, 8)).reshape(x.shape)
        out[i:i + 2048] = (x * s[i:i + 2048]).half()
    return out, s.reshape(n, h)


def _prepare_attend(case, seed):
    b, h, dt = case["batch"], case["heads"], _DT[case["dtype"]]
    count, tail = _lens(case)
    width, total = max(1, max(count)), sum(count)
    n = total + 1 + total // 16                          # some pages of the pool are free
    order = torch.rand(n, generator=_gen(seed, 8), device="cuda").argsort().to(torch.int32)
    pages = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(count):
        pages[i, :c] = order[at:at + c]
        at += c
    st = {"case": case, "q": _rand((b, h * case["group"], 1, HD), seed, 2, dt), "pages": pages, "count": _int32(count),
          "tail": _int32(tail), "tail_k": _rand((b, h, PAGE, HD), seed, 4, dt),
          "tail_v": _rand((b, h, PAGE, HD), seed, 5, dt), "weights": None}
    if case["weights"]:
        st["weights"] = torch.rand(b, width, generator=_gen(seed, 6), device="cuda")
    for i, kv in enumerate("kv"):
        rows, s = _pool(case, seed, i, n)
        if own:                                          # the plan: the pool and a workspace
            from latticequant_amd.llm.paged import PagedKV
            p = PagedKV(h, n, device="cuda")
            for j in range(0, n, 4096):
                p.write(rows[j:j + 4096], torch.arange(j, min(j + 4096, n), device="cuda")[:, None], s[j:j + 4096],
                        s[j:j + 4096].half())
            st["pool_" + kv] = p
        else:
            st["rows_" + kv] = rows
    if own:
        from latticequant_amd.llm.paged import paged_attn_workspace
        st["work"] = paged_attn_workspace(b, h, case["group"], width, PAGE, weights=case["weights"], device="cuda")
    return st


def _prepare_evict(case, seed):
    b, w, g = case["batch"], case["pages"], _gen(seed)
    rng = random.Random(b * 1000003 + w)
    count = [w] + [rng.randint(0, w) for _ in range(b - 1)]
    pages = torch.rand(b * w, generator=g, device="cuda").argsort().to(torch.int32).reshape(b, w)
    # accumulated weights: a few pages take most, many next to nothing, some have seen no query yet
    weight = torch.randn(b, w, generator=g, device="cuda").mul_(2.0).exp_()
    weight = torch.where(torch.rand(b, w, generator=g, device="cuda") < 0.05, 0.0, weight)
    return {"case": case, "pages": pages, "count": _int32(count), "weights": weight}


def _prepare_logprobs(case, seed):
    n, v = case["rows"], case["vocab"]
    x = _rand((n, v + case["pad"]), seed, 0, _DT[case["dtype"]], 2.5)[:, :v]
    g = _gen(seed, 1)
    tokens = torch.randint(0, v, (n,), generator=g, device="cuda")
    sure = torch.rand(n, generator=g, device="cuda") < 0.7            # most tokens of a text are expected
    x[sure.nonzero()[:, 0], tokens[sure]] = 14.0
    return {"case": case, "logits": x, "tokens": tokens}


def prepare(case, seed):
    return {"attend": _prepare_attend, "evict": _prepare_evict, "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


# -------------------------------------------------------------------- pass --

def _attend(st):
    case, pages = st["case"], st["pages"].long()
    b, h, g = case["batch"], case["heads"], case["group"]
    count, tail, weights = st["count"], st["tail"], st["weights"]
    out = torch.empty_like(st["q"])
    width = pages.shape[1]
    step = max(1, 8 * 131072 // (h * width * PAGE))      # sequences at a time: fp32 copies of a gigabyte or two
    for lo in range(0, b, step):
        i = slice(lo, lo + step)
        m = pages[i].shape[0]
        at = pages[i].clamp_min(0)
        k, v = (torch.cat([st["rows_" + kv][at].transpose(1, 2).reshape(m, h, width * PAGE, HD).to(torch.float32),
                           st["tail_" + kv][i].float()], 2) for kv in "kv")
        t = torch.arange(PAGE, device="cuda")
        sees = torch.cat([(torch.arange(width, device="cuda") < count[i, None]).repeat_interleave(PAGE, 1),
                          t < tail[i, None]], 1)[:, None, None]
        s = torch.matmul(st["q"][i].float().reshape(m, h, g, HD), k.transpose(2, 3).contiguous()) / math.sqrt(HD)
        s = s.masked_fill_(~sees, -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp_()
        p = p / p.sum(-1, keepdim=True)
        out[i] = torch.matmul(p, v).reshape(m, h * g, 1, HD).to(out.dtype)
        if weights is not None:
            w = p[..., :width * PAGE].reshape(m, h * g, width, PAGE).sum((1, 3))
            weights[i] = torch.where(torch.arange(width, device="cuda") < count[i, None], w, weights[i])
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _evict(st):
    case, n = st["case"], st["count"].long()[:, None]
    j = torch.arange(case["pages"], device="cuda")[None]
    on = j < n
    first = torch.where((j < case["sink"]) | (j >= n - case["recent"]), 2, 1) * on    # always kept, others, none
    order = (-st["weights"]).sort(dim=1, stable=True).indices
    order = order.gather(1, (-first.gather(1, order)).sort(dim=1, stable=True).indices)
    rank = torch.empty_like(order).scatter_(1, order, j.expand_as(order))
    kept = on & (rank < case["keep"])

    def packed(mask, values, empty):
        at = mask.cumsum(1) - 1
        out = torch.full_like(values, empty)
        row = torch.arange(values.shape[0], device="cuda")[:, None].expand_as(values)
        out[row[mask], at[mask]] = values[mask]
        return out
    return {"pages": packed(kept, st["pages"], -1), "count": kept.sum(1).to(torch.int32),
            "weights": packed(kept, st["weights"], 0.0), "freed": packed(on & ~kept, st["pages"], -1)}


def _logprobs(st):
    n, k = st["logits"].shape[0], st["case"]["top"]
    got = {"logprob": [], "entropy": [], "ids": [], "top": []}
    for lo in range(0, n, 256):                          # a few rows at a time in 32 bits
        x = st["logits"][lo:lo + 256].float()
        x = x - x.amax(1, keepdim=True)
        p = x.exp()
        s = p.sum(1, keepdim=True)
        lse = s.log()
        got["logprob"].append(x.gather(1, st["tokens"][lo:lo + 256, None])[:, 0] - lse[:, 0])
        got["entropy"].append(lse[:, 0] - (p * x).sum(1) / s[:, 0])
        if k:
            v, at = x.sort(dim=1, descending=True, stable=True)
            got["ids"].append(at[:, :k])
            got["top"].append(v[:, :k] - lse)
    return {name: torch.cat(v) for name, v in got.items() if v}


def run(state):
    st, case = state, state["case"]
    if not own:
        return {"attend": _attend, "evict": _evict, "logprobs": _logprobs}[case["kind"]](st)
    if case["kind"] == "attend":
        from latticequant_amd.llm.paged import paged_decode_attention
        out = paged_decode_attention(st["pool_k"], st["pool_v"], st["q"], st["pages"], st["count"], st["tail_k"],
                                     st["tail_v"], tail_len=st["tail"], weights=st["weights"], decay=0.0,
                                     work=st["work"])
        return {"out": out} if st["weights"] is None else {"out": out, "weights": st["weights"]}
    if case["kind"] == "evict":
        from latticequant_amd.llm.paged import evict_pages
        r = evict_pages(st["pages"], st["count"], st["weights"], case["keep"], sink=case["sink"], recent=case["recent"])
        return {"pages": r.pages, "count": r.n_pages, "weights": r.weights, "freed": r.freed}
    from latticequant_amd.llm.logprobs import token_logprobs
    r = token_logprobs(st["logits"], st["tokens"], top=case["top"])
    out = {"logprob": r.logprob, "entropy": r.entropy}
    return {**out, "ids": r.top_ids, "top": r.top_logprobs} if case["top"] else out


# ------------------------------------------------------------------- floor --

def work(case):
    if case["kind"] == "attend":
        b, h, g = case["batch"], case["heads"], case["group"]
        count, tail = _lens(case)
        pages, rows = sum(count), sum(tail)
        n = 2 * h * (pages * PAGE_BYTES + rows * HD * 2) + 2 * b * h * g * HD * 2 + 4 * pages
        return {"bytes": n + (4 * pages if case["weights"] else 0),
                "flops": 4 * h * g * HD * (pages * PAGE + rows)}
    if case["kind"] == "evict":
        rng = random.Random(case["batch"] * 1000003 + case["pages"])
        n = [case["pages"]] + [rng.randint(0, case["pages"]) for _ in range(case["batch"] - 1)]
        return {"bytes": 8 * sum(n) + 12 * case["batch"] * case["pages"], "flops": 0}
    el = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    n = case["rows"] * case["vocab"]
    return {"bytes": n * el + case["rows"] * (16 + 12 * case["top"]), "flops": 4 * n}


# ------------------------------------------------------- 64-bit reference --

def _exact_attend(case, seed):
    global own
    was, own = own, False
    try:
        st = _prepare_attend(case, seed)
    finally:
        own = was
    count, tail = _lens(case)
    h, g = case["heads"], case["group"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    weights = None if st["weights"] is None else st["weights"].double()
    for b, (c, t) in enumerate(zip(count, tail)):
        at = st["pages"][b, :c].long()
        for j in range(h):
            k, v = (torch.cat([st["rows_" + kv][at, j].reshape(-1, HD), st["tail_" + kv][b, j, :t]]).double()
                    for kv in "kv")
            p = torch.softmax(k @ st["q"][b, g * j:g * j + g, 0].double().t().contiguous() * HD ** -0.5, 0)
            out[b, g * j:g * j + g, 0] = p.t().contiguous() @ v
            if weights is not None and c:
                w = p[:c * PAGE].sum(1).reshape(c, PAGE).sum(1)
                weights[b, :c] = w if j == 0 else weights[b, :c] + w
    return {"out": out} if weights is None else {"out": out, "weights": weights}


def _exact_evict(case, seed):
    st = _prepare_evict(case, seed)
    pages, count, weight = (st[k].cpu().numpy() for k in ("pages", "count", "weights"))
    out = {"pages": np.full_like(pages, -1), "count": np.zeros_like(count), "weights": np.zeros(weight.shape),
           "freed": np.full_like(pages, -1)}
    for b, n in enumerate(count):
        lo, hi = min(case["sink"], n), max(min(case["sink"], n), n - case["recent"])
        room = max(0, case["keep"] - lo - (n - hi))
        best = lo + np.lexsort((np.arange(hi - lo), -weight[b, lo:hi].astype(np.float64)))[:room]
        keep = np.sort(np.concatenate([np.arange(lo), best, np.arange(hi, n)])).astype(np.int64)
        gone = np.setdiff1d(np.arange(n), keep)
        out["count"][b] = len(keep)
        out["pages"][b, :len(keep)], out["weights"][b, :len(keep)] = pages[b, keep], weight[b, keep]
        out["freed"][b, :len(gone)] = pages[b, gone]
    return out


def _exact_logprobs(case, seed):
    st = _prepare_logprobs(case, seed)
    n, k = case["rows"], case["top"]
    logprob, entropy, top = [], [], []
    for i in range(0, n, 64):
        lp = torch.log_softmax(st["logits"][i:i + 64].double(), 1)
        logprob.append(lp[torch.arange(lp.shape[0], device="cuda"), st["tokens"][i:i + 64]])
        entropy.append(-(lp.exp() * lp).sum(1))
        if k:
            top.append(lp.topk(k, 1).values)
    out = {"logprob": torch.cat(logprob), "entropy": torch.cat(entropy)}
    return {**out, "ids": None, "top": torch.cat(top)} if k else out


def exact(case, seed):
    return {"attend": _exact_attend, "evict": _exact_evict, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
