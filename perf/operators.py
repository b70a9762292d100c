"""Operators for decoding along several continuations over a compressed KV cache.

A case is a dict of plain values.  `kind` names the operator:

  tree      resident_tree_attention: the drafted tokens of a tree (or chain) attend
            to the resident prefix, the fp16 tail and their own ancestors
  accept    accept_drafts: argmax of every node's logits, then the walk from node 0
            along the children whose token was chosen
  append    append_accepted: the accepted drafts' K / V rows of all layers behind
            their sequences' tails
  reorder   reorder_sequences: the sequences of a resident cache permuted in place
            (beams), K and V of all layers
  select    ResidentKV.select: a new resident prefix of chosen sequences and blocks
            (fork, eviction), its exception list rebuilt

With `own` false, run() computes them in elementary torch operations on fp16 rows
and integer planes.
"""
import math
import random

import numpy as np
import torch

own = False

HD = 128
RB = 16                                                  # tokens of a resident block
PLANES = ("a", "b", "mask", "meta", "scale")
_PLANE = {"a": (256, torch.int32), "b": (256, torch.uint8), "mask": (4, torch.int64), "meta": (4, torch.int32),
          "scale": (16, torch.float16)}                  # elements of a block in each plane
BLOCK_BYTES = 1024 + 256 + 32 + 16 + 32
_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the smallest step: one token over a short prompt (single-token decoding through the tree path; latency)
        {"name": "tree_token", "kind": "tree", "batch": 1, "heads": 8, "group": 4, "nodes": 1, "tokens": 1024,
         "tail": 37, "dtype": "fp16", "shape": "chain", "start": False},
        # four sequences of different lengths (left-padded, ragged tails), a drafted chain of five, bf16 model
        {"name": "tree_chain_batch", "kind": "tree", "batch": 4, "heads": 8, "group": 4, "nodes": 5, "tokens": 4096,
         "tail": 143, "dtype": "bf16", "shape": "chain", "start": True},
        # an ordinary draft tree, odd node count, group 7
        {"name": "tree_odd", "kind": "tree", "batch": 1, "heads": 4, "group": 7, "nodes": 27, "tokens": 8208,
         "tail": 101, "dtype": "fp16", "shape": "tree", "start": False},
        # a wide tree over a 32k prefix
        {"name": "tree_long", "kind": "tree", "batch": 1, "heads": 8, "group": 4, "nodes": 64, "tokens": 32768,
         "tail": 128, "dtype": "fp16", "shape": "tree", "start": False},
        # acceptance of a short chain of one sequence
        {"name": "accept_chain", "kind": "accept", "batch": 1, "nodes": 5, "vocab": 32000, "dtype": "bf16"},
        # acceptance of eight wide trees, the vocabulary of the repository's model benchmark
        {"name": "accept_trees", "kind": "accept", "batch": 8, "nodes": 64, "vocab": 128256, "dtype": "bf16"},
        # accepted rows of one sequence, 32 layers (latency)
        {"name": "append_one", "kind": "append", "layers": 32, "batch": 1, "heads": 8, "nodes": 5, "tail": 143,
         "dtype": "fp16"},
        # accepted rows of sixteen sequences, 32 layers
        {"name": "append_batch", "kind": "append", "layers": 32, "batch": 16, "heads": 8, "nodes": 27, "tail": 160,
         "dtype": "bf16"},
        # four beams that share their prompt: only the 80 generated tokens move, 28 layers
        {"name": "reorder_beams", "kind": "reorder", "layers": 28, "batch": 4, "heads": 4, "tokens": 1104,
         "from": 1024},
        # eight beams' whole prefixes, 32 layers
        {"name": "reorder_whole", "kind": "reorder", "layers": 32, "batch": 8, "heads": 8, "tokens": 2048, "from": 0},
        # a prompt forked into four sequences
        {"name": "select_fork", "kind": "select", "batch": 1, "heads": 8, "tokens": 8192, "out": 4, "keep": 1.0},
        # eviction: four long sequences keep two thirds of their blocks, each its own
        {"name": "select_evict", "kind": "select", "batch": 4, "heads": 8, "tokens": 32768, "out": 4, "keep": 0.66},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "accept", "append", "reorder", "select"])
    heads = rng.choice([1, 2, 4, 8, 8])
    if kind == "tree":
        batch, group, nodes = rng.choice([1, 1, 2, 4]), rng.choice([1, 2, 4, 4, 7, 8]), _log(rng, 1, 100)
        tokens = RB * _log(rng, 1, 2048)
        most = min(8 * 32768 // (batch * heads), 8 * 256 * 32768 // (batch * heads * group * nodes))
        return {"kind": kind, "batch": batch, "heads": heads, "group": group, "nodes": nodes,
                "tokens": max(RB, min(tokens, most) // RB * RB), "tail": rng.randint(0, 200),
                "dtype": rng.choice(["fp16", "bf16"]), "shape": rng.choice(["chain", "tree", "tree"]),
                "start": batch > 1 and rng.random() < 0.5}
    if kind == "accept":
        batch, nodes, vocab = _log(rng, 1, 16), _log(rng, 1, 100), _log(rng, 500, 128256)
        nodes = max(1, min(nodes, 8 * 64 * 128256 // (2 * batch * vocab)))
        return {"kind": kind, "batch": batch, "nodes": nodes, "vocab": vocab,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "append":
        return {"kind": kind, "layers": rng.randint(1, 32), "batch": _log(rng, 1, 16), "heads": heads,
                "nodes": _log(rng, 1, 64), "tail": rng.randint(64, 200), "dtype": rng.choice(["fp16", "bf16"])}
    if kind == "reorder":
        tokens = RB * _log(rng, 4, 128)
        return {"kind": kind, "layers": rng.randint(1, 32), "batch": rng.randint(2, 8), "heads": heads,
                "tokens": tokens, "from": rng.choice([0, tokens // 32 * RB, tokens - 2 * RB])}
    out = rng.randint(1, 4)
    return {"kind": "select", "batch": rng.randint(1, 4), "heads": heads, "tokens": RB * _log(rng, 8, 2048), "out": out,
            "keep": rng.choice([1.0, round(rng.uniform(0.2, 0.95), 3)])}


# ------------------------------------------------------------------ inputs --

def _gen(seed, k=0):
    return torch.Generator(device="cuda").manual_seed(seed * 16 + k)


def _rand(shape, seed, k, dtype, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed, k), device="cuda") * scale).to(dtype)


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


def _prefix(case, seed, k):
    """Rows (batch, heads, tokens, 128) that a 4-bit resident prefix holds (lattice
    points times an fp16 scale per head, a few outlier channels as rotary keys show
    them), and the scales."""
    b, h, t = case["batch"], case["heads"], case["tokens"]
    g = _gen(seed, k)
    s = (0.2 + 0.1 * torch.rand(b, h, 1, 1, generator=g, device="cuda")).half().float()
    loud = torch.rand(b, h, 1, HD, generator=g, device="cuda").argsort(-1) < (2 if k == 0 else 0)
    out = torch.empty(b, h, t, HD, dtype=torch.float16, device="cuda")
    for i in range(b):                                   # sequence by sequence: few fp32 copies at a time
        x = torch.randn(h, t, HD, generator=g, device="cuda") * torch.where(loud[i], 5.0, 1.0)
        out[i] = (_e8((x / s[i]).reshape(-1, 8)).reshape(h, t, HD) * s[i]).half()
    return out, s.reshape(-1)


def _parents(case, seed):
    """Drafted trees: node 0 is the newest token, every other node's parent stands
    before it; of several sequences the later ones draft fewer nodes (padding: -2)."""
    rng, b, n = random.Random(seed), case["batch"], case["nodes"]
    rows = []
    for i in range(b):
        m = n if i == 0 else rng.randint(1, n)
        row = [-1] + [j - 1 if case.get("shape") == "chain" else max(0, j - 1 - int(rng.expovariate(0.2)))
                      for j in range(1, m)]
        rows.append(row + [-2] * (n - m))
    return rows


def _lengths(case, seed):
    """Valid tail tokens and first visible token (left padding) of each sequence."""
    rng, b = random.Random(seed + 1), case["batch"]
    lens = [case["tail"]] + [rng.randint(0, case["tail"]) for _ in range(b - 1)]
    start = [0] + [rng.randint(0, case["tokens"] // 2) for _ in range(b - 1)]
    return lens, start if case["start"] else [0] * b


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_tree(case, seed):
    b, h, n, dt = case["batch"], case["heads"], case["nodes"], _DT[case["dtype"]]
    lens, start = _lengths(case, seed)
    st = {"case": case, "q": _rand((b, n, h * case["group"], HD), seed, 2, dt).transpose(1, 2),
          "parents": _int32(_parents(case, seed)), "len": _int32(lens), "start": _int32(start) if case["start"] else None}
    for i, kv in enumerate("kv"):
        rows, s = _prefix(case, seed, i)
        st["tail_" + kv] = _rand((b, h, case["tail"], HD), seed, 4 + i, dt)
        st["draft_" + kv] = _rand((b, n, h, HD), seed, 6 + i, dt).transpose(1, 2)
        if own:                                          # the plan: the prefix in its resident form
            from latticequant_amd.llm.resident import ResidentKV
            r = ResidentKV(b * h, case["tokens"], device="cuda")
            r.append(rows, s, s.half())
            st["res_" + kv] = r
        else:
            st["rows_" + kv] = rows
    if own:
        from latticequant_amd.llm.tree import tree_attn_workspace
        st["work"] = tree_attn_workspace(b * h, case["group"], n, case["tokens"], case["tail"], device="cuda")
    return st


def _prepare_accept(case, seed):
    b, n, v = case["batch"], case["nodes"], case["vocab"]
    par = _parents(dict(case, shape="tree"), seed)
    rng = random.Random(seed + 2)
    tokens = [[rng.randrange(v) for _ in range(n)] for _ in range(b)]
    logits = _rand((b, n, v), seed, 0, _DT[case["dtype"]], 2.0)
    at = [(i, p, tokens[i][j]) for i in range(b) for j, p in enumerate(par[i]) if p >= 0 and rng.random() < 0.6]
    if at:                                               # the target agrees with some of the drafts
        i, p, t = (torch.tensor(x, device="cuda") for x in zip(*at))
        logits[i, p, t] = 24.0                           # two agreed children of one node tie
    return {"case": case, "tokens": torch.tensor(tokens, device="cuda"), "parents": _int32(par), "logits": logits}


def _prepare_append(case, seed):
    b, h, n, cap = case["batch"], case["heads"], case["nodes"], case["tail"]
    rng, dt = random.Random(seed), _DT[case["dtype"]]
    count = [rng.randint(1, min(n, 8)) for _ in range(b)]
    path = [sorted(rng.sample(range(n), c)) + [-1] * (n - c) for c in count]
    lens = [rng.randint(0, cap - n) for _ in range(b)]
    tails = _rand((2 * case["layers"], b, h, cap, HD), seed, 0, dt)
    drafts = _rand((2 * case["layers"], b, n, h, HD), seed, 1, dt).transpose(2, 3)
    st = {"case": case, "tails": tails, "drafts": drafts, "path": _int32(path), "count": _int32(count),
          "len": _int32(lens)}
    if own:                                              # a cache's own lists: K and V of every layer
        st["lists"] = list(tails.unbind(0)), list(drafts.unbind(0))
    return st


def _blocks(lead, case, seed):
    """Planes (lead.., batch, heads, blocks, elements) as a resident prefix holds them:
    words, and masks with their exception counts and list offsets."""
    shape = tuple(lead) + (case["batch"], case["heads"], case["tokens"] // RB)
    g = _gen(seed)
    pl = {}
    for p in ("a", "b"):
        w, dt = _PLANE[p]
        hi = 1 << (31 if p == "a" else 8)
        pl[p] = torch.randint(0, hi, shape + (w,), generator=g, device="cuda", dtype=dt)
    pl["scale"] = (0.2 + 0.1 * torch.rand(shape + (16,), generator=g, device="cuda")).half()
    bit = torch.randint(0, 63, shape + (4,), generator=g, device="cuda")
    at = torch.arange(shape[-1] * 4, device="cuda").reshape(-1, 4)
    some = ((at * 40503 >> 4) % 10 == 0).expand(bit.shape)   # as many exceptions whatever the seed: outputs of one size
    pl["mask"] = torch.where(some, torch.ones_like(bit) << bit, 0)
    count = some.sum(-1).to(torch.int32).reshape(tuple(lead) + (-1,))
    base = (count.cumsum(-1) - count).to(torch.int32)
    meta = torch.randint(0, 1 << 30, shape + (4,), generator=g, device="cuda", dtype=torch.int32)
    meta[..., 2], meta[..., 3] = base.reshape(shape), count.reshape(shape)
    pl["meta"] = meta
    return pl, count.sum(-1)


def _resident(case, planes, exc=None):
    """A ResidentKV whose planes are these tensors (layers allocated together)."""
    from latticequant_amd.llm.resident import ResidentKV
    r = ResidentKV(case["batch"] * case["heads"], case["tokens"], device="cuda", n_seq=case["batch"])
    for p, t in planes.items():
        setattr(r, p, t.reshape(-1))
    if exc is not None:
        r.exc = exc.reshape(-1)
        r.n_exc.fill_(exc.shape[0])
    r.n_tokens = case["tokens"]
    return r


def _index(case, seed, n):
    """The sequence that each output continues: some continue twice, some end."""
    rng = random.Random(seed + 3)
    return [rng.randrange(case["batch"]) for _ in range(n)]


def _kept(case):
    """Kept blocks of every output sequence, in order; None for all of them (as
    many exceptions in them whatever the seed)."""
    nb = case["tokens"] // RB
    if case["keep"] >= 1.0:
        return None
    n = max(1, int(nb * case["keep"]))
    g = _gen(n, 9)
    return torch.rand(case["out"], nb, generator=g, device="cuda").argsort(-1)[:, :n].sort(-1).values.to(torch.int32)


def prepare(case, seed):
    kind = case["kind"]
    if kind == "tree":
        return _prepare_tree(case, seed)
    if kind == "accept":
        return _prepare_accept(case, seed)
    if kind == "append":
        return _prepare_append(case, seed)
    if kind == "reorder":
        n = 2 * case["layers"]
        pl, _ = _blocks((n,), case, seed)
        st = {"case": case, "planes": pl, "index": _int32(_index(case, seed, case["batch"]))}
        if own:
            st["res"] = [_resident(case, {p: t[i] for p, t in pl.items()}) for i in range(n)]
        return st
    pairs = []
    for k in range(2):                                   # K and V of a layer
        pl, total = _blocks((), case, seed + k)
        exc = torch.randint(-600, 600, (max(1, int(total)), 8), generator=_gen(seed, 10 + k), device="cuda",
                            dtype=torch.int16)
        pairs.append((pl, exc))
    st = {"case": case, "pairs": pairs, "index": _int32(_index(case, seed, case["out"])), "blocks": _kept(case)}
    if own:
        st["res"] = [_resident(case, pl, exc) for pl, exc in pairs]
    return st


# -------------------------------------------------------------------- pass --

def _visible(parents):
    """(sees, valid): sees[b, i, j] where node j is i or an ancestor of it, valid
    nodes only (their chain of parents ends in a root, -1)."""
    n = parents.shape[1]
    idx = torch.arange(n, device=parents.device)
    has = (parents >= 0) & (parents < idx)
    up = (torch.where(has, parents, -1)[..., None] == idx).float()
    reach = up + torch.eye(n, device=parents.device)
    k = 1
    while k < n:                                         # closure by doubling
        reach = (torch.matmul(reach, reach) > 0).float()
        k *= 2
    valid = torch.matmul(reach, (parents == -1).float()[..., None])[..., 0] > 0
    return (reach > 0) & valid[..., None], valid


def _tree(st):
    case = st["case"]
    b, h, n, g, t = case["batch"], case["heads"], case["nodes"], case["group"], case["tokens"]
    sees, _ = _visible(st["parents"])
    pos = torch.arange(t + case["tail"], device="cuda")
    cache = pos[None] < t + st["len"][:, None]
    if st["start"] is not None:
        cache = cache & (pos[None] >= st["start"][:, None])
    valid = sees.any(-1)
    see = torch.cat([cache[:, None, :] & valid[..., None], sees], -1)          # (b, nodes, tokens)
    k = torch.cat([st["rows_k"], st["tail_k"], st["draft_k"]], 2).float()
    v = torch.cat([st["rows_v"], st["tail_v"], st["draft_v"]], 2).float()
    q = st["q"].float().reshape(b, h, g * n, HD)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(HD)
    s = s.reshape(b, h, g, n, -1).masked_fill_(~see[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - torch.where(m == -math.inf, 0.0, m)).exp_()
    o = torch.matmul(p.reshape(b, h, g * n, -1), v) / p.sum(-1).clamp_min(1e-30).reshape(b, h, g * n, 1)
    return o.reshape(b, h * g, n, HD).to(st["q"].dtype)


def _accept(st):
    choice = st["logits"].float().argmax(-1)
    par, tok = st["parents"].long(), st["tokens"]
    b, n = par.shape
    idx = torch.arange(n, device=par.device)
    path = torch.full((b, n), -1, dtype=torch.int32, device=par.device)
    cur = torch.zeros(b, dtype=torch.int64, device=par.device)
    live = torch.ones(b, dtype=torch.bool, device=par.device)
    count = torch.zeros(b, dtype=torch.int32, device=par.device)
    for j in range(n):
        path[:, j] = torch.where(live, cur, -1).to(torch.int32)
        count += live
        want = choice.gather(1, cur[:, None])
        hit = (par == cur[:, None]) & (tok == want) & (idx > cur[:, None]) & live[:, None]
        live = hit.any(1)
        cur = torch.where(live, torch.where(hit, idx, n).amin(1), cur)
    return {"path": path, "count": count, "next": choice.gather(1, cur[:, None])[:, 0]}


def _append(st):
    b, n = st["path"].shape
    j = torch.arange(n, device="cuda")
    on = j[None] < st["count"][:, None]
    bi = torch.arange(b, device="cuda")[:, None].expand(b, n)[on]
    at = (st["len"][:, None] + j)[on].long()
    src = st["path"][on].long()
    st["tails"][:, bi, :, at] = st["drafts"][:, bi, :, src]
    return {"tails": st["tails"], "len": st["len"] + st["count"]}


def _reorder(st):
    b0 = st["case"]["from"] // RB
    idx = st["index"].long()
    for p in PLANES:
        part = st["planes"][p][:, :, :, b0:]
        part.copy_(part[:, idx])
    return st["planes"]


def _select(st):
    idx, out = st["index"].long(), []
    for pl, exc in st["pairs"]:
        new = {}
        for p in PLANES:
            t = pl[p][idx]
            if st["blocks"] is not None:
                at = st["blocks"].long()[:, None, :, None].expand(-1, t.shape[1], -1, t.shape[3])
                t = t.gather(2, at)
            new[p] = t
        count = new["meta"][..., 3].reshape(-1).long()
        old = new["meta"][..., 2].reshape(-1).long()
        base = count.cumsum(0) - count
        which = torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count)
        src = old[which] + torch.arange(which.numel(), device="cuda") - base[which]
        new["meta"][..., 2] = base.reshape(new["meta"].shape[:-1]).to(torch.int32)
        out.append({**{p: t.reshape(-1) for p, t in new.items()}, "exc": exc[src].reshape(-1)})
    return out


def run(state):
    st, kind = state, state["case"]["kind"]
    if not own:
        return {"tree": _tree, "accept": _accept, "append": _append, "reorder": _reorder, "select": _select}[kind](st)
    if kind == "tree":
        from latticequant_amd.llm.tree import resident_tree_attention
        return resident_tree_attention(st["res_k"], st["res_v"], st["q"], st["draft_k"], st["draft_v"], st["parents"],
                                       st["tail_k"], st["tail_v"], tail_len=st["len"], start=st["start"],
                                       work=st["work"])
    if kind == "accept":
        from latticequant_amd.llm.tree import accept_drafts
        path, count, nxt = accept_drafts(st["tokens"], st["parents"], logits=st["logits"])
        return {"path": path, "count": count, "next": nxt}
    if kind == "append":
        from latticequant_amd.llm.tree import append_accepted
        tails, drafts = st["lists"]
        return {"tails": st["tails"], "len": append_accepted(tails, drafts, st["path"], st["count"], st["len"])}
    if kind == "reorder":
        from latticequant_amd.llm.resident import reorder_sequences
        reorder_sequences(st["res"], st["index"], t_from=st["case"]["from"])
        return st["planes"]
    out = []
    for r in st["res"]:
        n = r.select(st["index"], blocks=st["blocks"])
        out.append({**{p: getattr(n, p) for p in PLANES}, "exc": n.exceptions().reshape(-1)})
    return out


# ------------------------------------------------------------------- floor --

def work(case):
    kind = case["kind"]
    el = {"fp16": 2, "bf16": 2, "fp32": 4}.get(case.get("dtype"), 2)
    if kind == "tree":
        bh, n, t = case["batch"] * case["heads"], case["nodes"], case["tokens"]
        rows = bh * case["group"] * n
        return {"bytes": 2 * bh * (t // RB) * BLOCK_BYTES + 2 * bh * (case["tail"] + n) * HD * 2 + 2 * rows * HD * 2,
                "flops": 4 * rows * HD * (t + case["tail"] + (n + 1) // 2)}
    if kind == "accept":
        n = case["batch"] * case["nodes"]
        return {"bytes": n * case["vocab"] * el + 16 * n, "flops": n * case["vocab"]}
    if kind == "append":
        rows = 2 * case["layers"] * case["heads"] * case["batch"] * (min(case["nodes"], 8) + 1) / 2
        return {"bytes": 2 * rows * HD * el, "flops": 0}
    if kind == "reorder":
        moved = 1.0 - 1.0 / case["batch"]                # beams that change, on average
        n = 2 * case["layers"] * case["batch"] * case["heads"] * ((case["tokens"] - case["from"]) // RB)
        return {"bytes": 2 * moved * n * BLOCK_BYTES, "flops": 0}
    nb = case["tokens"] // RB
    n = 2 * case["out"] * case["heads"] * max(1, int(nb * case["keep"]))
    src = 2 * min(case["batch"], case["out"]) * case["heads"] * max(1, int(nb * case["keep"]))
    return {"bytes": (n + src) * (BLOCK_BYTES + 0.4 * 16), "flops": 0}


# ------------------------------------------------------- 64-bit reference --

def _exact_tree(case, seed):
    global own
    was, own = own, False
    try:
        st = _prepare_tree(case, seed)
    finally:
        own = was
    lens, start = _lengths(case, seed)
    h, g, t = case["heads"], case["group"], case["tokens"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for b, par in enumerate(_parents(case, seed)):
        rows = []
        for kv in "kv":
            past = torch.cat([st["rows_" + kv][b], st["tail_" + kv][b, :, :lens[b]]], 1)[:, start[b]:]
            rows.append(torch.cat([past, st["draft_" + kv][b]], 1).double())
        past = rows[0].shape[1] - case["nodes"]
        for lo in range(0, case["nodes"], 16):           # a few nodes at a time: the scores are 64-bit
            nodes = [i for i in range(lo, min(lo + 16, case["nodes"])) if par[i] >= -1]
            if not nodes:
                continue
            see = torch.zeros(len(nodes), rows[0].shape[1], dtype=torch.bool)
            see[:, :past] = True
            for r, i in enumerate(nodes):
                while i >= 0:
                    see[r, past + i] = True
                    i = par[i]
            qq = st["q"][b, :, nodes].double().reshape(h, g * len(nodes), HD)
            s = torch.matmul(qq, rows[0].transpose(1, 2).contiguous()) * HD ** -0.5
            s = s.reshape(h, g, len(nodes), -1).masked_fill(~see.cuda(), -math.inf)
            o = torch.matmul(torch.softmax(s, -1).reshape(h, g * len(nodes), -1), rows[1])
            out[b, :, nodes] = o.reshape(h * g, len(nodes), HD)
    return out


def _exact_accept(case, seed):
    st = _prepare_accept(case, seed)
    best = st["logits"].double()
    best = (best == best.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1).cpu().numpy()
    par, tok = st["parents"].cpu().numpy(), st["tokens"].cpu().numpy()
    b, n = par.shape
    path, count, nxt = np.full((b, n), -1, np.int32), np.zeros(b, np.int32), np.zeros(b, np.int64)
    for i in range(b):
        walk = [0]
        while True:
            c = best[i, walk[-1]]
            kids = [j for j in range(walk[-1] + 1, n) if par[i, j] == walk[-1] and tok[i, j] == c]
            if not kids:
                break
            walk.append(kids[0])
        path[i, :len(walk)], count[i], nxt[i] = walk, len(walk), best[i, walk[-1]]
    return {"path": path, "count": count, "next": nxt}


def exact(case, seed):
    kind = case["kind"]
    if kind == "tree":
        return _exact_tree(case, seed)
    if kind == "accept":
        return _exact_accept(case, seed)
    if kind == "append":
        st = _prepare_append(case, seed)
        tails = st["tails"].double()
        path, count, lens = (st[k].tolist() for k in ("path", "count", "len"))
        for b, c in enumerate(count):
            for j in range(c):
                tails[:, b, :, lens[b] + j] = st["drafts"][:, b, :, path[b][j]].double()
        return {"tails": tails, "len": np.array([x + c for x, c in zip(lens, count)], np.int32)}
    if kind == "reorder":
        pl, _ = _blocks((2 * case["layers"],), case, seed)
        b0, out = case["from"] // RB, {}
        for p, t in pl.items():
            new = t.clone()
            for i, j in enumerate(_index(case, seed, case["batch"])):
                new[:, i, :, b0:] = t[:, j, :, b0:]
            out[p] = new.double() if p == "scale" else None
        return out
    st = prepare(case, seed) if not own else None
    if st is None:
        return None
    out = []
    for pl, _ in st["pairs"]:
        rows = [pl["scale"][j] if st["blocks"] is None else pl["scale"][j][:, st["blocks"][r].long()]
                for r, j in enumerate(_index(case, seed, case["out"]))]
        out.append({**dict.fromkeys(("a", "b", "mask", "meta", "exc")), "scale": torch.stack(rows).double().reshape(-1)})
    return out
