"""The operators around a serving engine's K/V cache, as calls that can be timed one by one.

A batch of prompts goes through attention_prefill, the tokens that a draft model proposes (or the one token of a
plain decoding step) through attention_tree over a paged binary16 cache; kv_pack_f16_pages writes the K/V rows into
the pages, kv_pages_assign forks, frees and grows sequences, kv_pages_compact keeps the accepted drafts,
token_logprobs scores tokens and lists the alternatives.

listed() names the cases, draw() makes more of the same ranges, prepare() builds what the engine holds before the
call, run() makes one pass, work() counts the bytes and operations a pass cannot do without, exact() gives the
computed numbers in 64 bits.  With own false run() computes the operators from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

NEG_INF = float("-inf")


def listed():
    return [
        # A batch of chat prompts of mixed lengths, packed without padding.
        {"name": "prefill_ragged", "op": "prefill", "seqs": 13, "tokens": 6001, "nq": 28, "nkv": 4, "hd": 128,
         "past": 0},
        # One long prompt.
        {"name": "prefill_long", "op": "prefill", "seqs": 1, "tokens": 8192, "nq": 32, "nkv": 8, "hd": 128, "past": 0},
        # A plain decoding step: one token of each of 37 sequences of very different lengths.
        {"name": "decode_37", "op": "tree", "seqs": 37, "drafts": 1, "lo": 200, "hi": 30000, "page": 64, "nq": 32,
         "nkv": 8, "hd": 128},
        # Trees of up to 60 drafted tokens of six sequences checked at once.
        {"name": "tree_6x60", "op": "tree", "seqs": 6, "drafts": 60, "lo": 700, "hi": 9000, "page": 32, "nq": 40,
         "nkv": 8, "hd": 128},
        # The K/V rows of one decoding step, each to a page of its own sequence: the smallest call.
        {"name": "pack_step", "op": "pack", "seqs": 64, "tokens": 64, "page": 64, "nkv": 8, "hd": 128},
        # The K/V rows of a packed batch of prompts.
        {"name": "pack_prompts", "op": "pack", "seqs": 5, "tokens": 8192, "page": 64, "nkv": 8, "hd": 128},
        # Beam search over 8 rows of one short prompt, all layers' last pages copied.
        {"name": "assign_beam", "op": "assign", "rows": 8, "width": 41, "page": 16, "layers": 28, "nkv": 2, "hd": 128,
         "pool": 700},
        # Parallel sampling: many rows forked from a few prompts, others freed and grown.
        {"name": "assign_fork", "op": "assign", "rows": 190, "width": 60, "page": 32, "layers": 6, "nkv": 8, "hd": 128,
         "pool": 5500},
        # Accepted drafts of one sequence moved down in every layer.
        {"name": "compact_1", "op": "compact", "rows": 1, "drafts": 24, "width": 100, "page": 32, "layers": 36, "nkv": 8,
         "hd": 128},
        # The same for a batch.
        {"name": "compact_48", "op": "compact", "rows": 48, "drafts": 60, "width": 20, "page": 64, "layers": 24,
         "nkv": 4, "hd": 128},
        # The score of one sampled token with its alternatives.
        {"name": "logprobs_1", "op": "logprobs", "tokens": 1, "vocab": 151936, "top": 20},
        # A prompt scored for an evaluation, five alternatives per token.
        {"name": "logprobs_1500", "op": "logprobs", "tokens": 1500, "vocab": 128256, "top": 5},
    ]


# ------------------------------------------------------------------------------------------------ drawing

MOST_BYTES = 1_300_000_000
MOST_FLOPS = 550_000_000_000
MOST_POOL = 4_000_000_000  # bytes of all K and V pages of a drawn case


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _draw(rng)
        if c["op"] in ("assign", "compact"):
            pages = c.get("pool", c["rows"] * c["width"])
            if 4 * c["layers"] * pages * c["page"] * c["nkv"] * c["hd"] > MOST_POOL:
                continue
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return c


def _heads(rng):
    nkv = rng.choice([1, 2, 3, 4, 5, 8, 8, 16])
    return nkv * rng.choice([1, 2, 4, 5, 7, 8]), nkv, rng.choice([64, 64, 96, 128, 128, 128, 160, 192, 256, 512])


def _draw(rng):
    op = rng.choice(["prefill", "prefill", "prefill", "tree", "tree", "tree", "pack", "assign", "compact",
                     "logprobs", "logprobs"])
    nq, nkv, hd = _heads(rng)
    page = rng.choice([16, 32, 64, 128])
    if op == "prefill":
        seqs = _log(rng, 1, 40)
        return {"op": op, "seqs": seqs, "tokens": max(seqs, _log(rng, 1, 9000)), "nq": nq, "nkv": nkv, "hd": hd,
                "past": rng.choice([0, 0, _log(rng, 1, 4000)])}
    if op == "tree":
        hi = _log(rng, 20, 60000)
        return {"op": op, "seqs": _log(rng, 1, 80), "drafts": rng.choice([1, 1, _log(rng, 2, 64)]),
                "lo": _log(rng, 1, hi), "hi": hi, "page": page, "nq": nq, "nkv": nkv, "hd": hd}
    if op == "pack":
        seqs = _log(rng, 1, 100)
        return {"op": op, "seqs": seqs, "tokens": max(seqs, _log(rng, 1, 9000)), "page": page, "nkv": nkv, "hd": hd}
    if op == "assign":
        rows = _log(rng, 2, 250)
        width = _log(rng, 4, 160)
        return {"op": op, "rows": rows, "width": width, "page": page, "layers": _log(rng, 1, 30),
                "nkv": min(nkv, 8), "hd": min(hd, 128), "pool": rows * width + rng.randint(1, 200)}
    if op == "compact":
        return {"op": op, "rows": _log(rng, 1, 64), "drafts": _log(rng, 1, 64), "width": _log(rng, 5, 60),
                "page": page, "layers": _log(rng, 1, 36), "nkv": min(nkv, 8), "hd": min(hd, 128)}
    return {"op": op, "tokens": _log(rng, 1, 2000), "vocab": _log(rng, 1000, 160000),
            "top": rng.choice([0, 1, 5, 10, 20, 32])}


# ------------------------------------------------------------------------------------------------ lengths

def _rng(case):
    """Lengths belong to the case, contents to the seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _split(rng, total, parts):
    """total tokens in parts lengths of at least one, some short and some long."""
    w = [math.exp(rng.gauss(0, 1)) for _ in range(parts)]
    lens = [1 + int((total - parts) * x / sum(w)) for x in w]
    lens[rng.randrange(parts)] += total - sum(lens)
    return lens


def _lens(case):
    rng = _rng(case)
    op = case["op"]
    if op == "prefill":
        q = _split(rng, case["tokens"], case["seqs"])
        return q, [n + (rng.randint(0, case["past"]) if case["past"] else 0) for n in q]
    if op == "tree":
        ctx = [_log(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
        d = case["drafts"]
        return ctx, [d if d == 1 else rng.randint(max(1, d // 2), d) for _ in ctx]
    if op == "pack":
        new = _split(rng, case["tokens"], case["seqs"])
        return [rng.randint(0, 4 * case["page"]) for _ in new], new
    if op == "compact":
        room = case["width"] * case["page"] - case["drafts"]
        return ([rng.randint(0, max(0, room)) for _ in range(case["rows"])],
                [rng.randint(0, min(12, case["drafts"])) for _ in range(case["rows"])])
    return None


def _assign_plan(case):
    """Rows with the pages they hold: groups of rows share the full pages of a prompt, some rows are empty, some
    hold a page more than their length needs."""
    rng = _rng(case)
    R, W, ps, P = case["rows"], case["width"], case["page"], case["pool"]
    ids = list(range(P))
    rng.shuffle(ids)
    table, lens = [], []
    while len(table) < R:
        if rng.random() < 0.15:
            table.append([])
            lens.append(0)
            continue
        n = rng.randint(1, max(1, (W - 2) * ps))
        full = n // ps
        shared = [ids.pop() for _ in range(full)]
        for _ in range(min(R - len(table), rng.choice([1, 1, 2, 4]))):
            extra = (1 if n % ps else 0) + (1 if rng.random() < 0.2 and full + 2 <= W else 0)
            table.append(shared + [ids.pop() for _ in range(extra)])
            lens.append(n)
    parents = []
    for r in range(R):
        u = rng.random()
        parents.append(-1 if u < 0.1 else r if u < 0.45 else rng.randrange(R))
    reserve = [rng.choice([0, 1, 1, ps, 2 * ps]) for _ in range(R)]
    return table, lens, parents, reserve


# ------------------------------------------------------------------------------------------------ inputs

def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _pool(g, shape):
    """Binary16 pages filled with what K/V rows look like."""
    t = torch.empty(shape, dtype=torch.float16, device="cuda")
    flat = t.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device="cuda").to(torch.float16)
    return t


def _tables(rng, need, pages, width):
    """Block table [rows, width], each row's pages drawn from the pool without order, -1 behind them."""
    ids = list(range(pages))
    rng.shuffle(ids)
    return _i32([[ids.pop() for _ in range(n)] + [-1] * (width - n) for n in need])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)
    rng = random.Random(int(seed) * 7919 + 5)
    op = case["op"]
    s = {"case": case}
    if op == "logprobs":
        T, V = case["tokens"], case["vocab"]
        x = torch.randn((T, V), generator=g, device="cuda").mul_(2.5)
        ids = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
        # a confident model: the scored token stands out in most rows
        x[torch.arange(T, device="cuda"), ids.long()] += 8.0 * torch.rand(T, generator=g, device="cuda")
        s.update(logits=x, ids=ids)
        return s
    if op == "assign":
        table, lens, parents, reserve = _assign_plan(case)
        W, P = case["width"], case["pool"]
        refs = [0] * P
        for row in table:
            for p in row:
                refs[p] += 1
        perm = list(range(P))
        rng.shuffle(perm)
        shape = (case["layers"], P, case["page"], case["nkv"], case["hd"])
        new_refs = [0] * P
        for p in range(P):
            new_refs[perm[p]] = refs[p]
        s.update(k=_pool(g, shape), v=_pool(g, shape),
                 table=_i32([[perm[p] for p in row] + [-1] * (W - len(row)) for row in table]), lens=_i32(lens),
                 refs=_i32(new_refs), parents=_i32(parents), reserve=_i32(reserve))
        return s
    nkv, hd = case["nkv"], case["hd"]
    if op == "prefill":
        nq_lens, kv_lens = _lens(case)
        T, S = sum(nq_lens), sum(kv_lens)
        qkv = torch.randn((T, (case["nq"] + 2 * nkv) * hd), generator=g, device="cuda")
        q = qkv[:, :case["nq"] * hd].mul_(1.5).view(T, case["nq"], hd)
        k = _pool(g, (S, nkv, hd))
        v = _pool(g, (S, nkv, hd))
        s.update(q=q, k=k, v=v, q_lens=nq_lens, kv_lens=kv_lens, cu=_cu(nq_lens), cuk=_cu(kv_lens))
        return s
    ps = case["page"]
    if op == "tree":
        ctx, drafts = _lens(case)
        need = [-(-(c + d) // ps) for c, d in zip(ctx, drafts)]
        width = max(need) + 2
        pages = sum(need) + 7
        T = sum(drafts)
        masks = []
        for d in drafts:
            rows = []
            for i in range(d):  # a random tree: each draft follows an earlier one, or the context
                parent = rng.randint(-1, i - 1)
                rows.append((rows[parent] if parent >= 0 else 0) | (1 << i))
            masks += [m - (1 << 64) if m >> 63 else m for m in rows]
        s.update(q=torch.randn((T, case["nq"], hd), generator=g, device="cuda").mul_(1.5),
                 k=_pool(g, (pages, ps, nkv, hd)), v=_pool(g, (pages, ps, nkv, hd)),
                 table=_tables(rng, need, pages, width), ctx=ctx, drafts=drafts, lens=_i32(ctx), cu=_cu(drafts),
                 mask=torch.tensor(masks, dtype=torch.int64, device="cuda"))
        return s
    if op == "pack":
        old, new = _lens(case)
        need = [-(-(a + b) // ps) for a, b in zip(old, new)]
        pages = sum(need) + 3
        T = sum(new)
        qkv = torch.randn((T, 3 * nkv * hd), generator=g, device="cuda")
        s.update(ks=qkv[:, nkv * hd:2 * nkv * hd], vs=qkv[:, 2 * nkv * hd:],
                 k=torch.zeros((pages, ps, nkv, hd), dtype=torch.float16, device="cuda"),
                 v=torch.zeros((pages, ps, nkv, hd), dtype=torch.float16, device="cuda"),
                 table=_tables(rng, need, pages, max(need)),
                 pos=_i32([a + i for a, b in zip(old, new) for i in range(b)]),
                 seqs=_i32([r for r, b in enumerate(new) for _ in range(b)]))
        return s
    if op == "compact":
        lens, n_path = _lens(case)
        R, D, W = case["rows"], case["drafts"], case["width"]
        need = [min(W, -(-(n + D) // ps)) for n in lens]
        pages = sum(need) + 3
        path = [sorted(rng.sample(range(D), n)) + [0] * (D - n) for n in n_path]
        shape = (case["layers"], pages, ps, nkv, hd)
        s.update(k=_pool(g, shape), v=_pool(g, shape), table=_tables(rng, need, pages, W), lens=_i32(lens),
                 path=_i32(path), n_path=_i32(n_path))
        return s
    raise ValueError(op)


# ------------------------------------------------------------------------------------------------ the pass

def run(s):
    op = s["case"]["op"]
    return (_own if own else _plain)[op](s)


def _own_ops():
    from v7multiplikator_amd import ops
    return ops


class _Table:
    def __init__(self, **fns):
        self.fns = fns

    def __getitem__(self, op):
        return self.fns[op]


def _own_prefill(s):
    same = s["case"]["past"] == 0
    return _own_ops().attention_prefill(s["q"], s["k"], s["v"], s["cu"], None if same else s["cuk"])


def _own_tree(s):
    if s["case"]["drafts"] == 1:
        return _own_ops().attention_tree(s["q"], s["k"], s["v"], s["table"], s["lens"])
    return _own_ops().attention_tree(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], s["mask"])


def _own_pack(s):
    _own_ops().kv_pack_f16_pages(s["ks"], s["vs"], s["k"], s["v"], s["table"], s["pos"], s["seqs"])
    return s["k"], s["v"]


def _own_assign(s):
    t, n, r, short = _own_ops().kv_pages_assign(s["k"], s["v"], s["table"], s["lens"], s["refs"], s["parents"],
                                                s["reserve"])
    return t, n, r, short, s["k"], s["v"]


def _own_compact(s):
    n = _own_ops().kv_pages_compact(s["k"], s["v"], s["table"], s["lens"], s["path"], s["n_path"])
    return n, s["k"], s["v"]


def _own_logprobs(s):
    return _own_ops().token_logprobs(s["logits"], s["ids"], s["case"]["top"])


_own = _Table(prefill=_own_prefill, tree=_own_tree, pack=_own_pack, assign=_own_assign, compact=_own_compact,
              logprobs=_own_logprobs)


def _attend(q, k, v, seen):
    """q [n, nq, hd] f32 against k, v [m, nkv, hd]; seen [n, m] says which keys a token attends to."""
    n, nq, hd = q.shape
    m, nkv, _ = k.shape
    G = nq // nkv
    qh = q.view(n, nkv, G, hd).permute(1, 2, 0, 3).reshape(nkv, G * n, hd)
    kh = k.float().permute(1, 2, 0).contiguous()
    vh = v.float().permute(1, 0, 2).contiguous()
    out = torch.empty((nkv, G * n, hd), dtype=torch.float32, device=q.device)
    for h in range(nkv):
        sc = torch.mm(qh[h], kh[h]).mul_(1.0 / math.sqrt(hd)).view(G, n, m)
        sc.masked_fill_(~seen, NEG_INF)
        sc.sub_(sc.amax(-1, keepdim=True)).exp_()
        den = sc.sum(-1).view(G * n, 1)
        out[h] = torch.mm(sc.view(G * n, m), vh[h]).div_(den)
    return out.view(nkv, G, n, hd).permute(2, 0, 1, 3).reshape(n, nq, hd)


def _plain_prefill(s):
    out = torch.empty(s["q"].shape, dtype=torch.float32, device="cuda")
    a = b = 0
    for n, m in zip(s["q_lens"], s["kv_lens"]):
        i = torch.arange(n, device="cuda").view(n, 1)
        j = torch.arange(m, device="cuda").view(1, m)
        out[a:a + n] = _attend(s["q"][a:a + n].contiguous(), s["k"][b:b + m], s["v"][b:b + m], j <= i + (m - n))
        a, b = a + n, b + m
    return out


def _plain_tree(s):
    ps = s["case"]["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float32, device="cuda")
    a = 0
    for r, (c, d) in enumerate(zip(s["ctx"], s["drafts"])):
        m = c + d
        pages = s["table"][r, :-(-m // ps)].long()
        k = s["k"][pages].flatten(0, 1)[:m]
        v = s["v"][pages].flatten(0, 1)[:m]
        j = torch.arange(d, device="cuda")
        seen = torch.ones((d, m), dtype=torch.bool, device="cuda")
        seen[:, c:] = (s["mask"][a:a + d].view(d, 1) >> j) & 1 != 0
        out[a:a + d] = _attend(s["q"][a:a + d], k, v, seen)
        a += d
    return out


def _plain_pack(s):
    ps = s["case"]["page"]
    pos = s["pos"].long()
    page = s["table"][s["seqs"].long(), pos // ps].long()
    shape = (pos.numel(), s["case"]["nkv"], s["case"]["hd"])
    s["k"][page, pos % ps] = s["ks"].reshape(shape).to(torch.float16)
    s["v"][page, pos % ps] = s["vs"].reshape(shape).to(torch.float16)
    return s["k"], s["v"]


def _plain_assign(s):
    table, lens, refs, parents, reserve = (s[n].long() for n in ("table", "lens", "refs", "parents", "reserve"))
    (R, W), P, ps = table.shape, refs.numel(), s["case"]["page"]
    dev = table.device
    col, row = torch.arange(W, device=dev), torch.arange(R, device=dev)
    held = (table >= 0).long().cumprod(1).sum(1)
    live = parents >= 0
    par = parents.clamp(min=0)
    # the row that takes over a parent's last and spare pages: the parent itself, else the lowest of its children
    first = torch.full((R,), R, device=dev).scatter_reduce(0, par, torch.where(live, row, R), "amin")
    owner = torch.where(parents == row, row, first)
    owns = live & (owner[par] == row)
    n = torch.where(live, torch.minimum(lens[par], held[par] * ps), 0)
    full = n // ps
    keep = torch.where(owns, held[par], torch.where(live, full, 0))
    want = torch.where(live, torch.maximum(keep, ((n + reserve + ps - 1) // ps).clamp(max=W)), 0)
    tail = live & ~owns & (n % ps != 0)
    want = torch.maximum(want, torch.where(tail, full + 1, 0))
    kept = col < keep.view(R, 1)
    out = torch.where(kept, table[par], -1)
    count = refs.clone()
    old = col < held.view(R, 1)
    count.index_add_(0, table.clamp(min=0).flatten(), -old.long().flatten())
    count.index_add_(0, out.clamp(min=0).flatten(), kept.long().flatten())
    asked = (col >= keep.view(R, 1)) & (col < want.view(R, 1))
    rank = asked.flatten().long().cumsum(0).view(R, W) - 1
    free = torch.argsort((count > 0).long() * P + torch.arange(P, device=dev))
    n_free = (count <= 0).sum()
    got = asked & (rank < n_free)
    out = torch.where(got, free[rank.clamp(0, P - 1)], out)
    count = count.clamp(min=0)
    count.index_add_(0, out.clamp(min=0).flatten(), got.long().flatten())
    at = full.clamp(max=W - 1).view(R, 1)
    src = torch.gather(table[par], 1, at).squeeze(1)
    dst = torch.gather(out, 1, at).squeeze(1)
    copied = tail & (dst >= 0)
    n = torch.where(tail & ~copied, full * ps, n)
    # a row that copies nothing copies its first page onto itself: rows are moved without asking the host which
    inside = torch.arange(ps, device=dev) < (n % ps).view(R, 1)
    moved = (copied.view(R, 1) & inside).flatten().nonzero().squeeze(1)
    r, i = moved // ps, moved % ps
    for pool in (s["k"], s["v"]):
        pool[:, dst[r], i] = pool[:, src[r], i]
    short = asked.sum() - got.sum()
    i32 = torch.int32
    return out.to(i32), n.to(i32), count.to(i32), short.to(i32).view(1), s["k"], s["v"]


def _plain_compact(s):
    ps = s["case"]["page"]
    lens, path, n_path, table = s["lens"].long(), s["path"].long(), s["n_path"].long(), s["table"].long()
    R, A = path.shape
    i = torch.arange(A, device=path.device)
    on = (i < n_path.view(R, 1)).flatten().nonzero().squeeze(1)
    r, i = on // A, on % A
    src, dst = lens[r] + path[r, i], lens[r] + i
    for pool in (s["k"], s["v"]):
        pool[:, table[r, dst // ps], dst % ps] = pool[:, table[r, src // ps], src % ps]
    return (lens + n_path).to(torch.int32), s["k"], s["v"]


def _plain_logprobs(s):
    x, ids, K = s["logits"], s["ids"].long(), s["case"]["top"]
    T, V = x.shape
    z = x - x.amax(-1, keepdim=True)
    e = z.exp()
    den = e.sum(-1, keepdim=True)
    lse = den.log()
    entropy = lse.squeeze(1) - (e.mul_(z)).sum(-1) / den.squeeze(1)
    logp = torch.gather(z, 1, ids.view(T, 1)) - lse
    vals = torch.empty((T, K), dtype=torch.float32, device=x.device)
    tops = torch.empty((T, K), dtype=torch.int64, device=x.device)
    for j in range(K):  # argmax gives the lowest index of the greatest value
        tops[:, j] = z.argmax(-1)
        vals[:, j] = torch.gather(z, 1, tops[:, j:j + 1]).squeeze(1)
        z.scatter_(1, tops[:, j:j + 1], NEG_INF)
    return logp.squeeze(1), entropy, vals - lse, tops.to(torch.int32)


_plain = _Table(prefill=_plain_prefill, tree=_plain_tree, pack=_plain_pack, assign=_plain_assign,
                compact=_plain_compact, logprobs=_plain_logprobs)


# ------------------------------------------------------------------------------------------------ the work

def work(case):
    op = case["op"]
    if op == "logprobs":
        T, V, K = case["tokens"], case["vocab"], case["top"]
        return {"bytes": T * (4 * V + 4 + 8 + 8 * K), "flops": 5 * T * V}
    if op == "assign":
        table, lens, parents, reserve = _assign_plan(case)
        ps = case["page"]
        seen, copies = set(r for r, p in enumerate(parents) if p == r), 0
        for r, p in enumerate(parents):
            if p < 0 or p == r:
                continue
            if p in seen:
                copies += lens[p] % ps
            seen.add(p)
        row = 2 * case["layers"] * case["nkv"] * case["hd"] * 2
        books = 4 * (2 * case["rows"] * case["width"] + 2 * case["pool"] + 4 * case["rows"])
        return {"bytes": books + 2 * copies * row, "flops": 0}
    nkv, hd = case["nkv"], case["hd"]
    a, b = _lens(case)
    if op == "prefill":
        nq = case["nq"]
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(a, b))
        return {"bytes": 2 * 4 * sum(a) * nq * hd + 2 * 2 * sum(b) * nkv * hd, "flops": 4 * pairs * nq * hd}
    if op == "tree":
        nq = case["nq"]
        keys = sum(c + d for c, d in zip(a, b))
        pairs = sum(d * (c + (d + 1) / 2) for c, d in zip(a, b))
        return {"bytes": 2 * 4 * sum(b) * nq * hd + 2 * 2 * keys * nkv * hd + 4 * (keys // case["page"]),
                "flops": int(4 * pairs * nq * hd)}
    if op == "pack":
        return {"bytes": sum(b) * (2 * nkv * hd * (4 + 2) + 8), "flops": 0}
    moved = sum(b)
    return {"bytes": 2 * moved * 2 * case["layers"] * nkv * hd * 2 + 4 * (case["rows"] * 3 + moved), "flops": 0}


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    op = case["op"]
    if op == "pack" or op == "compact" or op == "assign":
        return _exact_moves(case, seed)
    s = prepare(case, seed)
    if op == "logprobs":
        x = s["logits"]
        T, K = x.shape[0], case["top"]
        logp = torch.empty(T, dtype=torch.float64, device="cuda")
        ent = torch.empty(T, dtype=torch.float64, device="cuda")
        tops = torch.empty((T, K), dtype=torch.float64, device="cuda")
        for a in range(0, T, 128):
            d = x[a:a + 128].double()
            lse = torch.logsumexp(d, -1)
            p = torch.exp(d - lse.view(-1, 1))
            ent[a:a + 128] = -(p * (d - lse.view(-1, 1))).sum(-1)
            logp[a:a + 128] = d[torch.arange(d.shape[0]), s["ids"][a:a + 128].long()] - lse
            if K:
                tops[a:a + 128] = d.sort(-1, descending=True).values[:, :K] - lse.view(-1, 1)
        return logp, ent, tops, None
    # attention, one query head at a time
    q, hd, G = s["q"], case["hd"], case["nq"] // case["nkv"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    at = kv = 0
    first, second = _lens(case)
    for r in range(case["seqs"]):
        if op == "prefill":
            n, m = first[r], second[r]
            k, v = s["k"][kv:kv + m], s["v"][kv:kv + m]
            bias = torch.zeros((n, m), dtype=torch.float64, device="cuda")
            bias.masked_fill_(torch.ones((n, m), dtype=torch.bool, device="cuda").triu(m - n + 1), NEG_INF)
            kv += m
        else:
            c, n = first[r], second[r]
            m, ps = c + n, case["page"]
            ids = torch.arange(m, device="cuda")
            page = s["table"][r].long()[ids // ps]
            k, v = s["k"][page, ids % ps], s["v"][page, ids % ps]
            bias = torch.zeros((n, m), dtype=torch.float64, device="cuda")
            words = s["mask"][at:at + n].tolist()
            off = [[NEG_INF if not (w >> j) & 1 else 0.0 for j in range(n)] for w in words]
            bias[:, c:] = torch.tensor(off, dtype=torch.float64, device="cuda")
        for h in range(case["nq"]):
            kd, vd = k[:, h // G].double(), v[:, h // G].double()
            sc = torch.mm(q[at:at + n, h].double(), kd.t().contiguous()) / math.sqrt(hd) + bias
            out[at:at + n, h] = torch.mm(torch.softmax(sc, -1), vd)
        at += n
    return out


def _exact_moves(case, seed):
    """Nothing is computed but a rounding to binary16, whose unrounded values exist for the packed rows only."""
    if case["op"] != "pack":
        return None
    s = prepare(case, seed)
    ps = case["page"]
    outs = []
    for src, pool in ((s["ks"], s["k"]), (s["vs"], s["v"])):
        d = pool.double()
        pos, seq = s["pos"].long(), s["seqs"].long()
        d.view(-1, *d.shape[2:])[s["table"].long()[seq, pos // ps] * ps + pos % ps] = \
            src.double().reshape(-1, case["nkv"], case["hd"])
        outs.append(d)
    return tuple(outs)
