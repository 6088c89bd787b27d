"""GPU: the pages of a K/V cache (kv_pack_f16_pages, kv_pages_assign, kv_pages_compact), bit for bit against plain
Python on the CPU, and a serving loop that uses them together with the attention and the token scores."""
from __future__ import annotations

import random

import numpy as np
import pytest

from . import attention_ref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X")
    from v7multiplikator_amd import ops as o
    return o


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(seed, layers, P, ps, H, D, layout=0):
    """Random binary16 bit patterns, NaN among them: pages move bits."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lead = (layers, P) if layers else (P,)

    def bits(*shape):
        return torch.randint(-32768, 32768, shape, generator=g, device="cuda", dtype=torch.int16).view(torch.float16)
    if layout == 1:
        kv = bits(*lead, 2, ps, H, D)
        return kv.select(len(lead), 0), kv.select(len(lead), 1)
    if layout == 2:  # rows of 12 bytes more: no 16-byte alignment
        k, v = bits(*lead, ps, H * D + 4), bits(*lead, ps, H * D + 4)
        return tuple(t[..., :H * D].unflatten(-1, (H, D)) for t in (k, v))
    return bits(*lead, ps, H, D), bits(*lead, ps, H, D)


def as_bits(t):
    return t.cpu().contiguous().view(torch.int16).numpy().copy()


# ------------------------------------------------------------------------------------------------ pack

@pytest.mark.parametrize("H,D,ps,layout", [(1, 64, 16, 0), (8, 128, 64, 0), (2, 96, 32, 1), (3, 160, 16, 2), (16, 256, 128, 0),
                                           (5, 64, 16, 0), (8, 512, 16, 1)])
@pytest.mark.parametrize("given", [True, False])
def test_pack_pages(ops, H, D, ps, layout, given):
    B, W, P = 9, 5, 60
    kp, vp = pool(H * D, 0, P, ps, H, D, layout)
    want_k, want_v = as_bits(kp), as_bits(vp)
    rng = random.Random(D)
    ids = list(range(P))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(W)] for _ in range(B)]
    table[2][1], table[3][0] = -1, P
    T = 200 if given else B
    cells = [(b, p) for b in range(B) for p in range(W * ps)]
    places = rng.sample(cells, T) if given else [(b, rng.randrange(W * ps)) for b in range(B)]
    if given:  # none of these has a place
        places[5], places[6], places[7], places[8] = (-1, 3), (B, 0), (1, -1), (4, W * ps)
        places[9] = (0, 2147483647)
    else:
        places[2] = (2, ps)
    src = torch.randn(T, 3 * H * D + 4, device="cuda") * torch.logspace(-9, 5, T, device="cuda")[:, None]
    k, v = src[:, 4:4 + H * D], src[:, 4 + H * D:4 + 2 * H * D]
    ops.kv_pack_f16_pages(k, v, kp, vp, i32(table), i32([p for _, p in places]),
                          i32([b for b, _ in places]) if given else None)
    kn, vn = (as_bits(t.to(torch.float16)).reshape(T, H, D) for t in (k, v))
    for t, (b, p) in enumerate(places):
        if 0 <= b < B and 0 <= p < W * ps and 0 <= table[b][p // ps] < P:
            want_k[table[b][p // ps], p % ps] = kn[t]
            want_v[table[b][p // ps], p % ps] = vn[t]
    assert np.array_equal(as_bits(kp), want_k) and np.array_equal(as_bits(vp), want_v)


# ------------------------------------------------------------------------------------------------ compact

@pytest.mark.parametrize("layers,H,D,ps,layout", [(1, 1, 64, 16, 0), (3, 2, 128, 32, 0), (2, 3, 96, 16, 1), (2, 8, 64, 64, 2),
                                                  (0, 4, 512, 16, 0)])
@pytest.mark.parametrize("A", [1, 7, 8, 9, 64, 150])
def test_compact(ops, layers, H, D, ps, layout, A):
    B, W = 11, 14
    P = B * W
    kp, vp = pool(A + ps, layers, P, ps, H, D, layout)
    want = [as_bits(kp), as_bits(vp)]
    rng = random.Random(A * 7 + ps)
    ids = list(range(P))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(W)] for _ in range(B)]
    cap = W * ps
    lens = [rng.randrange(0, max(1, cap - A)) for _ in range(B)]
    path = [sorted(rng.sample(range(A), rng.randint(0, A))) for _ in range(B)]
    n_path = [len(p) for p in path]
    path = [p + [0] * (A - len(p)) for p in path]
    lens[0], lens[1] = 0, cap  # nothing behind the second
    if A >= 7:
        path[2][:5], n_path[2] = [0, 2, 2, 3, 4], 5   # stops ascending after two
        path[3][:3], n_path[3] = [-1, 1, 2], 3        # never starts
        path[4][:3], n_path[4] = [1, 2147483647, 3], 3
        n_path[5] = A + 1000                          # read to the path's width
        path[5] = list(range(A))
        n_path[6] = -4
        lens[7] = -3                                  # as 0
        lens[8] = ps * 2
        table[8][2] = P + 5                           # no page behind its context
    got = ops.kv_pages_compact(kp, vp, i32(table), i32(lens), i32(path), i32(n_path))
    new_lens = []
    for r in range(B):
        ln = min(max(lens[r], 0), cap)
        place = lambda pos: (table[r][pos // ps], pos % ps)  # noqa: E731
        n, before = 0, -1
        for i in range(min(max(n_path[r], 0), A)):
            s = path[r][i]
            if s <= before or ln + s >= cap or ln + i >= cap:
                break
            if not (0 <= place(ln + s)[0] < P and 0 <= place(ln + i)[0] < P):
                break
            before, n = s, n + 1
        for w in want:
            old = w.copy()
            for i in range(n):
                (ps_, si), (pd, di) = place(ln + path[r][i]), place(ln + i)
                w[..., pd, di, :, :] = old[..., ps_, si, :, :]
        new_lens.append(ln + n)
    assert got.tolist() == new_lens
    assert np.array_equal(as_bits(kp), want[0]) and np.array_equal(as_bits(vp), want[1])


# ------------------------------------------------------------------------------------------------ assign

def plain_assign(table, lens, refs, parents, reserve, ps, pools):
    """The definition, one row after the other."""
    B, W, P = len(table), len(table[0]) if table else 0, len(refs)

    def held(row):
        n = 0
        while n < W and 0 <= table[row][n] < P:
            n += 1
        return n
    refs = list(refs)
    out, new_lens, asks = [], [], []
    owners = {}
    for r, p in enumerate(parents):
        if 0 <= p < B and (p == r or (parents[p] != p and p not in owners)):
            owners[p] = r
    for r in range(B):
        for i in range(held(r)):
            refs[table[r][i]] -= 1
    for r, p in enumerate(parents):
        if not 0 <= p < B:
            out.append([])
            new_lens.append(0)
            asks.append((0, None))
            continue
        h = held(p)
        n = min(max(lens[p], 0), h * ps)
        full = n // ps
        row = [table[p][i] for i in range(h if owners[p] == r else full)]
        for pg in row:
            refs[pg] += 1
        copy = p if owners[p] != r and n % ps else None
        want = min(W, -(-(n + max(reserve[r] if reserve else 0, 0)) // ps))
        want = max(want, len(row), full + 1 if copy is not None else 0)
        out.append(row)
        new_lens.append(n)
        asks.append((want - len(row), copy))
    free = iter([p for p in range(P) if refs[p] <= 0])
    short, gone = 0, False
    for r, (need, copy) in enumerate(asks):
        full = len(out[r])
        for j in range(need):
            pg = None if gone else next(free, None)
            if pg is None:
                gone = True
                short += 1
                if j == 0 and copy is not None:
                    new_lens[r] = full * ps
                continue
            out[r].append(pg)
            refs[pg] = 1
            if j == 0 and copy is not None:
                for w in pools:
                    rest = new_lens[r] - full * ps
                    w[..., pg, :rest, :, :] = w[..., table[copy][full], :rest, :, :]
    return [row + [-1] * (W - len(row)) for row in out], new_lens, refs, short


def random_state(rng, B, W, ps, P):
    """Tables whose rows share prefixes, with counts that fit, and some pages held from outside."""
    ids = list(range(P))
    rng.shuffle(ids)
    refs = [0] * P
    table, lens = [], []
    for _ in range(B):
        if table and rng.random() < 0.4:
            src = rng.randrange(len(table))
            full = lens[src] // ps
            row = [p for p in table[src][:rng.randint(0, full)] if p >= 0]
        else:
            row = []
        grow = rng.randint(0, min(W - len(row), 4))
        row = row + [ids.pop() for _ in range(min(grow, len(ids)))]
        for p in row:
            refs[p] += 1
        lens.append(rng.randint(0, len(row) * ps))
        table.append(row + [-1] * (W - len(row)))
    for _ in range(min(3, len(ids))):
        refs[ids.pop()] += 2
    return table, lens, refs


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("B,W,ps,spare,layers,H,D,layout", [
    (1, 1, 16, 4, 1, 1, 64, 0), (8, 6, 16, 5, 2, 2, 64, 0), (40, 9, 32, 30, 1, 1, 96, 1), (33, 20, 16, 200, 3, 1, 64, 2),
    (130, 5, 16, 2, 0, 1, 64, 0),
    (40, 9, 16, 25000, 1, 1, 64, 0), (1100, 3, 16, 7, 1, 1, 64, 0), (20, 70, 16, 600, 1, 1, 64, 0),
])
def test_assign(ops, seed, B, W, ps, spare, layers, H, D, layout):
    rng = random.Random(seed * 1009 + B)
    P = 4 * B + spare
    table, lens, refs = random_state(rng, B, W, ps, P)
    kp, vp = pool(seed, layers, P, ps, H, D, layout)
    pools = [as_bits(kp), as_bits(vp)]
    parents = [rng.choice([r, rng.randrange(B), rng.randrange(B), -1]) for r in range(B)]
    if seed % 4 == 1:
        parents = [0] * B
    if seed % 4 == 2:
        parents = list(range(B))
    if seed % 4 == 3 and B > 4:
        parents[1], parents[2] = B, -7
        lens[0], lens[3] = 1 << 30, -5  # as the most and the least they can be
        if W > 2:
            table[3][1] = P + 9  # the row ends here
            table[3][2:] = [-1] * (W - 2)
    # a broken row's pages stay counted as they were found
    reserve = [rng.choice([0, 1, ps, 3 * ps, -2]) for _ in range(B)] if seed % 3 else None
    t, n, c, short = ops.kv_pages_assign(kp, vp, i32(table), i32(lens), i32(refs), i32(parents),
                                         i32(reserve) if reserve else None)
    wt, wn, wc, ws = plain_assign(table, lens, refs, parents, reserve, ps, pools)
    assert t.tolist() == wt and n.tolist() == wn and c.tolist() == wc and short.tolist() == [ws]
    assert np.array_equal(as_bits(kp), pools[0]) and np.array_equal(as_bits(vp), pools[1])


def test_assign_many_rows_and_pages(ops):
    """More rows than one scan takes, and a pool whose free pages lie far apart."""
    rng = random.Random(3)
    B, W, ps, P = 2500, 4, 16, 70000
    table = [[-1] * W for _ in range(B)]
    lens = [0] * B
    refs = [1] * P
    for p in rng.sample(range(P), 6000):
        refs[p] = 0
    kp, vp = (torch.zeros((P, ps, 1, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    reserve = [rng.randint(0, 60) for _ in range(B)]
    t, n, c, short = ops.kv_pages_assign(kp, vp, i32(table), i32(lens), i32(refs), i32(range(B)), i32(reserve))
    wt, wn, wc, ws = plain_assign(table, lens, refs, list(range(B)), reserve, ps, [])
    assert t.tolist() == wt and n.tolist() == wn and c.tolist() == wc and short.tolist() == [ws]


def test_assign_empty(ops):
    kp = torch.zeros((0, 16, 1, 64), dtype=torch.float16, device="cuda")
    t, n, c, short = ops.kv_pages_assign(kp, kp.clone(), i32([[-1, -1]]), i32([5]), i32([]).int(), i32([0]), i32([40]))
    assert t.tolist() == [[-1, -1]] and n.tolist() == [0] and short.tolist() == [2]
    kp = torch.zeros((2, 16, 1, 64), dtype=torch.float16, device="cuda")
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    t, n, c, short = ops.kv_pages_assign(kp, kp.clone(), none, e, i32([0, 4]), e)
    assert t.shape == (0, 3) and c.tolist() == [0, 4] and short.tolist() == [0]


def test_pages_past_32_bit_offsets(ops):
    """Pages whose element offsets pass 2^32: written, copied and moved at the far end."""
    P, ps, H, D = 17000, 256, 8, 128
    kp = torch.zeros((P, ps, H, D), dtype=torch.float16, device="cuda")
    vp = torch.zeros((P, ps, H, D), dtype=torch.float16, device="cuda")
    src = torch.randn(3, 2 * H * D, device="cuda")
    ops.kv_pack_f16_pages(src[:, :H * D], src[:, H * D:], kp, vp, i32([[P - 1]]), i32([0, 2, 5]), i32([0, 0, 0]))
    half = src.half()
    assert torch.equal(kp[P - 1, 2].flatten(), half[1, :H * D]) and torch.equal(vp[P - 1, 5].flatten(), half[2, H * D:])
    assert ops.kv_pages_compact(kp, vp, i32([[P - 1]]), i32([1]), i32([[1, 4]]), i32([2])).tolist() == [3]
    assert torch.equal(kp[P - 1, 1].flatten(), half[1, :H * D]) and torch.equal(kp[P - 1, 2].flatten(), half[2, :H * D])
    refs = torch.ones(P, dtype=torch.int32, device="cuda")
    refs[P - 3] = 0
    t, n, c, short = ops.kv_pages_assign(kp, vp, i32([[P - 1], [-1]]), i32([3, 0]), refs, i32([0, 0]))
    assert t.tolist() == [[P - 1], [P - 3]] and n.tolist() == [3, 3] and short.tolist() == [0]
    assert torch.equal(kp[P - 3, :3], kp[P - 1, :3]) and torch.equal(vp[P - 3, :3], vp[P - 1, :3])
    assert (kp[P - 3, 3:] == 0).all()


def test_pages_refusals(ops):
    from v7multiplikator_amd._lib import V7GError
    kp = torch.zeros((2, 4, 16, 2, 64), dtype=torch.float16, device="cuda")
    vp = kp.clone()
    t, one = i32([[0, 1]]), i32([1])
    src = torch.zeros(1, 128, device="cuda")
    with pytest.raises(ValueError):  # a layer is packed at a time
        ops.kv_pack_f16_pages(src, src.clone(), kp, vp, t, one)
    with pytest.raises(ValueError):
        ops.kv_pack_f16_pages(src[:, :64], src[:, 64:], kp[0], vp[0], t, one)
    with pytest.raises(ValueError):  # two tokens, one row, no seqs
        ops.kv_pack_f16_pages(src.repeat(2, 1), src.repeat(2, 1), kp[0], vp[0], t, i32([0, 1]))
    with pytest.raises(V7GError):  # K pages over V pages
        ops.kv_pack_f16_pages(src, src.clone(), kp[0], kp[0], t, one)
    with pytest.raises(ValueError):
        ops.kv_pages_assign(kp, vp, t, one, i32([0, 0]), one)
    with pytest.raises(TypeError):
        ops.kv_pages_assign(kp, vp, t.long(), one, i32([0] * 4), one)
    with pytest.raises(V7GError):
        ops.kv_pages_assign(kp, kp, t, one, i32([0] * 4), one)
    with pytest.raises(ValueError):
        ops.kv_pages_compact(kp, vp, t, one, i32([[1], [2]]), one)
    with pytest.raises(V7GError):
        ops.kv_pages_compact(kp, kp, t, one, i32([[1]]), one)


# ------------------------------------------------------------------------------------------------ together

def _serving_loop(ops, seed, captured):
    """Prompts packed and attended, forked, drafts packed, attended as trees, scored, the accepted ones kept; every
    attention result against 64 bits over the rows the cache should hold."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    H, G, D, ps, W, P, V = 2, 4, 128, 16, 8, 40, 500
    B = 5
    kp, vp = (torch.full((P, ps, H, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    prompts = [21, 40, 1]
    refs = torch.zeros(P, dtype=torch.int32, device="cuda")
    table, lens = torch.full((B, W), -1, dtype=torch.int32, device="cuda"), i32([0] * B)
    rows = list(range(B))
    table, lens, refs, short = ops.kv_pages_assign(kp, vp, table, lens, refs, i32(rows), i32(prompts + [0, 0]))
    assert short.tolist() == [0]

    def rnd(*s):
        return torch.randn(s, generator=g, device="cuda")
    T = sum(prompts)
    qkv = rnd(T, (G * H + 2 * H) * D)
    q = qkv[:, :G * H * D].view(T, G * H, D)
    k, v = qkv[:, G * H * D:(G + 1) * H * D], qkv[:, (G + 1) * H * D:]
    pos = i32([i for n in prompts for i in range(n)])
    seq = i32([b for b, n in enumerate(prompts) for _ in range(n)])
    ops.kv_pack_f16_pages(k, v, kp, vp, table, pos, seq)
    cu = i32([0, 21, 61, 62])
    kh, vh = k.half().view(T, H, D), v.half().view(T, H, D)
    out = ops.attention_prefill(q, kh, vh, cu)
    cache = []
    for a, n in zip((0, 21, 61), prompts):
        want, bound = R.attend(q[a:a + n], kh[a:a + n], vh[a:a + n], R.causal(n, n))
        R.check(out[a:a + n], want, bound)
        cache.append((kh[a:a + n], vh[a:a + n]))
    lens = i32(prompts + [0, 0])
    # rows 1 and 3 continue prompt 1, row 4 prompt 0, row 0 stays, row 2 is freed
    parents, drafts = [0, 1, -1, 1, 0], [6, 5, 0, 9, 1]
    table, lens, refs, short = ops.kv_pages_assign(kp, vp, table, lens, refs, i32(parents), i32(drafts))
    assert short.tolist() == [0] and lens.tolist() == [21, 40, 0, 40, 21]
    cache = [cache[p] if p >= 0 else (kh[:0], vh[:0]) for p in parents]
    base = lens.tolist()
    T = sum(drafts)
    dq, dk, dv = rnd(T, G * H, D), rnd(T, H * D), rnd(T, H * D)
    masks, trees = [], []
    for d in drafts:
        rows_ = []
        for i in range(d):
            parent = rng.randint(-1, i - 1)
            rows_.append((rows_[parent] if parent >= 0 else 0) | 1 << i)
        trees.append(rows_)
        masks += rows_
    dcu = [0]
    for d in drafts:
        dcu.append(dcu[-1] + d)
    accepted = []
    for rows_ in trees:  # the longest path
        best = max(rows_, key=lambda m: bin(m).count("1"), default=0)
        accepted.append([j for j in range(len(rows_)) if best >> j & 1])
    args = dict(pos=i32([b + i for b, d in zip(base, drafts) for i in range(d)]),
                seq=i32([r for r, d in enumerate(drafts) for _ in range(d)]), cu=i32(dcu),
                mask=torch.tensor(masks, dtype=torch.int64, device="cuda"),
                path=i32([a + [0] * (9 - len(a)) for a in accepted]), n=i32([len(a) for a in accepted]))
    logits, ids = rnd(T, V), i32([rng.randrange(V) for _ in range(T)])

    def step():
        ops.kv_pack_f16_pages(dk, dv, kp, vp, table, args["pos"], args["seq"])
        o = ops.attention_tree(dq, kp, vp, table, lens, args["cu"], args["mask"])
        scores = ops.token_logprobs(logits, ids, 3)
        return o, scores, ops.kv_pages_compact(kp, vp, table, lens, args["path"], args["n"])

    if captured:
        keep = kp.clone(), vp.clone()
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, scores, new_lens = step()
        for _ in range(3):
            kp.copy_(keep[0])
            vp.copy_(keep[1])
            graph.replay()
            torch.cuda.synchronize()
    else:
        o, scores, new_lens = step()
    lp = torch.log_softmax(logits.double(), -1)
    ref = lp[torch.arange(T), ids.long()]
    assert ((scores[0].double() - ref).abs() < 1e-5).all()
    dkh, dvh = dk.half().view(T, H, D), dv.half().view(T, H, D)
    a = 0
    for r, d in enumerate(drafts):
        ck, cv = (torch.cat([c, n[a:a + d]]) for c, n in zip(cache[r], (dkh, dvh)))
        seen = torch.zeros(d, base[r] + d, dtype=torch.bool)
        seen[:, :base[r]] = True
        for i in range(d):
            for j in range(d):
                seen[i, base[r] + j] = bool(trees[r][i] >> j & 1)
        want, bound = R.attend(dq[a:a + d], ck, cv, seen)
        R.check(o[a:a + d], want, bound, f"drafts of row {r}")
        pick = torch.tensor([a + j for j in accepted[r]], dtype=torch.long, device="cuda")
        cache[r] = tuple(torch.cat([c, n[pick]]) for c, n in zip(cache[r], (dkh, dvh)))
        a += d
    assert new_lens.tolist() == [b + len(x) for b, x in zip(base, accepted)]
    # one plain decoding step on what is left
    table, lens, refs, short = ops.kv_pages_assign(kp, vp, table, new_lens, refs, i32([0, 1, -1, 3, 4]), i32([1] * B))
    sk, sv, sq = rnd(B, H * D), rnd(B, H * D), rnd(B, G * H, D)
    ops.kv_pack_f16_pages(sk, sv, kp, vp, table, lens)
    o = ops.attention_tree(sq, kp, vp, table, lens)
    for r in (0, 1, 3, 4):
        ck, cv = (torch.cat([c, n[r:r + 1].half().view(1, H, D)]) for c, n in zip(cache[r], (sk, sv)))
        want, bound = R.attend(sq[r:r + 1], ck, cv, torch.ones(1, ck.shape[0], dtype=torch.bool))
        R.check(o[r:r + 1], want, bound, f"decoding row {r}")
    assert (o[2] == 0).all()  # freed: no page


@pytest.mark.parametrize("seed", [1, 2, 3])
@pytest.mark.parametrize("captured", [False, True])
def test_serving_loop(ops, seed, captured):
    _serving_loop(ops, seed, captured)
