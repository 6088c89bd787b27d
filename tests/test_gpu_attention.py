"""GPU: attention_prefill and attention_tree against 64-bit attention, at the sizes and masks where they can go wrong."""
from __future__ import annotations

import random

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


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=torch.float32, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sigma).to(dtype)


def cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ packed prompts

def prefill_case(ops, seed, q_lens, kv_lens, Hq, Hk, D, sigma=1.0, scale=None, extra=3, same=False):
    g = gen(seed)
    T, S = sum(q_lens) + extra, sum(kv_lens) + extra
    qkv = rnd(g, T, (Hq + 2 * Hk) * D, sigma=sigma)
    q = qkv[:, :Hq * D].view(T, Hq, D)
    if same:
        S = T
    kv = rnd(g, S, 2, Hk, D, dtype=torch.float16)
    k, v = kv[:, 0], kv[:, 1]
    out = torch.full((T, Hq + 1, D), 7.5, device="cuda")[:, :Hq]
    r = ops.attention_prefill(q, k, v, cu(q_lens), None if same else cu(kv_lens), scale=scale, out=out)
    assert r is out
    a = b = 0
    for n, m in zip(q_lens, kv_lens):
        want, bound = R.attend(q[a:a + n], k[b:b + m], v[b:b + m], R.causal(n, m), scale)
        R.check(out[a:a + n], want, bound, f"sequence of {n} tokens, {m} keys at {a}")
        a, b = a + n, b + m
    assert (out[a:] == 7.5).all()


@pytest.mark.parametrize("D", list(range(64, 513, 32)))
def test_prefill_every_head_dim(ops, D):
    prefill_case(ops, D, [5, 0, 33, 70], [5, 0, 33, 70], 6, 2, D, same=True)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (2, 1), (3, 3), (5, 1), (7, 1), (28, 4), (16, 8), (40, 8), (48, 2), (128, 1)])
def test_prefill_head_groups(ops, Hq, Hk):
    prefill_case(ops, Hq * 100 + Hk, [1, 19, 2, 66], [1, 19, 2, 66], Hq, Hk, 128)


@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1], [1]), ([1], [2000]), ([0, 0, 1], [0, 5, 1]), ([3, 4], [0, 0]), ([9, 5], [4, 5]), ([40, 1, 0, 7], [41, 300, 9, 3]),
    ([31, 32, 33], [31, 32, 33]), ([63, 64, 65], [63, 64, 65]), ([127, 128, 129], [200, 128, 129]), ([257], [257]),
    ([2] * 70, [3] * 70), ([1] * 200, list(range(200))), ([700], [1900]), ([1500], [1500]),
])
def test_prefill_lengths(ops, q_lens, kv_lens):
    prefill_case(ops, sum(q_lens) + len(kv_lens), q_lens, kv_lens, 8, 2, 128)
    prefill_case(ops, sum(q_lens) + len(kv_lens) + 1, q_lens, kv_lens, 4, 4, 64)


@pytest.mark.parametrize("sigma,scale", [(1e-30, 1e29), (1e-38, 1.0), (3e4, 1e-5), (1e30, 1e-31), (1.0, -0.3), (1.0, 0.0),
                                         (40.0, 0.1)])
def test_prefill_magnitudes(ops, sigma, scale):
    """q rows far outside binary16's range, steep softmaxes, negative and zero scales."""
    prefill_case(ops, 5, [50, 130], [50, 130], 4, 2, 128, sigma=sigma, scale=scale)


def test_prefill_hidden_rows_hold_anything(ops):
    """NaN and infinities in K/V rows that a token does not see: behind every sequence, and ahead of the token."""
    for D, G in ((128, 4), (64, 1), (256, 2), (96, 8)):
        g = gen(D)
        lens = [37, 64, 130]
        T = sum(lens)
        q, k, v = rnd(g, T, 2 * G, D), rnd(g, T + 40, 2, D, dtype=torch.float16), rnd(g, T + 40, 2, D, dtype=torch.float16)
        k[T:] = float("nan")
        v[T:] = float("inf")
        clean_k, clean_v = k.clone(), v.clone()
        a = 0
        for n in lens:  # the last keys of each sequence are seen by its last tokens only
            k[a + n - 5, 0, 3] = float("nan")
            v[a + n - 3, :, 1] = float("inf")
            v[a + n - 9, 1, D - 1] = float("nan")
            a += n
        c = i32([0, 37, 101, 231])
        out = ops.attention_prefill(q, k, v, c, c)
        a = 0
        for n in lens:
            want, bound = R.attend(q[a:a + n], clean_k[a:a + n], clean_v[a:a + n], R.causal(n, n))
            ok = n - 9  # tokens before the first touched row
            R.check(out[a:a + ok], want[:ok], bound[:ok], f"D {D}")
            # the tokens that see them: only what those elements reach is lost
            assert torch.isnan(out[a + n - 9:a + n, G:, D - 1]).all()
            assert not torch.isfinite(out[a + n - 3:a + n, :, 1]).any()
            mid = out[a + n - 9:a + n - 5, G:, :D - 1].cpu().double()
            assert ((mid - want[n - 9:n - 5, G:, :D - 1]).abs() <= bound[n - 9:n - 5, G:, :D - 1]).all()
            a += n


def test_prefill_offsets_out_of_range_stay_inside(ops):
    """Offsets that no buffer has give some rows, and touch nothing outside."""
    g = gen(9)
    q, k, v = rnd(g, 40, 4, 64), rnd(g, 50, 2, 64, dtype=torch.float16), rnd(g, 50, 2, 64, dtype=torch.float16)
    out = torch.full((44, 4, 64), 3.0, device="cuda")
    ops.attention_prefill(q, k, v, i32([-5, 20, 10, 2000000000]), i32([0, 2147483647, -7, 60]), out=out[:40])
    torch.cuda.synchronize()
    assert (out[40:] == 3.0).all() and torch.isfinite(out).all()


def test_offsets_that_do_not_rise_stay_inside(ops):
    """Sequences that overlap hold more tiles than the call has tokens for: what the scratch has no room for is left
    out, of either kernel, whole or cut in pieces."""
    g = gen(10)
    for T, S, n in ((40, 3000, 30), (600, 9000, 20), (64, 64, 50), (2000, 2000, 9)):
        q, k, v = rnd(g, T, 8, 64), rnd(g, S, 2, 64, dtype=torch.float16), rnd(g, S, 2, 64, dtype=torch.float16)
        back = [0, T] * n
        keys = [0, S] * n
        out = torch.full((T + 64, 8, 64), 3.0, device="cuda")
        ops.attention_prefill(q, k, v, i32(back + [0]), i32(keys + [0]), out=out[:T])
        torch.cuda.synchronize()
        assert (out[T:] == 3.0).all() and not torch.isnan(out).any()
    kp, vp, table, ks, vs = paged(g, [3000, 100], 64, 2, 64)
    table = table[:1].repeat(60, 1).contiguous()
    kp, vp = torch.nan_to_num(kp), torch.nan_to_num(vp)
    out = torch.full((100, 8, 64), 3.0, device="cuda")
    for T in (10, 70):
        ops.attention_tree(rnd(g, T, 8, 64), kp, vp, table, i32([2000] * 60), i32([0, T] * 30 + [0]), out=out[:T])
        torch.cuda.synchronize()
        assert (out[T:] == 3.0).all() and not torch.isnan(out).any()


def test_subnormal_rows(ops):
    """binary16 subnormals in K and V count as what they are."""
    g = gen(12)
    for n in (9, 300):
        q = rnd(g, n, 4, 128, sigma=3e4)
        k = rnd(g, n, 2, 128, sigma=1.5e-5, dtype=torch.float16)
        v = rnd(g, n, 2, 128, sigma=4e-6, dtype=torch.float16)
        out = ops.attention_prefill(q, k, v, cu([n]))
        want, bound = R.attend(q, k, v, R.causal(n, n))
        R.check(out, want, bound)


def test_prefill_past_32_bit_offsets(ops):
    """K/V rows and tokens whose element offsets pass 2^31 and 2^32."""
    g = gen(11)
    base = torch.empty((5 << 30) // 2 + 4096 * 64, dtype=torch.float16, device="cuda")  # 2^31.3 elements
    stride = 67108864  # 64 rows of 2^26 elements pass 2^32 bytes; 40 rows pass 2^31 elements
    n = base.numel() // stride
    k = base.as_strided((n, 1, 64), (stride, 64, 1), 0)
    v = base.as_strided((n, 1, 64), (stride, 64, 1), 64)
    k.copy_(rnd(g, n, 1, 64))
    v.copy_(rnd(g, n, 1, 64))
    q = rnd(g, n, 2, 64)
    out = ops.attention_prefill(q, k, v, i32([0, n]))
    want, bound = R.attend(q, k, v, R.causal(n, n))
    R.check(out, want, bound)


# ------------------------------------------------------------------------------------------------ paged, trees

def paged(g, lens, ps, H, D, spare=3, layout=0):
    """Pages of sequences of these lengths (tokens incl. the new ones) in shuffled order; unused rows hold NaN."""
    need = [-(-n // ps) for n in lens]
    P, W = sum(need) + spare, max(need + [1]) + 1
    shape = (P, ps, H, D)
    if layout == 1:  # K and V of a page side by side
        kv = torch.full((P, 2, ps, H, D), float("nan"), dtype=torch.float16, device="cuda")
        kp, vp = kv[:, 0], kv[:, 1]
    elif layout == 2:  # K and V of a token side by side
        kv = torch.full((P, ps, 2, H, D), float("nan"), dtype=torch.float16, device="cuda")
        kp, vp = kv[:, :, 0], kv[:, :, 1]
    else:
        kp, vp = (torch.full(shape, float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    ids = list(range(P))
    random.Random(P * 31 + ps).shuffle(ids)
    table = [[-1] * W for _ in lens]
    ks, vs = [], []
    for b, n in enumerate(lens):
        k, v = rnd(g, n, H, D, dtype=torch.float16), rnd(g, n, H, D, dtype=torch.float16)
        for i in range(need[b]):
            p = ids.pop()
            table[b][i] = p
            m = min(ps, n - i * ps)
            kp[p, :m] = k[i * ps:i * ps + m]
            vp[p, :m] = v[i * ps:i * ps + m]
        ks.append(k)
        vs.append(v)
    return kp, vp, i32(table), ks, vs


def tree_masks(rng, d):
    rows = []
    for i in range(d):
        parent = rng.randint(-1, i - 1)
        rows.append((rows[parent] if parent >= 0 else 0) | (1 << i))
    return rows


def tree_case(ops, seed, ctx, drafts, Hq, Hk, D, ps, mask=True, layout=0, words=1, cu_given=True, scale=None):
    g, rng = gen(seed), random.Random(seed)
    kp, vp, table, ks, vs = paged(g, [c + d for c, d in zip(ctx, drafts)], ps, Hk, D, layout=layout)
    T = sum(drafts)
    q = rnd(g, T, Hq, D)
    masks = [m for d in drafts for m in tree_masks(rng, d)]
    tm = None
    if mask:
        def word(m, w):
            x = (m >> (64 * w)) & ((1 << 64) - 1)
            return x - (1 << 64) if x >> 63 else x
        tm = torch.tensor([[word(m, w) for w in range(words)] for m in masks], dtype=torch.int64, device="cuda")
        if words == 1 and seed % 2:
            tm = tm[:, 0].contiguous()
    out = ops.attention_tree(q, kp, vp, table, i32(ctx), cu(drafts) if cu_given else None, tm, scale=scale)
    a = 0
    for b, (c, d) in enumerate(zip(ctx, drafts)):
        seen = R.causal(d, c + d)
        if mask:
            for i in range(d):
                for j in range(d):
                    seen[i, c + j] = bool(masks[a + i] >> j & 1) and j < 64 * words
        want, bound = R.attend(q[a:a + d], ks[b], vs[b], seen, scale)
        R.check(out[a:a + d], want, bound, f"sequence {b}: {c} + {d}")
        a += d


@pytest.mark.parametrize("D", list(range(64, 513, 32)))
def test_tree_every_head_dim(ops, D):
    tree_case(ops, D, [70, 0, 130], [3, 5, 1], 6, 2, D, 16)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", [0, 1, 2])
def test_tree_page_sizes_and_layouts(ops, ps, layout):
    tree_case(ops, ps + layout, [ps - 1, ps, ps + 1, 3 * ps + 5, 0], [4, 9, 1, 17, 2], 8, 2, 128, ps, layout=layout)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (3, 3), (7, 1), (28, 4), (40, 8), (64, 8), (128, 1)])
@pytest.mark.parametrize("drafts", [1, 7, 60])
def test_tree_head_groups(ops, Hq, Hk, drafts):
    tree_case(ops, Hq + drafts, [200, 31], [drafts, max(1, drafts // 2)], Hq, Hk, 128, 32)


@pytest.mark.parametrize("ctx", [[0], [1], [31], [32], [33], [511, 0, 4000], [20000], [5000, 3, 700, 9000],
                                 list(range(0, 150))])
def test_decode_lengths(ops, ctx):
    """One token per sequence; short contexts, and long ones whose keys are cut in pieces."""
    tree_case(ops, len(ctx), ctx, [1] * len(ctx), 8, 2, 128, 64, mask=False, cu_given=False)
    tree_case(ops, len(ctx) + 1, ctx, [1] * len(ctx), 4, 1, 64, 16, mask=False, cu_given=False)


@pytest.mark.parametrize("ctx,drafts", [([5000], [64]), ([0], [64]), ([777, 12], [63, 64]), ([3000, 100, 0], [0, 30, 64])])
def test_tree_long_contexts(ops, ctx, drafts):
    tree_case(ops, 3, ctx, drafts, 8, 2, 128, 64)


def test_tree_many_words(ops):
    """More than 64 drafts: two words per token; with one word, drafts from 64 on are seen by none."""
    tree_case(ops, 2, [100, 5], [100, 128], 4, 2, 64, 16, words=2)
    tree_case(ops, 4, [100, 5], [100, 70], 4, 2, 64, 16, words=1)


def test_tree_without_mask_is_a_piece_of_a_prompt(ops):
    tree_case(ops, 6, [0, 333, 64], [150, 90, 1], 8, 2, 128, 32, mask=False)


def test_tree_given_out_and_tokens_outside(ops):
    """A strided result; q rows in front of the first sequence and behind the last keep what the result held."""
    g = gen(13)
    kp, vp, table, ks, vs = paged(g, [70, 33], 32, 2, 64)
    q = rnd(g, 12, 9, 64)[:, :8]
    buf = torch.full((12, 9, 64), 5.0, device="cuda")
    out = ops.attention_tree(q, kp, vp, table, i32([66, 30]), i32([2, 6, 9]), out=buf[:, :8])
    assert out.data_ptr() == buf.data_ptr()
    for a, b, n, m in ((2, 0, 4, 70), (6, 1, 3, 33)):
        want, bound = R.attend(q[a:a + n], ks[b], vs[b], R.causal(n, m))
        R.check(out[a:a + n], want, bound)
    assert (buf[:2] == 5.0).all() and (buf[9:] == 5.0).all() and (buf[:, 8] == 5.0).all()


def test_tree_empty_rows_give_zeros(ops):
    """No context and no bit: nothing is seen."""
    g = gen(1)
    kp, vp, table, ks, vs = paged(g, [2, 40], 16, 2, 128)
    q = rnd(g, 4, 4, 128)
    mask = torch.tensor([0, 2, 0, 1], dtype=torch.int64, device="cuda")
    out = ops.attention_tree(q, kp, vp, table, i32([0, 38]), cu([2, 2]), mask)
    assert (out[0] == 0).all()
    want, bound = R.attend(q[1:2], ks[0], vs[0], torch.tensor([[False, True]]))
    R.check(out[1:2], want, bound)
    seen = torch.ones(2, 40, dtype=torch.bool)
    seen[0, 38:] = False
    seen[1, 39] = False
    want, bound = R.attend(q[2:], ks[1], vs[1], seen)
    R.check(out[2:], want, bound)


def test_tree_absent_pages(ops):
    """Keys on no page, or behind the table's last column, take no part; wild lengths stay inside."""
    g = gen(2)
    kp, vp, table, ks, vs = paged(g, [100, 100, 64], 16, 1, 64)
    table = table[:, :6].contiguous()  # 96 positions
    table[0, 2] = -1
    table[1, 0] = kp.shape[0]
    table[1, 4] = 1 << 30
    q = rnd(g, 3, 3, 64)
    out = ops.attention_tree(q, kp, vp, table, i32([80, 2147483647, -9]))
    seen = torch.zeros(1, 100, dtype=torch.bool)
    seen[0, :81] = True
    seen[0, 32:48] = False
    want, bound = R.attend(q[:1], ks[0], vs[0], seen)
    R.check(out[:1], want, bound)
    seen[:] = False
    seen[0, 16:96] = True
    seen[0, 64:80] = False
    want, bound = R.attend(q[1:2], ks[1], vs[1], seen)
    R.check(out[1:2], want, bound)
    want, bound = R.attend(q[2:], ks[2], vs[2], torch.arange(64)[None, :] < 1)
    R.check(out[2:], want, bound)
    # no pages at all, no table at all
    none = torch.empty((0, 16, 1, 64), dtype=torch.float16, device="cuda")
    assert (ops.attention_tree(q, none, none, table, i32([80, 3, 0])) == 0).all()
    assert (ops.attention_tree(q, kp, vp, table[:, :0].contiguous(), i32([80, 3, 0])) == 0).all()


def test_tree_hidden_drafts_hold_anything(ops):
    """A draft's NaN and infinite V elements reach only the drafts that see it."""
    g = gen(3)
    c, d = 50, 40
    kp, vp, table, ks, vs = paged(g, [c + d], 32, 2, 128)
    q = rnd(g, d, 8, 128)
    clean_k, clean_v = ks[0].clone(), vs[0].clone()
    page, at = int(table[0, (c + 7) // 32]), (c + 7) % 32
    kp[page, at, 0] = float("nan")
    vp[page, at, 1, 5] = float("inf")
    seen = R.causal(d, c + d)
    seen[:, c + 7] = False
    seen[7, c + 7] = True
    bits = [sum(1 << j for j in range(d) if seen[i, c + j]) for i in range(d)]
    out = ops.attention_tree(q, kp, vp, table, i32([c]), cu([d]), torch.tensor(bits, dtype=torch.int64, device="cuda"))
    want, bound = R.attend(q, clean_k, clean_v, seen)
    others = [i for i in range(d) if i != 7]
    R.check(out[others], want[others], bound[others])
    assert torch.isnan(out[7, :4]).all() and not torch.isfinite(out[7, 4:, 5]).any()


def test_tree_page_offsets_past_32_bits(ops):
    """A pool of more than 2^32 elements, read at both ends."""
    g = gen(4)
    P, ps, H, D = 16500, 256, 8, 128
    kp = torch.zeros((P, ps, H, D), dtype=torch.float16, device="cuda")
    vp = torch.zeros((P, ps, H, D), dtype=torch.float16, device="cuda")
    ids = [P - 1, 0, P - 2]
    ks, vs = rnd(g, 700, H, D, dtype=torch.float16), rnd(g, 700, H, D, dtype=torch.float16)
    for i, p in enumerate(ids):
        n = min(256, 700 - 256 * i)
        kp[p, :n], vp[p, :n] = ks[256 * i:256 * i + n], vs[256 * i:256 * i + n]
    q = rnd(g, 1, 16, D)
    out = ops.attention_tree(q, kp, vp, i32([ids]), i32([699]))
    want, bound = R.attend(q, ks, vs, torch.ones(1, 700, dtype=torch.bool))
    R.check(out, want, bound)


# ------------------------------------------------------------------------------------------------ streams, graphs

def test_attention_captured_and_replayed(ops):
    """A graph of both calls, replayed with new contents between eager calls of other sizes; two graphs at once."""
    g = gen(5)
    q = rnd(g, 90, 8, 128)
    k, v = rnd(g, 90, 2, 128, dtype=torch.float16), rnd(g, 90, 2, 128, dtype=torch.float16)
    c = cu([40, 50])
    kp, vp, table, _, _ = paged(g, [3001, 700], 64, 2, 128)
    kp, vp = torch.nan_to_num(kp), torch.nan_to_num(vp)
    lens = i32([3000, 699])
    qd = rnd(g, 2, 8, 128)

    def call():
        return ops.attention_prefill(q, k, v, c), ops.attention_tree(qd, kp, vp, table, lens)

    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = call()
        graphs.append((gr, outs))
    for i in range(4):
        q.copy_(rnd(g, 90, 8, 128))
        qd.copy_(rnd(g, 2, 8, 128))
        lens.copy_(i32([3000 - 700 * i, 699 - i]))
        want = [t.clone() for t in call()]
        for gr, _ in graphs:
            gr.replay()
        eager = ops.attention_tree(rnd(g, 1, 8, 128), kp, vp, table[:1].contiguous(), i32([50 * i]))
        torch.cuda.synchronize()
        assert torch.isfinite(eager).all()
        for _, outs in graphs:
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_attention_on_another_stream(ops):
    g = gen(6)
    q = rnd(g, 70, 8, 128)
    k, v = rnd(g, 70, 2, 128, dtype=torch.float16), rnd(g, 70, 2, 128, dtype=torch.float16)
    c = cu([70])
    want = ops.attention_prefill(q, k, v, c)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        big = torch.zeros(1 << 26, device="cuda")
        q2 = q.clone()
        for _ in range(20):
            big.add_(1.0)
        q2.add_(big[:1] - 20.0)
        got = ops.attention_prefill(q2, k, v, c)
    st.synchronize()
    assert torch.equal(got, want)


def test_attention_refusals(ops):
    g = gen(7)
    q, k, v = rnd(g, 8, 4, 64), rnd(g, 8, 2, 64, dtype=torch.float16), rnd(g, 8, 2, 64, dtype=torch.float16)
    c = cu([8])
    from v7multiplikator_amd._lib import V7GError
    with pytest.raises(TypeError):
        ops.attention_prefill(q.half(), k, v, c)
    with pytest.raises(TypeError):
        ops.attention_prefill(q, k.float(), v, c)
    with pytest.raises(TypeError):
        ops.attention_prefill(q, k, v, c.long())
    with pytest.raises(ValueError):
        ops.attention_prefill(q, k, v[:, :1], c)
    with pytest.raises(ValueError):
        ops.attention_prefill(q.transpose(0, 1), k, v, c)
    with pytest.raises(ValueError):
        ops.attention_prefill(q.cpu(), k, v, c)
    with pytest.raises(V7GError):  # 3 heads over 2
        ops.attention_prefill(q[:, :3].contiguous(), k, v, c)
    with pytest.raises(V7GError):  # fewer K/V rows without their own offsets
        ops.attention_prefill(q, k[:7], v[:7], c)
    with pytest.raises(V7GError):  # out over q
        ops.attention_prefill(q, k, v, c, out=q)
    with pytest.raises(V7GError):  # head_dim outside the contract
        ops.attention_prefill(rnd(g, 2, 4, 48), k[:2, :, :48].contiguous(), v[:2, :, :48].contiguous(), cu([2]))
    pages = torch.zeros((4, 16, 2, 64), dtype=torch.float16, device="cuda")
    t = i32([[0, 1]])
    with pytest.raises(ValueError):  # two tokens, one sequence, no offsets
        ops.attention_tree(q[:2], pages, pages, t, i32([3]))
    with pytest.raises(TypeError):
        ops.attention_tree(q[:1], pages, pages, t.long(), i32([3]))
    with pytest.raises(TypeError):
        ops.attention_tree(q[:1], pages, pages, t, i32([3]), cu([1]), i32([1]))
    with pytest.raises(ValueError):
        ops.attention_tree(q[:1], pages, pages[:3], t, i32([3]))
    with pytest.raises(V7GError):  # pages of 24 tokens
        p24 = torch.zeros((4, 24, 2, 64), dtype=torch.float16, device="cuda")
        ops.attention_tree(q[:1], p24, p24, t, i32([3]))
    assert ops.attention_prefill(q[:0], k[:0], v[:0], cu([0])).shape == (0, 4, 64)
    assert ops.attention_tree(q[:0], pages, pages, t[:0], i32([]).int()).shape == (0, 4, 64)
