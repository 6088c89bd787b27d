"""GPU: token_logprobs against 64 bits; the alternatives' ids exactly, ties to the lower index."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X")
    from v7multiplikator_amd import ops as o
    return o


def check(x, ids, K, got):
    """x [T, V] f32 on the device.  Bounds: z = x - m rounds by u|z|; e^z by 2u + u|z| (a product with log2 e and
    exp2's own step); the sums' relative error by the roundings of a chain of V/64 terms of a lane plus joins of
    relative size u each, (V/64 + 40) u on s, and the same on w with |z|-weighted terms."""
    lp, ent, tl, ti = (t.cpu() for t in got)
    xd = x.cpu().double().numpy()
    T, V = xd.shape
    m = xd.max(1, keepdims=True)
    z = xd - m
    e = np.exp(z)
    s = e.sum(1)
    p = e / s[:, None]
    zf = np.where(np.isfinite(z), z, 0.0)
    H = np.log(s) - (p * zf).sum(1)
    chain = V / 64 + 40
    per = U * (chain + (p * np.abs(zf)).sum(1) * 3 + 4)           # relative error of s
    rel_w = U * ((chain + 6) * (p * np.abs(zf)).sum(1) + 3 * (p * zf * zf).sum(1))
    lse_err = per + U * np.abs(np.log(s)) * 2
    lse = np.log(s)
    i = ids.cpu().numpy()
    ok = (i >= 0) & (i < V)
    want = np.where(ok, z[np.arange(T), np.clip(i, 0, V - 1)] - lse, np.nan)
    bound = lse_err + 4 * U * (np.abs(np.where(np.isfinite(want), want, 0)) + np.abs(lse)) + 1e-37
    g = lp.double().numpy()
    same = (g == want) | (np.isnan(g) & np.isnan(want)) | (np.abs(np.where(np.isfinite(g), g, 1e300) - np.where(np.isfinite(want), want, 0)) <= bound)
    assert same.all(), (np.nonzero(~same)[0][:5], g[~same][:5], want[~same][:5])
    eb = lse_err + rel_w + per * (p * np.abs(zf)).sum(1) + 8 * U * (H + np.abs(lse)) + 1e-37
    assert (np.abs(ent.double().numpy() - H) <= eb).all()
    assert tl.shape == (T, K) and ti.shape == (T, K) and ti.dtype == torch.int32
    for t in range(T):
        order = np.lexsort((np.arange(V), -xd[t]))[:K]  # by value, then by index
        assert ti[t].tolist() == order.tolist(), t
        w = z[t][order] - lse[t]
        b = lse_err[t] + 4 * U * (np.abs(np.where(np.isfinite(w), w, 0)) + abs(lse[t])) + 1e-37
        gv = tl[t].double().numpy()
        assert ((gv == w) | (np.abs(np.where(np.isfinite(gv), gv, 1e300) - np.where(np.isfinite(w), w, 0)) <= b)).all(), t


def run(ops, x, ids, K):
    check(x, ids, K, ops.token_logprobs(x, ids, K))


def rnd(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def some_ids(T, V, seed=0):
    return torch.randint(0, V, (T,), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda",
                         dtype=torch.int32)


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 32000, 151936, 128257])
@pytest.mark.parametrize("T,K", [(1, 0), (1, 1), (3, 5), (7, 20), (2, 64)])
def test_sizes(ops, V, T, K):
    if V > 100000 and T == 7:
        T = 4
    run(ops, rnd(V + T, T, V) * 3, some_ids(T, V), min(K, V))


@pytest.mark.parametrize("T", [500, 2047, 2048, 5000])
def test_many_rows(ops, T):
    run(ops, rnd(T, T, 777) * 2, some_ids(T, 777), 4)


def test_strides_and_offsets(ops):
    x = rnd(1, 40, 1203)
    for view in (x[:, 1:1200], x[:, 2:1203], x[::3, 5:900]):
        run(ops, view, some_ids(view.shape[0], view.shape[1]), 8)


def test_ids_outside_the_vocabulary(ops):
    run(ops, rnd(2, 4, 300), torch.tensor([-1, 300, 2147483647, 299], dtype=torch.int32, device="cuda"), 2)


def test_ties_fall_to_the_lower_index(ops):
    """Constant rows, rows of few values, and signed zeros, across lanes, waves and parts of a row."""
    for V in (64, 1500, 40000):
        x = torch.zeros(4, V, device="cuda")
        x[1] = -3.0
        x[2] = (torch.arange(V, device="cuda") % 3).float()
        x[3, ::2] = -0.0
        run(ops, x, some_ids(4, V), 40)
        y = torch.full((2, V), float("-inf"), device="cuda")
        y[0, V - 7], y[1, 3], y[1, V - 1] = 1.0, 2.0, 2.0
        run(ops, y, torch.tensor([V - 7, 0], dtype=torch.int32, device="cuda"), 30)


def test_denormals_count_as_zero(ops):
    """Denormal logits tie with 0 and -0, whatever their bits: the lower index first."""
    for V in (500, 9000):
        x = torch.full((2, V), -1.0, device="cuda")
        at = [3, 7, 70, 200, 300, V - 1]
        x[0, at] = torch.tensor([0.0, 1e-40, -1e-41, -0.0, 3e-39, 1e-45], device="cuda")
        x[1, at] = torch.tensor([-1e-45, 0.0, 1e-38, 2e-39, 0.0, 1.2e-38], device="cuda")
        ti = ops.token_logprobs(x, some_ids(2, V), 5)[3]
        assert ti[0].tolist() == at[:5]
        assert ti[1].tolist() == [V - 1, 3, 7, 70, 200]


def test_sorted_rows(ops):
    """Every step of a wave brings better candidates than all before, or none."""
    for V in (3000, 50000):
        up = torch.arange(V, device="cuda").float() * (20.0 / V)
        run(ops, torch.stack([up, up.flip(0)]), some_ids(2, V), 64)


def test_masked_logits(ops):
    """-inf and the type's lowest value, as vocabulary masks write them, and magnitudes far apart."""
    x = rnd(3, 6, 5000) * 4
    x[0, 100:] = float("-inf")
    x[1, :4900] = float("-inf")
    x[2, 1:] = -3.4028234663852886e38
    x[3] *= 1e4
    x[4] *= 1e-6
    x[5, ::2] = float("-inf")
    run(ops, x, torch.tensor([100, 4950, 0, 7, 8, 2], dtype=torch.int32, device="cuda"), 16)


def test_rows_without_probabilities(ops):
    """NaN, +inf, or nothing above -inf: every probability of the row is NaN, its neighbours' are not."""
    x = rnd(4, 5, 3000)
    x[1, 2999], x[2, 5] = float("nan"), float("inf")
    x[3] = float("-inf")
    ids = some_ids(5, 3000)
    lp, ent, tl, ti = ops.token_logprobs(x, ids, 3)
    for t in (1, 2, 3):
        assert torch.isnan(lp[t]) and torch.isnan(ent[t]) and torch.isnan(tl[t]).all()
    assert ti[1, 0] == 2999 and ti[2, 0] == 5 and ti[3].tolist() == [0, 1, 2]
    keep = [0, 4]
    check(x[keep], ids[keep], 3, tuple(t[keep] for t in (lp, ent, tl, ti)))


def test_long_rows(ops):
    """A row past 2^31 bytes in all, rows whose offsets pass 2^31 elements."""
    V = 1 << 20
    x = torch.zeros(2100, V, device="cuda")
    x[2099] = rnd(5, V)
    x[2099, 77] = 9.0
    lp, ent, tl, ti = ops.token_logprobs(x, torch.full((2100,), 77, dtype=torch.int32, device="cuda"), 2)
    check(x[2099:], torch.tensor([77], dtype=torch.int32), 2, (lp[2099:], ent[2099:], tl[2099:], ti[2099:]))
    assert ti[:2099].eq(torch.tensor([0, 1], dtype=torch.int32, device="cuda")).all()


def test_captured(ops):
    x, ids = rnd(6, 3, 30000), some_ids(3, 30000)
    ops.token_logprobs(x, ids, 5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.token_logprobs(x, ids, 5)
    for i in range(3):
        x.copy_(rnd(10 + i, 3, 30000))
        g.replay()
        torch.cuda.synchronize()
        check(x, ids, 5, out)
        run(ops, rnd(20 + i, 2, 9000), some_ids(2, 9000), 7)


def test_refusals(ops):
    from v7multiplikator_amd._lib import V7GError
    x, ids = rnd(7, 2, 50), some_ids(2, 50)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), ids)
    with pytest.raises(TypeError):
        ops.token_logprobs(x, ids.long())
    with pytest.raises(ValueError):
        ops.token_logprobs(x, ids[:1])
    with pytest.raises(ValueError):
        ops.token_logprobs(x.t(), some_ids(50, 2))
    with pytest.raises(ValueError):
        ops.token_logprobs(x, ids, 65)
    with pytest.raises(V7GError):
        ops.token_logprobs(x, ids, 51)
    with pytest.raises(V7GError):
        ops.token_logprobs(x[:, :0], ids)
    assert [t.shape for t in ops.token_logprobs(x[:0], ids[:0], 4)] == [(0,), (0,), (0, 4), (0, 4)]
