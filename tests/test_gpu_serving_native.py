"""The native path of the ops around the K/V cache against their Python bodies: the same results and returned objects
on accepted calls, which it makes itself, and the same exceptions on refused ones, which it leaves to Python."""
from __future__ import annotations

import pytest

from .test_gpu_ops_native import Recorder, outcome

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible MI355X")
    from v7multiplikator_amd import ops as o
    x = torch.ones(4, 64, device="cuda")
    o.add_inplace(x, x.clone())
    assert o._fast.__name__ == "_ops_native", "the native module is not in use"
    return o


def rnd(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape))
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prompt():
    qkv = rnd(9, 8 * 64)
    return qkv[:, :256].view(9, 4, 64), rnd(9, 2, 64, seed=1, dtype=torch.float16), rnd(9, 2, 64, seed=2, dtype=torch.float16)


def pages(layers=0):
    lead = (layers,) if layers else ()
    return rnd(*lead, 6, 16, 2, 64, seed=3, dtype=torch.float16), rnd(*lead, 6, 16, 2, 64, seed=4, dtype=torch.float16)


TABLE = [[5, 0, -1], [2, 3, -1]]
CU = [0, 4, 9]


def calls():
    out = []

    def add(name, f):
        out.append(pytest.param(name, f, id=name))

    def prefill(o, **kw):
        return o.attention_prefill(*prompt(), i32(CU), **kw)

    def prefill_given(o):
        buf = torch.zeros(9, 5, 64, device="cuda")[:, :4]
        got = prefill(o, cu_seqlens_k=i32(CU), scale=2, out=buf)
        return got, buf, got is buf

    def tree(o, T=5, **kw):
        kp, vp = pages()
        return o.attention_tree(rnd(T, 4, 64), kp, vp, i32(TABLE), i32([17, 3]), **kw)

    def pack(o, seqs=None, T=2):
        kp, vp = pages()
        rows = rnd(T, 256)
        r = o.kv_pack_f16_pages(rows[:, :128], rows[:, 128:], kp, vp, i32(TABLE), i32(list(range(T))), seqs)
        return r, kp, vp

    def assign(o, reserve=None, layers=3):
        kp, vp = pages(layers)
        return (*o.kv_pages_assign(kp, vp, i32(TABLE), i32([20, 31]), i32([1, 0, 1, 1, 0, 1]), i32([0, 0]), reserve), kp, vp)

    def compact(o, layers=3):
        kp, vp = pages(layers)
        return o.kv_pages_compact(kp, vp, i32(TABLE), i32([20, 3]), i32([[1, 3], [0, 2]]), i32([2, 2])), kp, vp

    # accepted
    add("prefill", lambda o: prefill(o))
    add("prefill_given", prefill_given)
    add("tree", lambda o: tree(o, cu_seqlens=i32([0, 3, 5]), tree_mask=torch.tensor([1, 3, 7, 1, 2], device="cuda")))
    add("tree_words", lambda o: tree(o, cu_seqlens=i32([0, 3, 5]), tree_mask=torch.ones(5, 2, dtype=torch.int64, device="cuda"),
                                     scale=0.5, out=torch.zeros(5, 4, 64, device="cuda")))
    add("decode", lambda o: tree(o, T=2))
    add("pack", lambda o: pack(o))
    add("pack_seqs", lambda o: pack(o, i32([1, 0, 1, 1]), 4))
    add("assign", lambda o: assign(o))
    add("assign_reserve", lambda o: assign(o, i32([20, 3]), 0))
    add("compact", lambda o: compact(o))
    add("compact_one_layer", lambda o: compact(o, 0))
    add("logprobs", lambda o: o.token_logprobs(rnd(3, 5000)[:, 1:4000], i32([5, 6, 7]), 6))
    add("logprobs_no_top", lambda o: o.token_logprobs(rnd(3, 50), i32([5, 6, 7])))
    add("parameter", lambda o: o.token_logprobs(torch.nn.Parameter(rnd(3, 50)).detach(), i32([5, 6, 7]), 2))
    # the library's refusals
    add("lib_heads", lambda o: o.attention_prefill(rnd(9, 3, 64), *prompt()[1:], i32(CU)))
    add("lib_alias", compact_alias)
    # refused by Python's checks
    add("py_cu_type", lambda o: o.attention_prefill(*prompt(), torch.tensor(CU, device="cuda")))
    add("py_out", lambda o: prefill(o, out=torch.zeros(9, 3, 64, device="cuda")))
    add("py_tokens", lambda o: tree(o, T=5))
    add("py_mask", lambda o: tree(o, T=2, tree_mask=i32([1, 1])))
    add("py_host", lambda o: o.token_logprobs(rnd(3, 50).cpu(), i32([1, 2, 3])))
    add("py_top", lambda o: o.token_logprobs(rnd(3, 50), i32([1, 2, 3]), 70))
    add("py_table", lambda o: o.kv_pages_compact(*pages(), i32([0]), i32([1]), i32([[1]]), i32([1])))
    add("py_strides", lambda o: o.kv_pages_compact(pages()[0], pages()[1].transpose(1, 2).contiguous().transpose(1, 2),
                                                   i32(TABLE), i32([1, 1]), i32([[1], [1]]), i32([1, 1])))
    add("py_rows", lambda o: o.kv_pack_f16_pages(rnd(2, 64), rnd(2, 64), *pages(), i32(TABLE), i32([0, 1])))
    add("py_refs", lambda o: o.kv_pages_assign(*pages(), i32(TABLE), i32([1, 1]), i32([1]), i32([0, 1])))
    return out


def compact_alias(o):
    kp, _ = pages()
    return o.kv_pages_compact(kp, kp, i32(TABLE), i32([20, 3]), i32([[1, 3], [0, 2]]), i32([2, 2]))


@pytest.mark.parametrize("name,f", calls())
def test_native_is_the_python_path(ops, monkeypatch, name, f):
    rec = Recorder(ops._fast)
    monkeypatch.setattr(ops, "_fast", rec)
    native = outcome(f, ops)
    assert rec.made == [not name.startswith("py_")]
    monkeypatch.setattr(ops, "_fast", ops._NoNative())
    python = outcome(f, ops)
    assert len(native) == len(python)
    for a, b in zip(native, python):
        if isinstance(b, torch.Tensor):
            assert type(a) is type(b) and a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride()
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        else:
            assert a == b
    if name.startswith(("lib_", "py_")):
        assert isinstance(native[0], type)  # an exception


def test_follows_the_current_stream(ops):
    """Every op runs on the stream that is current: its inputs are only ready there."""
    st = torch.cuda.Stream()
    q, k, v = prompt()
    kp, vp = pages()
    x = rnd(2, 3000)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        big = torch.zeros(1 << 26, device="cuda")
        for _ in range(30):
            big.add_(1.0)
        late = big[:1] - 30.0  # 0, once the stream gets there
        q2, x2, kp2 = q + late, x + late, kp + late.half()
        got = (ops.attention_prefill(q2, k, v, i32(CU)), ops.token_logprobs(x2, i32([1, 2]), 2)[2],
               ops.attention_tree(q2[:2], kp2, vp, i32(TABLE), i32([17, 3])))
    st.synchronize()
    want = (ops.attention_prefill(q, k, v, i32(CU)), ops.token_logprobs(x, i32([1, 2]), 2)[2],
            ops.attention_tree(q[:2], kp, vp, i32(TABLE), i32([17, 3])))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
