"""Torch-facing host API of the fused per-layer kernels.

Mirrors the reference's kernel entry points (src/v7_lib.h:113-128,269-281) for
batched device tensors.  Every function validates its tensors, binds the
library to torch's current stream and makes ONE call through the C ABI of
libv7g.so; nothing runs on the CPU and there is no fallback: without the built
library the first call raises.

  fused_add_rmsnorm  <- v7s_fused_add_rmsnorm   (src/asm/add_rmsnorm_kernel.inc:15-129)
  rmsnorm            <- v7s_rmsnorm             (src/asm/rmsnorm_kernel.inc:12-75)
  rmsnorm_quantize   <- v7s_rmsnorm_quantize    (src/asm/rmsnorm_quantize_kernel.inc:62-218)
  add_rmsnorm_quantize <- v7s_add_inplace then v7s_rmsnorm_quantize, one pass (src/asm/forward_q8.inc:386-387)
  add_inplace        <- v7s_add_inplace         (src/asm/add_kernel.inc:26-49)
  rmsnorm_rope_heads <- v7s_rmsnorm_rope_heads  (src/asm/rmsnorm_rope_dispatch.inc:11-52)
  qk_rmsnorm_rope    <- v7s_qk_fork_heads, both sides in one launch (src/asm/qk_fork_kernel.inc:40-62)
  swiglu             <- .pq_ffn_silu            (src/asm/prefill_q8.inc:1159-1166)
  quantize_q8        <- v7d_quantize            (src/asm/utility_dispatch.inc:108-212)
  swiglu_q8          <- SwiGLU then v7d_quantize (src/asm/prefill_q8.inc:1154-1183)
  embedding_gather_q8 <- v7s_embedding_row      (src/asm/forward.inc:13-42)
  rope_tables        <- v7s_rope_init           (src/asm/fused_dispatch.inc:58-76; Llama 3 scaling
                                                  src/asm/fused_f32_kernel.inc:149-256)
  kv_pack_f16        <- v7s_kv_pack_f16         (src/asm/kv_f16c.inc:12-52)
  kv_pack_f16_kv     <- v7s_kv_pack_f16 for K then V (src/asm/forward_q8.inc:345-358), one launch
  rope_only_heads    <- v7s_rope_only_heads     (src/asm/rope_only_dispatch.inc:11-47)
  qkv_rope_stage     <- the per-token Q/K/V stage of the prefill, one launch (src/asm/prefill_q8.inc:848-883)

Around the K/V cache, with no reference export of these forms (a call makes one launch, or a few where pieces are
joined): attention_prefill, attention_tree, kv_pack_f16_pages, kv_pages_assign, kv_pages_compact, token_logprobs.
"""
from __future__ import annotations

import ctypes
import importlib.util
import math
import os
import sys

import torch

from . import _lib

Q8_EMBED_GS = 64  # scale group of the Q8 embedding table (src/asm/forward.inc:14, GS=64)


# torch's current stream of a device as a raw handle: the query torch's own generated code makes (about 0.1 us
# per call, against about 2 us for torch.cuda.current_stream(), which builds a Stream object); the public call
# where this torch lacks it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def current_stream_handle(device: torch.device) -> int:
    """The hipStream_t of torch's current stream on `device`.  If the raw query rejects its argument (a torch
    that changed its signature), the public call takes over for the rest of the process."""
    global _raw_stream
    if _raw_stream is not None:
        try:
            return _raw_stream(device.index)
        except (TypeError, RuntimeError):
            _raw_stream = None
    return torch.cuda.current_stream(device).cuda_stream


# The accepted calls run in native/ops_native.cpp (built as _ops_native.so), which makes the checks below on the
# tensors themselves and the launch in one C call, and answers None, having done nothing, for every call that it does
# not accept; the Python bodies below then check, raise or launch.  Host time per call on the 16-core host of one
# MI355X, back to back, Python bodies against native: fused_add_rmsnorm 6.4 -> 3.0 us (7.3 -> 3.9 allocating its result),
# add_rmsnorm_quantize allocating 10.5 -> 4.8, qk_rmsnorm_rope 9.7 -> 3.1, qkv_rope_stage 14.1 -> 3.3; the library call
# itself takes 2.5-3.1.
_NATIVE_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_ops_native.so")


class _NoNative:
    """Stands in where the module is not built or cannot be used: no call is accepted."""

    def __getattr__(self, name):
        return lambda *args: None


class _Unbound:
    """Binds the module at the first call (not at import: the library may not be built yet)."""

    def __getattr__(self, name):
        global _fast
        try:
            L = _lib.load()
        except (RuntimeError, OSError, AttributeError):  # the Python body meets it again, after its own checks
            return lambda *args: None
        _fast = _bind_native(L)
        return getattr(_fast, name)


def torch_build() -> str:
    """Which torch and Python: the module reads tensors through the headers of the one that it was built against."""
    return (f"{torch.__version__} {torch.version.git_version} "
            f"{sys.implementation.name}-{sys.version_info[0]}.{sys.version_info[1]}")


def _bind_native(L):
    """The module, or no native path where it is not there, does not load, or was built for another torch or Python
    or with another include/v7g_lib.h than L: neither tensors nor the library may then be read through it."""
    device = getattr(torch._C, "_cuda_getDevice", None)
    if _raw_stream is None or device is None or not os.path.exists(_NATIVE_PATH):
        return _NoNative()
    spec = importlib.util.spec_from_file_location("_ops_native", _NATIVE_PATH)
    try:
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    except ImportError:  # a symbol that this torch does not have
        return _NoNative()
    if (getattr(mod, "torch_build", None), getattr(mod, "header_tag", None)) != (torch_build(),
                                                                                 L.v7g_header_tag().decode()):
        return _NoNative()
    mod.bind({n: ctypes.cast(getattr(L, n), ctypes.c_void_p).value for n in _lib.SIGNATURES}, _raw_stream, device,
             _lib.check)
    return mod


_fast = _Unbound()


def _bind(t: torch.Tensor) -> None:
    """Binds the calling thread's library stream to torch's current stream of t's device."""
    if not t.is_cuda:
        raise ValueError("v7g kernels take device tensors (cuda:N)")
    _lib.load().v7g_set_stream(current_stream_handle(t.device))


def _need(t: torch.Tensor, dtype, name: str, contiguous: bool = True) -> None:
    """Every tensor of a call lives on the current device, where the library launches."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a cuda device")
    cur = torch.cuda.current_device()
    if t.device.index != cur:
        raise ValueError(f"{name} is on {t.device} but the current device is cuda:{cur}; "
                         f"call under torch.cuda.device({t.device})")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def fused_add_rmsnorm(residual: torch.Tensor, add: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """residual += add (in place); returns out = rmsnorm(residual) * weight.  [rows, dim] f32."""
    r = _fast.fused_add_rmsnorm(residual, add, weight, eps, out)
    if r is not None:
        return r
    for t, n in ((residual, "residual"), (add, "add"), (weight, "weight")):
        _need(t, torch.float32, n)
    dim = residual.shape[-1]
    rows = residual.numel() // dim if dim else 0
    if add.shape != residual.shape or weight.numel() != dim:
        raise ValueError("shape mismatch: add must match residual, weight must be [dim]")
    if out is None:
        out = torch.empty_like(residual)
    _need(out, torch.float32, "out")
    if out.shape != residual.shape:
        raise ValueError("out must match residual")
    _bind(residual)
    rc = _lib.load().v7g_fused_add_rmsnorm(out.data_ptr(), residual.data_ptr(), add.data_ptr(), weight.data_ptr(),
                                           rows, dim, float(eps))
    _lib.check(rc, "fused_add_rmsnorm")
    return out


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """out = rmsnorm(x) * weight per row of x [rows, dim] (dim % 32 == 0); out may be x."""
    r = _fast.rmsnorm(x, weight, eps, out)
    if r is not None:
        return r
    _need(x, torch.float32, "x")
    _need(weight, torch.float32, "weight")
    dim = x.shape[-1]
    if weight.numel() != dim:
        raise ValueError("weight must be [dim]")
    if out is None:
        out = torch.empty_like(x)
    _need(out, torch.float32, "out")
    if out.shape != x.shape:
        raise ValueError("out must match x")
    _bind(x)
    rc = _lib.load().v7g_rmsnorm(out.data_ptr(), x.data_ptr(), weight.data_ptr(), x.numel() // dim if dim else 0, dim,
                                 float(eps))
    _lib.check(rc, "rmsnorm")
    return out


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, gs: int = 64,
                     out_q: torch.Tensor | None = None, out_s: torch.Tensor | None = None):
    """RMSNorm then Q8 per row of x [rows, dim]: returns (codes int8 like x, scales [rows, dim/gs])."""
    r = _fast.rmsnorm_quantize(x, weight, eps, gs, out_q, out_s)
    if r is not None:
        return r
    _need(x, torch.float32, "x")
    _need(weight, torch.float32, "weight")
    dim = x.shape[-1]
    if weight.numel() != dim:
        raise ValueError("weight must be [dim]")
    rows, out_q, out_s = _q8_out(x.shape, dim, gs, x.device, out_q, out_s)
    _bind(x)
    rc = _lib.load().v7g_rmsnorm_quantize(out_q.data_ptr(), out_s.data_ptr(), x.data_ptr(), weight.data_ptr(), rows,
                                          dim, int(gs), float(eps))
    _lib.check(rc, "rmsnorm_quantize")
    return out_q, out_s


def add_rmsnorm_quantize(residual: torch.Tensor, add: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                         gs: int = 64, out_q: torch.Tensor | None = None, out_s: torch.Tensor | None = None):
    """residual += add (in place), then RMSNorm -> Q8 of the updated rows: returns (codes, scales)."""
    r = _fast.add_rmsnorm_quantize(residual, add, weight, eps, gs, out_q, out_s)
    if r is not None:
        return r
    for t, n in ((residual, "residual"), (add, "add"), (weight, "weight")):
        _need(t, torch.float32, n)
    dim = residual.shape[-1]
    if add.shape != residual.shape or weight.numel() != dim:
        raise ValueError("shape mismatch: add must match residual, weight must be [dim]")
    rows, out_q, out_s = _q8_out(residual.shape, dim, gs, residual.device, out_q, out_s)
    _bind(residual)
    rc = _lib.load().v7g_add_rmsnorm_quantize(out_q.data_ptr(), out_s.data_ptr(), residual.data_ptr(), add.data_ptr(),
                                              weight.data_ptr(), rows, dim, int(gs), float(eps))
    _lib.check(rc, "add_rmsnorm_quantize")
    return out_q, out_s


def add_inplace(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """x += y elementwise (v7s_add_inplace); returns x."""
    r = _fast.add_inplace(x, y)
    if r is not None:
        return r
    _need(x, torch.float32, "x")
    _need(y, torch.float32, "y")
    if x.shape != y.shape:
        raise ValueError("x and y must have the same shape")
    _bind(x)
    _lib.check(_lib.load().v7g_add_inplace(x.data_ptr(), y.data_ptr(), x.numel()), "add_inplace")
    return x


def _heads_view(buf: torch.Tensor, name: str):
    """[T, H, D] view with unit stride inside a token's heads; returns (T, H, D, token_stride)."""
    if buf.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    T, H, D = buf.shape
    if buf.stride(2) != 1 or buf.stride(1) != D:
        raise ValueError(f"{name}: heads of one token must be contiguous")
    return T, H, D, buf.stride(0)


def _tables(cos_table: torch.Tensor, sin_table: torch.Tensor) -> None:
    for t, n in ((cos_table, "cos_table"), (sin_table, "sin_table")):
        _need(t, torch.float32, n)
    if cos_table.dim() != 2 or sin_table.shape != cos_table.shape:
        raise ValueError("cos_table and sin_table must both be [positions, rope_max_dim]")


def _head_weight(w: torch.Tensor, D: int, name: str) -> None:
    _need(w, torch.float32, name)
    if w.numel() != D:
        raise ValueError(f"{name} must hold head_dim = {D} floats")


def _positions(positions, T, device):
    if positions is None:
        return 0
    _need(positions, torch.int32, "positions")
    if positions.numel() != T:
        raise ValueError("positions must hold one int32 per token")
    return positions.data_ptr()


def rmsnorm_rope_heads(buf: torch.Tensor, norm_weight: torch.Tensor, cos_table: torch.Tensor,
                       sin_table: torch.Tensor, positions: torch.Tensor | None = None, pos0: int = 0,
                       eps: float = 1e-6) -> torch.Tensor:
    """In-place per-head RMSNorm + RoPE of buf [T, H, D] (token stride free); tables [P, rope_max_dim]."""
    r = _fast.rmsnorm_rope_heads(buf, norm_weight, cos_table, sin_table, positions, pos0, eps)
    if r is not None:
        return r
    _need(buf, torch.float32, "buf", contiguous=False)
    _tables(cos_table, sin_table)
    T, H, D, ts = _heads_view(buf, "buf")
    _head_weight(norm_weight, D, "norm_weight")
    _bind(buf)
    rc = _lib.load().v7g_rmsnorm_rope_heads(buf.data_ptr(), T, ts, H, D, norm_weight.data_ptr(),
                                            cos_table.data_ptr(), sin_table.data_ptr(),
                                            _positions(positions, T, buf.device), int(pos0), cos_table.shape[-1],
                                            cos_table.shape[0], float(eps))
    _lib.check(rc, "rmsnorm_rope_heads")
    return buf


def qk_rmsnorm_rope(q: torch.Tensor, k: torch.Tensor, q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor,
                    cos_table: torch.Tensor, sin_table: torch.Tensor, positions: torch.Tensor | None = None,
                    pos0: int = 0, eps: float = 1e-6, k_cache: torch.Tensor | None = None,
                    keep_k_f32: bool = True) -> None:
    """In-place RMSNorm+RoPE of Q [T, Hq, D] and K [T, Hk, D] in one launch.

    With k_cache (float16 [T, Hk, D], heads of a token contiguous, token stride free), the rotated K heads
    are also written there as binary16 (v7s_kv_pack_f16 fused); keep_k_f32=False leaves K's f32 storage
    untouched."""
    if k_cache is None and _fast.qk_rmsnorm_rope(q, k, q_norm_weight, k_norm_weight, cos_table, sin_table, positions,
                                                 pos0, eps):
        return
    for t, n in ((q, "q"), (k, "k")):
        _need(t, torch.float32, n, contiguous=False)
    _tables(cos_table, sin_table)
    T, Hq, D, qs = _heads_view(q, "q")
    Tk, Hk, Dk, ks = _heads_view(k, "k")
    if Tk != T or Dk != D:
        raise ValueError("q and k must have the same tokens and head_dim")
    _head_weight(q_norm_weight, D, "q_norm_weight")
    _head_weight(k_norm_weight, D, "k_norm_weight")
    _bind(q)
    if k_cache is None:
        rc = _lib.load().v7g_qk_rmsnorm_rope(q.data_ptr(), qs, Hq, q_norm_weight.data_ptr(), k.data_ptr(), ks, Hk,
                                             k_norm_weight.data_ptr(), T, D, cos_table.data_ptr(),
                                             sin_table.data_ptr(), _positions(positions, T, q.device), int(pos0),
                                             cos_table.shape[-1], cos_table.shape[0], float(eps))
        _lib.check(rc, "qk_rmsnorm_rope")
        return
    _need(k_cache, torch.float16, "k_cache", contiguous=False)
    Tc, Hc, Dc, cs = _heads_view(k_cache, "k_cache")
    if (Tc, Hc, Dc) != (T, Hk, D):
        raise ValueError("k_cache must be [tokens, kv_heads, head_dim]")
    rc = _lib.load().v7g_qk_rmsnorm_rope_kv(q.data_ptr(), qs, Hq, q_norm_weight.data_ptr(), k.data_ptr(), ks, Hk,
                                            k_norm_weight.data_ptr(), T, D, cos_table.data_ptr(),
                                            sin_table.data_ptr(), _positions(positions, T, q.device), int(pos0),
                                            cos_table.shape[-1], cos_table.shape[0], float(eps),
                                            k_cache.data_ptr(), cs, int(bool(keep_k_f32)))
    _lib.check(rc, "qk_rmsnorm_rope_kv")


def swiglu(gate: torch.Tensor, up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out = (sigmoid(gate)*gate)*up, f32 elementwise; out may be gate (in place)."""
    r = _fast.swiglu(gate, up, out)
    if r is not None:
        return r
    _need(gate, torch.float32, "gate")
    _need(up, torch.float32, "up")
    if up.shape != gate.shape:
        raise ValueError("gate and up must have the same shape")
    if out is None:
        out = torch.empty_like(gate)
    _need(out, torch.float32, "out")
    if out.shape != gate.shape:
        raise ValueError("out must match gate")
    _bind(gate)
    rc = _lib.load().v7g_swiglu_f32(out.data_ptr(), gate.data_ptr(), up.data_ptr(), gate.numel())
    _lib.check(rc, "swiglu")
    return out


def _q8_out(shape, row_len, gs, device, out_q, out_s):
    rows = 1
    for d in shape[:-1]:
        rows *= d
    spr = -(-row_len // gs)
    if out_q is None:
        out_q = torch.empty(shape, dtype=torch.int8, device=device)
    if out_s is None:
        out_s = torch.empty((rows, spr), dtype=torch.float32, device=device)
    _need(out_q, torch.int8, "out_q")
    _need(out_s, torch.float32, "out_s")
    if out_q.numel() != rows * row_len or out_s.numel() != rows * spr:
        raise ValueError("output buffers have the wrong size")
    return rows, out_q, out_s


def swiglu_q8(gate: torch.Tensor, up: torch.Tensor, gs: int = 32, out_q: torch.Tensor | None = None,
              out_s: torch.Tensor | None = None):
    """SwiGLU then Q8 block quantization per row: returns (codes int8 like gate, scales [rows, hidden/gs])."""
    r = _fast.swiglu_q8(gate, up, gs, out_q, out_s)
    if r is not None:
        return r
    _need(gate, torch.float32, "gate")
    _need(up, torch.float32, "up")
    if up.shape != gate.shape:
        raise ValueError("gate and up must have the same shape")
    hidden = gate.shape[-1]
    rows, out_q, out_s = _q8_out(gate.shape, hidden, gs, gate.device, out_q, out_s)
    _bind(gate)
    rc = _lib.load().v7g_swiglu_q8(out_q.data_ptr(), out_s.data_ptr(), gate.data_ptr(), up.data_ptr(), rows, hidden,
                                   int(gs))
    _lib.check(rc, "swiglu_q8")
    return out_q, out_s


def quantize_q8(x: torch.Tensor, gs: int = 64, out_q: torch.Tensor | None = None,
                out_s: torch.Tensor | None = None):
    """v7d_quantize per row of x [..., row_len]: returns (codes, scales [rows, ceil(row_len/gs)])."""
    r = _fast.quantize_q8(x, gs, out_q, out_s)
    if r is not None:
        return r
    _need(x, torch.float32, "x")
    row_len = x.shape[-1]
    rows, out_q, out_s = _q8_out(x.shape, row_len, gs, x.device, out_q, out_s)
    _bind(x)
    rc = _lib.load().v7g_quantize_q8(out_q.data_ptr(), out_s.data_ptr(), x.data_ptr(), rows, row_len, int(gs))
    _lib.check(rc, "quantize_q8")
    return out_q, out_s


def embedding_gather_q8(ids: torch.Tensor, table_q: torch.Tensor, table_s: torch.Tensor,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = dequant(table row ids[t]); table_q [vocab, dim] int8, table_s [vocab*dim/64] f32."""
    r = _fast.embedding_gather_q8(ids, table_q, table_s, out)
    if r is not None:
        return r
    _need(ids, torch.int32, "ids")
    _need(table_q, torch.int8, "table_q")
    _need(table_s, torch.float32, "table_s")
    if table_q.dim() != 2:
        raise ValueError("table_q must be [vocab, dim]")
    vocab, dim = table_q.shape
    if table_s.numel() != vocab * dim // Q8_EMBED_GS:
        raise ValueError("table_s must hold vocab*dim/64 scales")
    n = ids.numel()
    if out is None:
        out = torch.empty((n, dim), dtype=torch.float32, device=ids.device)
    _need(out, torch.float32, "out")
    if out.numel() != n * dim:
        raise ValueError("out must hold [ids, dim] floats")
    _bind(ids)
    rc = _lib.load().v7g_embedding_gather_q8(out.data_ptr(), ids.data_ptr(), n, table_q.data_ptr(),
                                             table_s.data_ptr(), dim, vocab)
    _lib.check(rc, "embedding_gather_q8")
    return out


def rope_only_heads(buf: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor,
                    positions: torch.Tensor | None = None, pos0: int = 0) -> torch.Tensor:
    """In-place RoPE (no per-head norm) of buf [T, H, D]; tables [P, rope_max_dim]."""
    r = _fast.rope_only_heads(buf, cos_table, sin_table, positions, pos0)
    if r is not None:
        return r
    _need(buf, torch.float32, "buf", contiguous=False)
    _tables(cos_table, sin_table)
    T, H, D, ts = _heads_view(buf, "buf")
    _bind(buf)
    rc = _lib.load().v7g_rope_only_heads(buf.data_ptr(), T, ts, H, D, cos_table.data_ptr(), sin_table.data_ptr(),
                                         _positions(positions, T, buf.device), int(pos0), cos_table.shape[-1],
                                         cos_table.shape[0])
    _lib.check(rc, "rope_only_heads")
    return buf


def _side(buf, norm_weight, bias, cache, keep, name):
    side = _lib.QkvSide()
    if buf is None:
        return side, None
    _need(buf, torch.float32, name, contiguous=False)
    T, H, D, ts = _heads_view(buf, name)
    side.buf, side.token_stride, side.n_heads, side.keep_f32 = buf.data_ptr(), ts, H, int(bool(keep))
    if norm_weight is not None:
        _head_weight(norm_weight, D, f"{name} norm_weight")
        side.norm_weight = norm_weight.data_ptr()
    if bias is not None:
        _need(bias, torch.float32, f"{name} bias")
        if bias.numel() != H * D:
            raise ValueError(f"{name} bias must hold heads*head_dim floats")
        side.bias = bias.data_ptr()
    if cache is not None:
        _need(cache, torch.float16, f"{name} cache", contiguous=False)
        Tc, Hc, Dc, cs = _heads_view(cache, f"{name} cache")
        if (Tc, Hc, Dc) != (T, H, D):
            raise ValueError(f"{name} cache must be [tokens, heads, head_dim]")
        side.cache, side.cache_stride = cache.data_ptr(), cs
    return side, (T, D)


def qkv_rope_stage(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, cos_table: torch.Tensor,
                   sin_table: torch.Tensor, positions: torch.Tensor | None = None, pos0: int = 0, eps: float = 1e-6,
                   q_norm_weight=None, k_norm_weight=None, q_bias=None, k_bias=None, v_bias=None, k_cache=None,
                   v_cache=None, keep_k_f32: bool = True, keep_v_f32: bool = True) -> None:
    """The Q/K/V stage of a prefill over T tokens in one launch: bias add (optional, per side), Q and K
    RMSNorm+RoPE (norm weight given) or RoPE only, binary16 K/V cache rows (optional); all in place."""
    r = _fast.qkv_rope_stage(q, k, v, cos_table, sin_table, positions, pos0, eps, q_norm_weight, k_norm_weight, q_bias,
                             k_bias, v_bias, k_cache, v_cache, keep_k_f32, keep_v_f32)
    if r is not None:
        return
    _tables(cos_table, sin_table)
    st = _lib.QkvStage()
    st.q, shq = _side(q, q_norm_weight, q_bias, None, True, "q")
    st.k, shk = _side(k, k_norm_weight, k_bias, k_cache, keep_k_f32, "k")
    st.v, shv = _side(v, None, v_bias, v_cache, keep_v_f32, "v")
    if shq != shk or (shv is not None and shv != shq):
        raise ValueError("q, k (and v) must have the same tokens and head_dim")
    T, D = shq
    st.n_tokens, st.head_dim = T, D
    st.cos_table, st.sin_table = cos_table.data_ptr(), sin_table.data_ptr()
    st.positions = _positions(positions, T, q.device) or None
    st.pos0, st.rope_max_dim, st.table_rows, st.eps = int(pos0), cos_table.shape[-1], cos_table.shape[0], float(eps)
    _bind(q)
    _lib.check(_lib.load().v7g_qkv_rope_stage(ctypes.addressof(st)), "qkv_rope_stage")


def kv_pack_f16(src: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """binary16 copy (round to nearest even) of src [rows, row_len] f32; row strides free (row_len % 4 == 0)."""
    r = _fast.kv_pack_f16(src, out)
    if r is not None:
        return r
    _need(src, torch.float32, "src", contiguous=False)
    if src.dim() != 2 or src.stride(1) != 1:
        raise ValueError("src must be [rows, row_len] with contiguous rows")
    rows, n = src.shape
    if out is None:
        out = torch.empty((rows, n), dtype=torch.float16, device=src.device)
    _need(out, torch.float16, "out", contiguous=False)
    if out.shape != src.shape or out.stride(1) != 1:
        raise ValueError("out must be [rows, row_len] with contiguous rows")
    _bind(src)
    rc = _lib.load().v7g_kv_pack_f16(out.data_ptr(), out.stride(0), src.data_ptr(), src.stride(0), rows, n)
    _lib.check(rc, "kv_pack_f16")
    return out


def kv_pack_f16_kv(k_src: torch.Tensor, v_src: torch.Tensor, k_out: torch.Tensor | None = None,
                   v_out: torch.Tensor | None = None):
    """binary16 copies of the K and V rows [rows, row_len] (views into one fused QKV buffer: the same row
    stride) in one launch; returns (k_out, v_out)."""
    r = _fast.kv_pack_f16_kv(k_src, v_src, k_out, v_out)
    if r is not None:
        return r
    _need(k_src, torch.float32, "k_src", contiguous=False)
    _need(v_src, torch.float32, "v_src", contiguous=False)
    if k_src.dim() != 2 or k_src.stride(1) != 1 or v_src.shape != k_src.shape or v_src.stride() != k_src.stride():
        raise ValueError("k_src and v_src must be [rows, row_len] with contiguous rows and the same row stride")
    rows, n = k_src.shape
    outs = []
    for o in (k_out, v_out):
        if o is None:
            o = torch.empty((rows, n), dtype=torch.float16, device=k_src.device)
        _need(o, torch.float16, "out", contiguous=False)
        if o.shape != k_src.shape or o.stride(1) != 1:
            raise ValueError("outputs must be [rows, row_len] with contiguous rows")
        outs.append(o)
    _bind(k_src)
    rc = _lib.load().v7g_kv_pack_f16_kv(outs[0].data_ptr(), outs[0].stride(0), outs[1].data_ptr(), outs[1].stride(0),
                                        k_src.data_ptr(), v_src.data_ptr(), k_src.stride(0), rows, n)
    _lib.check(rc, "kv_pack_f16_kv")
    return outs[0], outs[1]


def rope_tables(n_pos: int, head_dim: int, rope_base: float, device="cuda", llama3: dict | None = None):
    """Device cos/sin tables [n_pos, head_dim/2] (freq_j = base^(-j/half)), built on the host.

    llama3: the Llama 3 frequency scaling (rope type 1), a dict with factor, low_freq_factor,
    high_freq_factor and original_max_position_embeddings."""
    half = head_dim // 2
    c = torch.empty((n_pos, half), dtype=torch.float32, device=device)
    s = torch.empty((n_pos, half), dtype=torch.float32, device=device)
    torch.cuda.synchronize(c.device)
    L = _lib.load()
    if llama3 is None:
        rc = L.v7g_build_rope_tables(c.data_ptr(), s.data_ptr(), n_pos, head_dim, float(rope_base))
    else:
        rc = L.v7g_build_rope_tables_llama3(c.data_ptr(), s.data_ptr(), n_pos, head_dim, float(rope_base),
                                            float(llama3["factor"]), float(llama3["low_freq_factor"]),
                                            float(llama3["high_freq_factor"]),
                                            int(llama3["original_max_position_embeddings"]))
    _lib.check(rc, "rope_tables")
    return c, s


# ---------------------------------------------------------------- around the K/V cache

def _workspace(n: int, device):
    """Scratch of one call from torch's allocator: ordered on the stream the call runs on, and a captured graph's own."""
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _scale(scale, head_dim):
    return 1.0 / math.sqrt(head_dim) if scale is None else float(scale)


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                      cu_seqlens_k: torch.Tensor | None = None, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed sequences with grouped heads, out = softmax(q k^T * scale) v in f32.

    q [T, Hq, D] f32 and k, v [S, Hk, D] float16 (heads of a token contiguous, token strides free).  Sequence b has
    the tokens cu_seqlens[b] .. cu_seqlens[b+1]-1 of q and the rows cu_seqlens_k[b] .. of k and v (int32 on the
    device; None: the same as cu_seqlens); its token i of n sees its first i + 1 + m - n rows of m.  scale defaults
    to 1/sqrt(D).  A token that sees nothing gives zeros; tokens of out behind the last sequence are left as they
    were."""
    r = _fast.attention_prefill(q, k, v, cu_seqlens, cu_seqlens_k, scale, out)
    if r is not None:
        return r
    _need(q, torch.float32, "q", contiguous=False)
    T, Hq, D, qs = _heads_view(q, "q")
    for t, n in ((k, "k"), (v, "v")):
        _need(t, torch.float16, n, contiguous=False)
    S, Hk, Dk, ks = _heads_view(k, "k")
    Sv, Hv, Dv, vs = _heads_view(v, "v")
    if (Sv, Hv, Dv) != (S, Hk, Dk) or Dk != D:
        raise ValueError("k and v must both be [kv_tokens, kv_heads, head_dim] with q's head_dim")
    _need(cu_seqlens, torch.int32, "cu_seqlens")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must hold n_seqs + 1 offsets")
    if cu_seqlens_k is not None:
        _need(cu_seqlens_k, torch.int32, "cu_seqlens_k")
        if cu_seqlens_k.shape != cu_seqlens.shape:
            raise ValueError("cu_seqlens_k must match cu_seqlens")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=torch.float32, device=q.device)
    _need(out, torch.float32, "out", contiguous=False)
    To, Ho, Do, os_ = _heads_view(out, "out")
    if (To, Ho, Do) != (T, Hq, D):
        raise ValueError("out must match q")
    L = _lib.load()
    n_seqs = cu_seqlens.numel() - 1
    ws = _workspace(L.v7g_attention_prefill_workspace(n_seqs, T, S, Hq, Hk, D), q.device)
    _bind(q)
    rc = L.v7g_attention_prefill(out.data_ptr(), os_, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs,
                                 cu_seqlens.data_ptr(), _ptr(cu_seqlens_k), n_seqs, T, S, Hq, Hk, D,
                                 _scale(scale, D), _ptr(ws), 0 if ws is None else ws.numel())
    _lib.check(rc, "attention_prefill")
    return out


def _kv_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, layered: bool) -> _lib.KvPages:
    """v7g_kv_pages of the pages [n_pages, page_size, Hk, D] of one layer, or with `layered` also
    [layers, n_pages, page_size, Hk, D]; the K and V pages share their strides."""
    for t, n in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        _need(t, torch.float16, n, contiguous=False)
    if k_pages.dim() != 4 and not (layered and k_pages.dim() == 5):
        raise ValueError("k_pages must be [n_pages, page_size, kv_heads, head_dim]" +
                         (" or [layers, ...]" if layered else ""))
    if v_pages.shape != k_pages.shape or v_pages.stride() != k_pages.stride():
        raise ValueError("v_pages must have the shape and strides of k_pages")
    P, ps, H, D = k_pages.shape[-4:]
    st = k_pages.stride()
    if st[-1] != 1 or (H > 1 and st[-2] != D):
        raise ValueError("heads of one token must be contiguous in the pages")
    g = _lib.KvPages()
    g.k, g.v = k_pages.data_ptr() or None, v_pages.data_ptr() or None
    g.n_layers, g.layer_stride = (k_pages.shape[0], st[0]) if k_pages.dim() == 5 else (1, 0)
    g.n_pages, g.page_size, g.n_kv_heads, g.head_dim = P, ps, H, D
    g.page_stride, g.token_stride = st[-4], st[-3]
    return g


def _table(block_table, rows, name="block_table"):
    _need(block_table, torch.int32, name)
    if block_table.dim() != 2 or (rows is not None and block_table.shape[0] != rows):
        raise ValueError(f"{name} must be [sequences, pages per sequence]")


def _rows_i32(t, rows, name):
    _need(t, torch.int32, name)
    if t.dim() != 1 or t.numel() != rows:
        raise ValueError(f"{name} must hold {rows} int32")


def attention_tree(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                   context_lens: torch.Tensor, cu_seqlens: torch.Tensor | None = None,
                   tree_mask: torch.Tensor | None = None, scale: float | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over a paged binary16 cache: a decoding step, or a tree of drafts.

    q [T, Hq, D] f32; k_pages, v_pages [n_pages, page_size, Hk, D] float16; block_table [B, W] and context_lens [B]
    int32.  Sequence b's pages hold context_lens[b] tokens and behind them its new tokens, whose q rows are
    cu_seqlens[b] .. cu_seqlens[b+1]-1 (None: one each, T == B).  A new token sees the context and the new tokens up
    to itself, or, with tree_mask (int64, [T] or [T, words]), the new tokens j of its sequence whose bit j%64 of word
    j/64 is set.  Everything else as attention_prefill."""
    r = _fast.attention_tree(q, k_pages, v_pages, block_table, context_lens, cu_seqlens, tree_mask, scale, out)
    if r is not None:
        return r
    _need(q, torch.float32, "q", contiguous=False)
    T, Hq, D, qs = _heads_view(q, "q")
    g = _kv_pages(k_pages, v_pages, False)
    if g.head_dim != D:
        raise ValueError("the pages must have q's head_dim")
    _need(context_lens, torch.int32, "context_lens")
    B = context_lens.numel()
    _rows_i32(context_lens, B, "context_lens")
    _table(block_table, B)
    if cu_seqlens is not None:
        _rows_i32(cu_seqlens, B + 1, "cu_seqlens")
    elif T != B:
        raise ValueError("without cu_seqlens there is one token per sequence")
    words = 0
    if tree_mask is not None:
        _need(tree_mask, torch.int64, "tree_mask")
        if tree_mask.dim() not in (1, 2) or tree_mask.shape[0] != T:
            raise ValueError("tree_mask must be [tokens] or [tokens, words]")
        words = tree_mask.shape[1] if tree_mask.dim() == 2 else 1
        if words == 0:
            raise ValueError("tree_mask must hold at least one word per token")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=torch.float32, device=q.device)
    _need(out, torch.float32, "out", contiguous=False)
    To, Ho, Do, os_ = _heads_view(out, "out")
    if (To, Ho, Do) != (T, Hq, D):
        raise ValueError("out must match q")
    L = _lib.load()
    W = block_table.shape[1]
    ws = _workspace(L.v7g_attention_tree_workspace(B, T, W, g.page_size, Hq, g.n_kv_heads, D), q.device)
    _bind(q)
    rc = L.v7g_attention_tree(out.data_ptr(), os_, q.data_ptr(), qs, ctypes.addressof(g), block_table.data_ptr(), W,
                              context_lens.data_ptr(), _ptr(cu_seqlens), _ptr(tree_mask) if T else None,
                              words if T else 0, B, T, Hq, _scale(scale, D), _ptr(ws), 0 if ws is None else ws.numel())
    _lib.check(rc, "attention_tree")
    return out


def kv_pack_f16_pages(k_src: torch.Tensor, v_src: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                      block_table: torch.Tensor, positions: torch.Tensor, seqs: torch.Tensor | None = None) -> None:
    """binary16 copies of the K and V rows [T, Hk*D] f32 (views into one fused QKV buffer: the same row stride) into
    one layer's pages [n_pages, page_size, Hk, D]: token t's at position positions[t] of the sequence of block table
    row seqs[t] (None: row t).  A token with no such row, position or page is skipped; the places of one call are
    distinct."""
    if _fast.kv_pack_f16_pages(k_src, v_src, k_pages, v_pages, block_table, positions, seqs):
        return
    _need(k_src, torch.float32, "k_src", contiguous=False)
    _need(v_src, torch.float32, "v_src", contiguous=False)
    if k_src.dim() != 2 or k_src.stride(1) != 1 or v_src.shape != k_src.shape or v_src.stride() != k_src.stride():
        raise ValueError("k_src and v_src must be [tokens, row_len] with contiguous rows and the same row stride")
    g = _kv_pages(k_pages, v_pages, False)
    T, n = k_src.shape
    if n != g.n_kv_heads * g.head_dim:
        raise ValueError("a row must hold the pages' kv_heads*head_dim floats")
    _table(block_table, None)
    _rows_i32(positions, T, "positions")
    B, W = block_table.shape
    if seqs is not None:
        _rows_i32(seqs, T, "seqs")
    elif T > B:
        raise ValueError("without seqs there is at most one token per sequence")
    _bind(k_src)
    rc = _lib.load().v7g_kv_pack_f16_pages(ctypes.addressof(g), k_src.data_ptr(), v_src.data_ptr(), k_src.stride(0),
                                           block_table.data_ptr(), W, B, positions.data_ptr(), _ptr(seqs), T)
    _lib.check(rc, "kv_pack_f16_pages")


def kv_pages_assign(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                    refs: torch.Tensor, parents: torch.Tensor, reserve: torch.Tensor | None = None):
    """Forks, frees and grows the sequences of a paged cache: returns (block_table, lens, refs, short), all new.

    Row r of the new table [B, W] is the sequence of row parents[r] (r: stays, another row: a fork, -1: freed), with
    room for reserve[r] more tokens.  Full pages are shared and counted in refs [n_pages] (0: free); a partly filled
    last page is copied, in every layer of k_pages, v_pages [(layers,) n_pages, page_size, Hk, D], for every row but
    the one that takes it over (the parent itself, else its lowest fork).  New pages are the lowest free ones, in the
    order of the rows; short [1] counts those that were missing, whose entries stay -1 (a fork without its copy ends
    with its full pages).  All indices int32."""
    r = _fast.kv_pages_assign(k_pages, v_pages, block_table, lens, refs, parents, reserve)
    if r is not None:
        return r
    g = _kv_pages(k_pages, v_pages, True)
    _table(block_table, None)
    B, W = block_table.shape
    _rows_i32(lens, B, "lens")
    _rows_i32(refs, g.n_pages, "refs")
    _rows_i32(parents, B, "parents")
    if reserve is not None:
        _rows_i32(reserve, B, "reserve")
    table_out, lens_out, refs_out = torch.empty_like(block_table), torch.empty_like(lens), torch.empty_like(refs)
    short = torch.empty(1, dtype=torch.int32, device=refs.device)
    L = _lib.load()
    ws = _workspace(L.v7g_kv_pages_assign_workspace(B, g.n_pages), refs.device)
    _bind(refs)
    rc = L.v7g_kv_pages_assign(ctypes.addressof(g), table_out.data_ptr(), lens_out.data_ptr(), refs_out.data_ptr(),
                               short.data_ptr(), block_table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                               parents.data_ptr(), _ptr(reserve), B, W, _ptr(ws), 0 if ws is None else ws.numel())
    _lib.check(rc, "kv_pages_assign")
    return table_out, lens_out, refs_out, short


def kv_pages_compact(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
                     path: torch.Tensor, n_path: torch.Tensor) -> torch.Tensor:
    """Keeps accepted drafts: of the new tokens behind lens[r] tokens of row r, those numbered path[r, :n_path[r]]
    (strictly ascending; the path ends at the first entry that does not ascend or has no page) move to the places from
    lens[r] on, in every layer of k_pages, v_pages [(layers,) n_pages, page_size, Hk, D].  Returns the new lens."""
    r = _fast.kv_pages_compact(k_pages, v_pages, block_table, lens, path, n_path)
    if r is not None:
        return r
    g = _kv_pages(k_pages, v_pages, True)
    _table(block_table, None)
    B, W = block_table.shape
    _rows_i32(lens, B, "lens")
    _rows_i32(n_path, B, "n_path")
    _table(path, B, "path")
    lens_out = torch.empty_like(lens)
    _bind(lens)
    rc = _lib.load().v7g_kv_pages_compact(ctypes.addressof(g), lens_out.data_ptr(), block_table.data_ptr(), W,
                                          lens.data_ptr(), path.data_ptr(), path.shape[1], n_path.data_ptr(), B)
    _lib.check(rc, "kv_pages_compact")
    return lens_out


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top_k: int = 0):
    """Scores of logit rows [T, V] f32 (row stride free): returns (logprobs [T] of the tokens ids [T] int32, entropies
    [T] in nats, top log probabilities [T, top_k], top ids [T, top_k] int32; top_k <= 64).  Equal logits: the lower
    index first.  An id outside the vocabulary gives NaN, a row with NaN or +inf or nothing above -inf NaN for every
    probability."""
    r = _fast.token_logprobs(logits, ids, top_k)
    if r is not None:
        return r
    _need(logits, torch.float32, "logits", contiguous=False)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [tokens, vocab] with contiguous rows")
    T, V = logits.shape
    _rows_i32(ids, T, "ids")
    K = int(top_k)
    if not 0 <= K <= 64:
        raise ValueError("top_k must lie in 0..64")
    dev = logits.device
    lp, ent = (torch.empty(T, dtype=torch.float32, device=dev) for _ in range(2))
    tl = torch.empty((T, K), dtype=torch.float32, device=dev)
    ti = torch.empty((T, K), dtype=torch.int32, device=dev)
    L = _lib.load()
    ws = _workspace(L.v7g_token_logprobs_workspace(T, V, K), dev)
    _bind(logits)
    rc = L.v7g_token_logprobs(lp.data_ptr(), ent.data_ptr(), tl.data_ptr() if K else None, ti.data_ptr() if K else None,
                              logits.data_ptr(), logits.stride(0), ids.data_ptr(), T, V, K, _ptr(ws),
                              0 if ws is None else ws.numel())
    _lib.check(rc, "token_logprobs")
    return lp, ent, tl, ti
