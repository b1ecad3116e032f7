"""Serving operators: what a decode or prompt step runs between the qkv and o
linears (norm + rotary + cache write, attention) and after the lm_head (log
probabilities).  torch-tensor front end of libfp8gq, as ``ops``: dtypes,
shapes and layouts are checked here, outputs come from torch's caching
allocator, and the kernels run on the tensors' device, on torch's current stream
there.  There is no CPU path.

A paged cache is two tensors ``k_cache`` and ``v_cache`` of shape [pages,
page_size, kv heads, D], bf16 or float8_e4m3fn (a stored value then stands for
value * k_scale or value * v_scale); any strides with contiguous heads, in
multiples of 16 bytes.  Values on the device (positions, slots, page tables,
lengths, offsets, tokens) are not read on the host: one out of range is
recorded in the device error word (``device_error()``), not raised.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import warnings
from typing import NamedTuple

import torch

from . import _build, _lib
from .ops import RMS_EPS, ShapeError, _stream, _workspace_entry, _workspaces

HEAD_DIMS = (64, 128)
MAX_TOP = 32
PROMPT_COUNTER_BYTES = 16384   # FP8GQ_PROMPT_COUNTER_BYTES
_BF16, _E4M3, _F32 = 0, 1, 2   # FP8GQ_DTYPE_*
_byref = ctypes.byref
_decode_ws_bytes: dict = {}    # (device, Hq, Hkv, D) -> fp8gq_paged_decode_workspace_bytes


class _Binding:
    """The C++ binding (csrc/serve_python.cpp), loaded at the first call.  Its
    functions return None for anything but the plain form of the arguments; the
    checks below then raise, or complete the call.  Where it can be neither loaded
    nor built, they complete every call."""

    def __getattr__(self, name):
        _lib.load()
        try:
            loader = importlib.machinery.ExtensionFileLoader("_serve_native", str(_build.build_native()))
            mod = importlib.util.module_from_spec(importlib.util.spec_from_loader("_serve_native", loader))
            loader.exec_module(mod)
            mod.set_workspaces(_workspaces)
        except (ImportError, OSError, RuntimeError) as e:
            warnings.warn("fp8gq: the serving operators run without their C++ binding, 10 us more a call: "
                          f"{str(e).strip()}", RuntimeWarning)
            mod = _NoBinding()
        global _native
        _native = mod
        return getattr(mod, name)


class _NoBinding:
    @staticmethod
    def _step_aside(*args):
        return None

    qk_norm_rope_append = paged_decode_attention = prompt_attention = token_logprobs = _step_aside


_native = _Binding()


def _check_device(*ts):
    """The one CUDA device that all of the tensors (None: not given) are on."""
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("fp8gq ops take CUDA tensors only (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}")
    return dev


def _check_sizes(**sizes):
    """The C entry points take 32-bit sizes (ctypes would cut larger ones)."""
    for name, n in sizes.items():
        if n > 2 ** 31 - 1:
            raise ShapeError(f"at most 2^31 - 1 {name}, got {n}")


def _check_cache(k, v, k_scale, v_scale):
    """Checks a paged cache; returns (its struct, Hkv, D)."""
    if k.dim() != 4 or k.shape != v.shape:
        raise ShapeError(f"k_cache and v_cache must both be [pages, page_size, kv heads, D], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float8_e4m3fn):
        raise TypeError(f"the cache must be bfloat16 or float8_e4m3fn, got {k.dtype} and {v.dtype}")
    pages, page, hkv, d = k.shape
    _check_sizes(slots_per_page=page, heads=hkv)
    if d not in HEAD_DIMS:
        raise ShapeError(f"heads of {HEAD_DIMS} values, got {d}")
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("the cache's heads must be contiguous")
    return _lib.PagedCache(k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages, page,
                           _BF16 if k.dtype == torch.bfloat16 else _E4M3, k_scale, v_scale), hkv, d


def _check_heads(t, name, d=None):
    """A [tokens, heads, D] bf16 operand with contiguous heads; returns its shape and strides."""
    if t.dtype != torch.bfloat16 or t.dim() != 3:
        raise TypeError(f"{name} must be a 3-D bf16 tensor [tokens, heads, D]")
    if t.stride(2) != 1:
        raise ValueError(f"the heads of {name} must be contiguous")
    if d is not None and t.shape[2] != d:
        raise ShapeError(f"{name} has heads of {t.shape[2]} values, expected {d}")
    return t.shape, t.stride()


def _check_out(out, shape, device, dtype=torch.bfloat16):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_cuda:
        raise ShapeError(f"the output must be a CUDA {dtype} tensor of shape {tuple(shape)}")
    return out


def _check_vector(t, name, n, dtype):
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ShapeError(f"{name} must be a contiguous {dtype} tensor of {n} values")


def qk_norm_rope_append(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, cos_sin: torch.Tensor,
                        k_cache: torch.Tensor, v_cache: torch.Tensor, *, q_weight=None, k_weight=None,
                        eps: float = RMS_EPS, k_scale: float = 1.0, v_scale: float = 1.0, q_out=None, k_out=None,
                        return_k: bool = False):
    """qkv (T, (Hq + 2 Hkv) * D) bf16, the qkv linear's output -> q (T, Hq, D) bf16.

    Each head of q and k is RMS-normed with ``q_weight`` / ``k_weight`` (bf16
    [D]; None: no norm) and rotated by ``cos_sin[positions]`` (fp32 [P, D]: D/2
    cosines, then D/2 sines; the halves of a head are the rotated pairs).  k and
    v are written into the cache at ``slots`` (int64 [T], page * page_size +
    place; negative: not stored).  ``return_k`` also returns k (T, Hkv, D) as it
    is before the cache's rounding to e4m3, for prompt_attention.  ``q_out`` and
    ``k_out`` may be views of qkv."""
    if q_out is None and k_out is None:
        r = _native.qk_norm_rope_append(qkv, positions, slots, cos_sin, k_cache, v_cache, q_weight, k_weight, eps,
                                        k_scale, v_scale, return_k)
        if r is not None:
            return r
    dev = _check_device(qkv, positions, slots, cos_sin, k_cache, v_cache, q_weight, k_weight, q_out, k_out)
    cache, hkv, d = _check_cache(k_cache, v_cache, k_scale, v_scale)
    if qkv.dtype != torch.bfloat16 or qkv.dim() != 2 or qkv.stride(1) != 1:
        raise TypeError("qkv must be a 2-D bf16 tensor, contiguous along its last dimension")
    t, cols = qkv.shape
    _check_sizes(tokens=t, columns=cols)
    hq = cols // d - 2 * hkv
    if cols % d or hq < 1 or hq % hkv:
        raise ShapeError(f"qkv has {cols} columns: expected (Hq + 2 * {hkv}) * {d} with Hq a multiple of {hkv}")
    _check_vector(positions, "positions", t, torch.int64)
    _check_vector(slots, "slots", t, torch.int64)
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or cos_sin.shape[1] != d or not cos_sin.is_contiguous():
        raise ShapeError(f"cos_sin must be a contiguous fp32 tensor [positions, {d}]")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _check_vector(w, name, d, torch.bfloat16)
    q_out = _check_out(q_out, (t, hq, d), dev)
    if return_k or k_out is not None:
        k_out = _check_out(k_out, (t, hkv, d), dev)
    for o, name in ((q_out, "q_out"), (k_out, "k_out")):
        if o is not None and (o.stride(2) != 1 or (o.shape[1] > 1 and o.stride(1) != d)):
            raise ValueError(f"a token's heads must be contiguous in {name}")
    with torch.cuda.device(dev):
        st = _lib.load().fp8gq_qk_norm_rope_append(
            qkv.data_ptr(), qkv.stride(0), positions.data_ptr(), slots.data_ptr(), cos_sin.data_ptr(), cos_sin.shape[0],
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), eps,
            q_out.data_ptr(), q_out.stride(0), None if k_out is None else k_out.data_ptr(),
            0 if k_out is None else k_out.stride(0), _byref(cache), t, hq, hkv, d, _stream(dev))
    _lib.check(st, "fp8gq_qk_norm_rope_append")
    return (q_out, k_out) if return_k else q_out


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                           lens: torch.Tensor, *, scale: float | None = None, k_scale: float = 1.0,
                           v_scale: float = 1.0, out=None, return_lse: bool = False):
    """q (B, Hq, D) bf16, one new token per sequence -> (B, Hq, D) bf16:
    softmax(scale * q k^T) v over the ``lens[b]`` tokens (int32 [B], the new one
    included) that the sequence's pages hold (``page_table`` int32 [B, pages]).
    ``scale`` is 1 / sqrt(D) by default.  Hq is a multiple of the cache's heads.
    A sequence of length 0 gives 0.  ``return_lse`` also returns the log of the
    softmax's sum, fp32 (B, Hq)."""
    if out is None:
        r = _native.paged_decode_attention(q, k_cache, v_cache, page_table, lens, scale, k_scale, v_scale, return_lse)
        if r is not None:
            return r
    dev = _check_device(q, k_cache, v_cache, page_table, lens, out)
    cache, hkv, d = _check_cache(k_cache, v_cache, k_scale, v_scale)
    (b, hq, _), qs = _check_heads(q, "q", d)
    _check_sizes(sequences=b, heads=hq)
    if hq % hkv:
        raise ShapeError(f"{hq} query heads are not a multiple of the cache's {hkv}")
    _check_vector(lens, "lens", b, torch.int32)
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b \
            or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ShapeError(f"page_table must be an int32 tensor [{b}, pages], contiguous along its last dimension")
    _check_sizes(pages_per_sequence=page_table.shape[1])
    if out is None:
        out = torch.empty((b, hq, d), dtype=torch.bfloat16, device=dev)
        os = (hq * d, d)
    else:
        shape, os = _check_heads(out, "out", d)
        if tuple(shape) != (b, hq, d):
            raise ShapeError(f"out must be {(b, hq, d)}, got {tuple(shape)}")
    lse = torch.empty((b, hq), dtype=torch.float32, device=dev) if return_lse else None
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = _stream(dev)
        key = (dev.index, hq, hkv, d)
        nbytes = _decode_ws_bytes.get(key)
        if nbytes is None:
            nbytes = _decode_ws_bytes[key] = lib.fp8gq_paged_decode_workspace_bytes(hq, hkv, d)
        _, ws_ptr, ws_n = _workspace_entry(dev, nbytes, stream)
        st = lib.fp8gq_paged_decode_attention(
            q.data_ptr(), qs[0], qs[1], _byref(cache), page_table.data_ptr(), page_table.stride(0), page_table.shape[1],
            lens.data_ptr(), out.data_ptr(), os[0], os[1], None if lse is None else lse.data_ptr(), b, hq, hkv, d,
            d ** -0.5 if scale is None else scale, ws_ptr, ws_n, stream)
    _lib.check(st, "fp8gq_paged_decode_attention")
    return (out, lse) if return_lse else out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, cu_k=None, *,
                     causal: bool = True, scale: float | None = None, out=None, return_lse: bool = False):
    """Packed prompts: q (Tq, Hq, D), k and v (Tk, Hkv, D) bf16 (views of one
    qkv buffer will do) -> (Tq, Hq, D) bf16.  Sequence b has the q tokens
    ``cu_q[b] .. cu_q[b + 1]`` and the k tokens ``cu_k[b] .. cu_k[b + 1]`` (int32
    [B + 1] on the device; cu_k is cu_q by default).  Causal: row i sees the keys
    j <= i + (k tokens - q tokens), so that its last row sees all of them.  A row
    that sees none gives 0; rows past cu_q[B] are not written.  ``scale`` is
    1 / sqrt(D) by default.  ``return_lse`` also returns fp32 (Tq, Hq)."""
    if out is None:
        r = _native.prompt_attention(q, k, v, cu_q, cu_k, causal, scale, return_lse)
        if r is not None:
            return r
    dev = _check_device(q, k, v, cu_q, cu_k, out)
    (tq, hq, d), qs = _check_heads(q, "q")
    (tk, hkv, _), ks = _check_heads(k, "k", d)
    vshape, vs = _check_heads(v, "v", d)
    _check_sizes(tokens=max(tq, tk), heads=hq)
    if d not in HEAD_DIMS:
        raise ShapeError(f"heads of {HEAD_DIMS} values, got {d}")
    if vshape != k.shape or hkv < 1 or hq % hkv:
        raise ShapeError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(vshape)} do not match")
    if cu_k is None:
        cu_k = cu_q
    if cu_q.dim() != 1 or cu_q.shape[0] < 1:
        raise ShapeError("cu_q must hold one offset more than there are sequences")
    n = cu_q.shape[0]
    _check_sizes(offsets=n)
    _check_vector(cu_q, "cu_q", n, torch.int32)
    _check_vector(cu_k, "cu_k", n, torch.int32)
    if out is None:
        out = torch.empty((tq, hq, d), dtype=torch.bfloat16, device=dev)
        os = (hq * d, d)
    else:
        shape, os = _check_heads(out, "out", d)
        if shape != q.shape:
            raise ShapeError(f"out must be {tuple(q.shape)}, got {tuple(shape)}")
    lse = torch.empty((tq, hq), dtype=torch.float32, device=dev) if return_lse else None
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = _stream(dev)
        nbytes = lib.fp8gq_prompt_split_bytes(n - 1, tq, tk, hq, hkv, d, 1 if causal else 0)
        if nbytes:      # two launches: scratch of this call's own, since another thread's launch may come between them
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            ws_ptr, ws_n = ws.data_ptr(), nbytes
        else:
            _, ws_ptr, ws_n = _workspace_entry(dev, PROMPT_COUNTER_BYTES, stream)
        st = lib.fp8gq_prompt_attention(
            q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], out.data_ptr(), os[0],
            os[1], None if lse is None else lse.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), n - 1, tq, tk, hq, hkv, d,
            d ** -0.5 if scale is None else scale, 1 if causal else 0, ws_ptr, ws_n, stream)
    _lib.check(st, "fp8gq_prompt_attention")
    return (out, lse) if return_lse else out


class TokenLogprobs(NamedTuple):
    """token_logprobs' outputs (None where not asked for)."""
    logprobs: torch.Tensor | None      # fp32 (T,)
    entropy: torch.Tensor              # fp32 (T,), nats
    top_ids: torch.Tensor | None       # int64 (T, top_k), descending
    top_logprobs: torch.Tensor | None  # fp32 (T, top_k)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0) -> TokenLogprobs:
    """logits (T, V) bf16 or fp32 -> the log probabilities of ``tokens`` (int64
    [T]; negative: none given, 0), the entropy and the ``top_k`` <= 32 likeliest
    tokens of each row (equal logits by ascending index).  -inf rules a token
    out; a row with NaN or +inf, or with no finite logit, has NaN throughout."""
    r = _native.token_logprobs(logits, tokens, top_k)
    if r is not None:
        return TokenLogprobs._make(r)
    dev = _check_device(logits, tokens)
    if logits.dtype not in (torch.bfloat16, torch.float32) or logits.dim() != 2:
        raise TypeError("logits must be a 2-D bf16 or fp32 tensor")
    t, v = logits.shape
    _check_sizes(rows=t, logits_per_row=v)
    if v < 1 or (v > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be contiguous along the vocabulary")
    if not 0 <= top_k <= min(MAX_TOP, v):
        raise ShapeError(f"0 <= top_k <= {min(MAX_TOP, v)}, got {top_k}")
    lp = ids = tops = None
    if tokens is not None:
        _check_vector(tokens, "tokens", t, torch.int64)
        lp = torch.empty(t, dtype=torch.float32, device=dev)
    ent = torch.empty(t, dtype=torch.float32, device=dev)
    ids = torch.empty((t, top_k), dtype=torch.int64, device=dev)
    tops = torch.empty((t, top_k), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        st = _lib.load().fp8gq_token_logprobs(
            logits.data_ptr(), logits.stride(0), _BF16 if logits.dtype == torch.bfloat16 else _F32,
            None if tokens is None else tokens.data_ptr(), t, v, None if lp is None else lp.data_ptr(), ent.data_ptr(),
            ids.data_ptr(), tops.data_ptr(), top_k, _stream(dev))
    _lib.check(st, "fp8gq_token_logprobs")
    return TokenLogprobs(lp, ent, ids, tops)
