"""Paged serving: many requests over one pool of KV pages (ffts_page_plan, ffts_rope_append, ffts_paged_attn).

The reference's callers prefill one prompt and decode it over one contiguous
cache (eval/LongBench/pred.py:177-322).  A server keeps many requests whose caches grow token by token in
pages of a shared pool.  One step of it:

    plan = plan_pages(cached_lens, new_lens, block_table, free_pages, page_size, num_tokens)   # once
    for each layer:
        q = rope_append(q, k, v, plan.positions, plan.slot_map, k_pages, v_pages, inv_freq)
        out = paged_attention(q, k_pages, v_pages, block_table, plan.cu_q, plan.kv_lens)

New tokens are packed: request r owns rows ``cu_q[r] .. cu_q[r + 1] - 1`` of q, k, v and out.  One token is
decoding, more are a chunk of its prompt; a step may mix them.  Lengths and tables are device tensors that the
host never reads, so a step can be captured into a CUDA graph and replayed with other lengths.

The pool's tensors are [pages, Hkv, page_size, D], the head-major layout the other
operators use; a token-major pool [pages, page_size, Hkv, D] is passed as
``pool.transpose(1, 2)``.  A prompt that ``myattn_prefill`` has attended is
handed over with ``rope_append(None, k[0].transpose(0, 1), v[0].transpose(0, 1), ..., inv_freq=None)``,
which copies the already rotated k.
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .status import device_status

__all__ = ["PagePlan", "plan_pages", "rotary_inv_freq", "rope_append", "paged_attention"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
# The C calls' argument blocks (ffts_*_args): 64-bit pointers, strides and sizes, then the 32-bit fields.
_PLAN = struct.Struct("=16q")
_ROPE = struct.Struct("=31qiifi")
_ATTN = struct.Struct("=32qif")
_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(device).cuda_stream without the Stream object


_I32 = torch.int32
_get_device = torch._C._cuda_getDevice

# The checks below run in every call of a decoding step: a device is compared by its index (-1 on the CPU).


def _call(index: int, fn, block: bytes) -> None:
    """One C call with device ``index`` current, on its current stream."""
    if index == _get_device():
        rc = fn(block, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(block, _raw_stream(index))
    if rc:
        _lib.check(rc)


def _check_ints(name: str, t: torch.Tensor, n: int, index: int) -> None:
    if t.dtype is not _I32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of shape [{n}], got {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on the other tensors' device, got {t.device}")


def _check_table(t: torch.Tensor, rows: int, index: int):
    """The table's row stride (its width for a single row) and width."""
    if t.dtype is not _I32:
        raise TypeError(f"block_table must be int32, got {t.dtype}")
    if t.dim() == 2:
        n, width = t.shape
        ld, unit = t.stride()
        if n == rows and (unit == 1 or width <= 1):
            if t.get_device() != index:
                raise ValueError(f"block_table must be on the other tensors' device, got {t.device}")
            return (ld if rows > 1 else width), width
    raise ValueError(f"block_table must be [{rows}, pages] with unit stride along a row, got {tuple(t.shape)}")


def _check_heads(name: str, t: torch.Tensor, dtype, index: int):
    """The token and head strides and the shape of a [tokens, heads, head_dim] tensor."""
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got shape {tuple(shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} must be on the other tensors' device, got {t.device}")
    st, sh, sd = t.stride()
    if sd != 1:
        raise ValueError(f"{name} must be contiguous in the head dimension")
    n, h, d = shape
    return ((st if n > 1 else h * d), (sh if h > 1 else d)), shape  # a single row's stride says nothing


def _check_pool(k_pages: torch.Tensor, v_pages: torch.Tensor, dtype, index: int):
    """The page, head and row strides of both pool tensors, and their shape."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError(f"k_pages and v_pages must both be [pages, Hkv, page_size, D], got "
                         f"{tuple(shape)} / {tuple(v_pages.shape)}")
    if k_pages.dtype is not dtype or v_pages.dtype is not dtype:
        raise TypeError(f"k_pages and v_pages must be {dtype}, got {k_pages.dtype} / {v_pages.dtype}")
    if k_pages.get_device() != index or v_pages.get_device() != index:
        raise ValueError("k_pages and v_pages must be on the other tensors' device")
    *ks, kd = k_pages.stride()
    *vs, vd = v_pages.stride()
    if kd != 1 or vd != 1:
        raise ValueError("k_pages and v_pages must be contiguous in the head dimension")
    P, h, n, d = shape
    if P == 1 or h == 1 or n == 1:  # the stride of a single page, head or row says nothing
        packed = (h * n * d, n * d, d)
        ks, vs = ([s if m > 1 else c for s, m, c in zip(st, shape, packed)] for st in (ks, vs))
    return ks, vs, shape


def _check_cuda(name: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")


class PagePlan(NamedTuple):
    """The bookkeeping of one step (``plan_pages``)."""

    cu_q: torch.Tensor       # int32 [R + 1]: first row of each request's new tokens
    kv_lens: torch.Tensor    # int32 [R]: cached + new tokens, 0 for a request that is not served
    positions: torch.Tensor  # int32 [num_tokens]
    slot_map: torch.Tensor   # int32 [num_tokens]: page * page_size + row in the pool, -1 for none
    info: torch.Tensor       # int32 [2]: pages taken from the free list, requests not served


def plan_pages(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
               free_pages: torch.Tensor, page_size: int, num_tokens: int) -> PagePlan:
    """Page bookkeeping of one step on the GPU (ffts_page_plan).

    ``cached_lens`` / ``new_lens`` int32 [R]: tokens each request has in the cache, and adds in this step.
    ``block_table`` int32 [R, width]: its page numbers, the first ceil(cached / page_size) of a row valid; the
    entries of the pages that the new tokens begin are filled in place with ``free_pages`` (int32, taken
    from the front in the order of the requests).  ``num_tokens``: rows of the step's token
    arrays, at least the sum of ``new_lens``; rows behind the last token get position 0 and slot -1, so a
    batch padded to a fixed size can be replayed from a graph.

    A request is served if its pages fit its row, its tokens fit ``num_tokens`` and its new pages, counted on
    from those of the requests before it, fit the free list.  Otherwise its kv_len is 0 and its slots are -1:
    its tokens are not appended and attend to nothing.  ``info`` holds the pages taken and the requests
    not served; the caller drops that many entries from the front of its list.  Nothing is read back.
    """
    index = cached_lens.get_device()
    if cached_lens.dim() != 1 or free_pages.dim() != 1:
        raise ValueError("cached_lens and free_pages must be 1-D")
    R, n_free = cached_lens.shape[0], free_pages.shape[0]
    _check_ints("cached_lens", cached_lens, R, index)
    _check_ints("new_lens", new_lens, R, index)
    _check_ints("free_pages", free_pages, n_free, index)
    table_ld, width = _check_table(block_table, R, index)
    if num_tokens < 0:
        raise ValueError(f"num_tokens must not be negative, got {num_tokens}")
    _check_cuda("cached_lens", cached_lens)
    buf = cached_lens.new_empty(2 * R + 2 * num_tokens + 3)
    plan = PagePlan(*buf.split_with_sizes([R + 1, R, num_tokens, num_tokens, 2]))
    cu = buf.data_ptr()
    kv = cu + 4 * (R + 1)
    pos = kv + 4 * R
    slot = pos + 4 * num_tokens
    _call(index, _lib.load().ffts_page_plan, _PLAN.pack(
        _PLAN.size, cached_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), cu, kv,
        pos, slot, slot + 4 * num_tokens, R, table_ld, width, n_free, page_size, num_tokens))
    return plan


def rotary_inv_freq(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                    seq_len: Optional[int] = None, device=None, *,
                    max_position_embeddings: Optional[int] = None) -> Tuple[torch.Tensor, float]:
    """(inv_freq fp32 [rotary_dim / 2], attn_factor) of a rotary embedding, as ``rope_append`` takes them.

    ``scaling`` is a model configuration's ``rope_scaling`` dict; its ``rope_type`` is one of

      default  f_i = base^(-2i / d)
      linear   f_i / factor
      dynamic  base grown to base (factor L / L0 - factor + 1)^(d / (d - 2)), L = max(seq_len, L0)
      llama3   f_i / factor for wavelengths above L0 / low_freq_factor, f_i below L0 / high_freq_factor, a linear
               blend between
      yarn     f_i / factor and f_i blended over the channels that turn beta_slow to beta_fast times within L0
               (whole channels unless truncate is false); attn_factor = attention_factor, or m(mscale) / m(mscale_all_dim)
               where both are given, or m(1), with m(x) = 0.1 x ln(factor) + 1

    with L0 = the dict's ``original_max_position_embeddings``, or, where it has none, ``max_position_embeddings`` (the
    configuration's own).  Computed in 64 bits, rounded once.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    d, scaling = rotary_dim, scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "dynamic" and d == 2:
        raise ValueError("rope scaling 'dynamic' needs rotary_dim above 2")
    i = torch.arange(0, d, 2, dtype=torch.float64)
    attn = 1.0

    def need(key):
        if scaling.get(key) is None:
            raise ValueError(f"rope scaling '{kind}' needs '{key}'")
        return float(scaling[key])

    def context():
        if scaling.get("original_max_position_embeddings") is None and max_position_embeddings is not None:
            return float(max_position_embeddings)
        return need("original_max_position_embeddings")

    if kind == "dynamic":
        L0, s = context(), need("factor")
        L = max(float(seq_len or 0), L0)
        base = base * (s * L / L0 - (s - 1.0)) ** (d / (d - 2))
    f = float(base) ** (-i / d)
    if kind == "linear":
        f = f / need("factor")
    elif kind == "llama3":
        L0, s = context(), need("factor")
        low, high = need("low_freq_factor"), need("high_freq_factor")
        turns = L0 * f / (2.0 * math.pi)  # within the original context
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / s
    elif kind == "yarn":
        L0, s = context(), need("factor")

        def channel(turns):  # the pair that turns so often within L0
            return d * math.log(L0 / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        lo, hi = (channel(float(scaling.get(k) or v)) for k, v in (("beta_fast", 32.0), ("beta_slow", 1.0)))
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, d - 1)
        slow = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = slow * f / s + (1.0 - slow) * f

        def m(x):
            return 0.1 * x * math.log(s) + 1.0 if s > 1.0 else 1.0

        given, ms, ms_all = (scaling.get(k) for k in ("attention_factor", "mscale", "mscale_all_dim"))
        attn = float(given) if given is not None else (m(float(ms)) / m(float(ms_all)) if ms and ms_all else m(1.0))
    elif kind not in ("default", "dynamic"):
        raise ValueError(f"unknown rope scaling '{kind}'")
    return f.to(torch.float32).to(device), attn


def rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                slot_map: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                inv_freq: Optional[torch.Tensor], *, interleaved: bool = False, attn_factor: float = 1.0,
                out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate q and k by their positions and append k and v to the paged cache, in one pass (ffts_rope_append).

    q [T, H, D] (or None), k / v [T, Hkv, D]: bf16 or fp16, D 64 or 128, unit stride over D (views of one fused
    QKV projection are fine).  ``positions`` / ``slot_map`` int32 [T] (``plan_pages``); a token whose
    slot lies outside the pool is not appended; no two tokens have the same slot.  ``inv_freq`` fp32 [rotary_dim / 2]
    (``rotary_inv_freq``), rotary_dim a multiple of 16: the first rotary_dim channels turn by position * inv_freq, in pairs (i, i + rotary_dim / 2),
    or (2i, 2i + 1) with ``interleaved``; cos and sin are multiplied by ``attn_factor``; the other channels are
    copied.  None copies k (and q) as they are.  ``k_pages`` / ``v_pages`` [pages, Hkv, page_size, D] are
    written in place.  Returns the rotated q [T, H, D] (``out``, which may be q itself, or a new tensor), None
    without q.  The angles are exact for far positions (64 bits), the rotation is fp32, rounded once.
    """
    index, dt = k.get_device(), k.dtype
    if dt not in _DTYPES:
        raise TypeError(f"rope_append supports bfloat16 and float16, got {dt}")
    ks, shape = _check_heads("k", k, dt, index)
    vs, v_shape = _check_heads("v", v, dt, index)
    T, Hkv, D = shape
    if v_shape != shape:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v_shape)} differ in shape")
    kps, vps, (P, kv_heads, page_size, dim) = _check_pool(k_pages, v_pages, dt, index)
    if kv_heads != Hkv or dim != D:
        raise ValueError(f"pages {tuple(k_pages.shape)} do not match k {tuple(shape)}")
    _check_ints("positions", positions, T, index)
    _check_ints("slot_map", slot_map, T, index)
    rd = freq = 0
    if inv_freq is not None:
        if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float32 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be a contiguous 1-D fp32 tensor")
        if inv_freq.get_device() != index:
            raise ValueError(f"inv_freq must be on the other tensors' device, got {inv_freq.device}")
        rd, freq = 2 * inv_freq.shape[0], inv_freq.data_ptr()
    H = q_ptr = o_ptr = 0
    qs = os_ = (0, 0)
    if q is not None:
        qs, (n, H, dim) = _check_heads("q", q, dt, index)
        if n != T or dim != D:
            raise ValueError(f"q {tuple(q.shape)} does not match k {tuple(shape)}")
    if out is not None:
        if q is None:
            raise ValueError("out without q")
        os_, o_shape = _check_heads("out", out, dt, index)
        if o_shape != q.shape:
            raise ValueError(f"out must have q's shape {tuple(q.shape)}, got {tuple(o_shape)}")
    _check_cuda("k", k)
    if q is not None:
        if out is None:
            out = q.new_empty((T, H, D))
            os_ = (H * D, D)
        q_ptr, o_ptr = q.data_ptr(), out.data_ptr()
    if T == 0:
        return out
    _call(index, _lib.load().ffts_rope_append, _ROPE.pack(
        _ROPE.size, q_ptr, k.data_ptr(), v.data_ptr(), positions.data_ptr(), slot_map.data_ptr(), freq, o_ptr,
        k_pages.data_ptr(), v_pages.data_ptr(), *qs, *ks, *vs, *os_, *kps, *vps, T, H, Hkv, D, rd, P, page_size,
        _DTYPES[dt], interleaved, attn_factor, 0))
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_lens: torch.Tensor, *, scale: Optional[float] = None,
                    window: Optional[int] = None, sinks: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each request's new tokens over its pages (ffts_paged_attn).

    q [T, H, D]: request r's new tokens are rows ``cu_q[r] .. cu_q[r + 1] - 1``, the last of its ``kv_lens[r]``
    tokens; ``k_pages`` / ``v_pages`` [pages, Hkv, page_size, D] hold all of them (append first), H % Hkv == 0,
    H / Hkv <= 128, page_size 16 to 256 (a power of two), D 64 or 128, bf16 or fp16.  ``block_table`` int32
    [R, width], ``cu_q`` int32 [R + 1], ``kv_lens`` int32 [R] (``plan_pages``); requests may have any number of
    new tokens, also none.  ``scale`` defaults to D ** -0.5.

    With ``window`` W a token at position p sees the keys p - W + 1 .. p and the first ``sinks`` keys of its
    request (the work does not grow with the rest); pages it does not see may be gone from the table.  Tokens that see
    nothing (kv_len 0) get zeros; a NaN or infinite score among the keys that a token sees makes its row NaN, as the
    softmax does (a score of -inf has no weight), and a v that is not finite reaches its channels of the tokens that see
    its key, no others.  Returns [T, H, D] (or fills ``out``); rows of no request are not written.

    A bounded wait that runs out in the kernel raises WaitTimeout at a later call or at ``check_status()``.  Before a
    capture into a CUDA graph make one call outside of it (it sets up the device's status word).
    """
    index, dt = q.get_device(), q.dtype
    if dt not in _DTYPES:
        raise TypeError(f"paged attention supports bfloat16 and float16, got {dt}")
    qs, (T, H, D) = _check_heads("q", q, dt, index)
    kps, vps, (P, Hkv, page_size, dim) = _check_pool(k_pages, v_pages, dt, index)
    if dim != D or Hkv == 0 or H % Hkv:
        raise ValueError(f"pages {tuple(k_pages.shape)} do not match q {tuple(q.shape)}")
    if kv_lens.dim() != 1:
        raise ValueError("kv_lens must be 1-D")
    R = kv_lens.shape[0]
    _check_ints("kv_lens", kv_lens, R, index)
    _check_ints("cu_q", cu_q, R + 1, index)
    table_ld, width = _check_table(block_table, R, index)
    if window is None:
        if sinks:
            raise ValueError("sinks need a window")
        window = 0
    elif window < 1:
        raise ValueError(f"window must be at least 1, got {window}")
    if sinks < 0:
        raise ValueError(f"sinks must not be negative, got {sinks}")
    if out is not None:
        os_, o_shape = _check_heads("out", out, dt, index)
        if o_shape != q.shape:
            raise ValueError(f"out must have q's shape {tuple(q.shape)}, got {tuple(o_shape)}")
    if P == 0:
        raise ValueError("the pool has no pages")
    _check_cuda("q", q)
    if out is None:
        out = q.new_empty((T, H, D))
        os_ = (H * D, D)
    if T == 0 or R == 0:
        return out
    lib = _lib.load()
    status = device_status(q.device)
    status.poll_direct()
    nbytes = lib.ffts_paged_workspace_bytes(T, R, H, Hkv, D)
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    _call(index, lib.ffts_paged_attn, _ATTN.pack(
        _ATTN.size, q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(), cu_q.data_ptr(),
        kv_lens.data_ptr(), out.data_ptr(), ws.data_ptr(), status.direct_ptr, *qs, *kps, *vps, *os_, T, R, H, Hkv, D, P,
        page_size, table_ld, width, window, sinks, nbytes, _DTYPES[dt], D ** -0.5 if scale is None else scale))
    return out
