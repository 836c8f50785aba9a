"""Slot KV caches of the hybrid stack's full-attention layers in bf16 or e4m3, and decode attention over them.

The reference's engine keeps bf16 K and V per slot, copies a prefill's HF cache rows into them
(src/cb_engine.py:198-205, :229-239) and attends to them at decode (src/cb_engine.py:265-276).  Here:
  * ``KVCache``                  -- the tensors of one layer's cache, bf16 or e4m3 (half the bytes)
  * ``kv_cache_store`` / ``kv_cache_load`` -- packed prompts' rows into the slots (quantised as they are written) and back
  * ``cached_decode_attention``  -- gqa_decode_attention over such a cache, optionally behind prefixes that several
    slots share (``SharedPrefix``), each read once for all of them
The layout of a cache is documented in include/gdn_mi355x.h.
"""
from typing import NamedTuple, Optional

import torch

from . import _lib
from .cb_engine import Partials
from .gdn_chunk_fast import Rows, Varlen, _to_device_int32

F8 = torch.float8_e4m3fn
_BLOCK = 64
_NO_PREFIX = (None,) * 6


class KVCache(NamedTuple):
    """One layer's cache of R rows (slots, or prefixes): k, v [R, kv, T / 64, 64 * hd] bf16 or float8_e4m3fn, each
    block's 64 tokens in the attention kernel's order; in e4m3 k_exp, v_exp uint8 [R, kv, T] hold the scales (byte e + 127:
    the row's values are code * 2^e)."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: Optional[torch.Tensor] = None
    v_exp: Optional[torch.Tensor] = None

    @classmethod
    def empty(cls, n_rows, kv_heads, head_dim, length, dtype=F8, device="cuda"):
        """A cache of zeros for at least ``length`` tokens a row (rounded up to a multiple of 64)."""
        if dtype not in (F8, torch.bfloat16):
            raise TypeError(f"KVCache: dtype must be torch.float8_e4m3fn or torch.bfloat16, got {dtype}")
        if head_dim not in (64, 128, 256) or length < 1 or n_rows < 1 or kv_heads < 1:
            raise ValueError("KVCache: head_dim 64, 128 or 256 and positive sizes expected")
        blocks = (length + _BLOCK - 1) // _BLOCK
        k, v = (torch.zeros(n_rows, kv_heads, blocks, _BLOCK * head_dim, dtype=dtype, device=device) for _ in range(2))
        if dtype != F8:
            return cls(k, v)
        return cls(k, v, *(torch.full((n_rows, kv_heads, blocks * _BLOCK), 127, dtype=torch.uint8, device=device)
                           for _ in range(2)))

    @property
    def length(self):
        return self.k.shape[2] * _BLOCK

    @property
    def head_dim(self):
        return self.k.shape[3] // _BLOCK


class SharedPrefix(NamedTuple):
    """Prefixes that slots continue: row r of ``cache`` holds positions 0 .. length[r] - 1 (int32 [P] on the device) for
    every slot n with of[n] == r (int32 [N] on the device; a value outside [0, P): the slot has none).  Such a slot's own
    cache row starts at position length[r]."""
    cache: KVCache
    length: torch.Tensor
    of: torch.Tensor


# (these run once per layer and step: each attribute of a tensor that Python looks at costs a good part of a microsecond)
def _check(name, c):
    """(cache dtype code, rows, kv heads, head_dim, length, device index) of a well-formed cache."""
    k, v, ke, ve = c
    shape, dtype, dev = k.shape, k.dtype, k.get_device()
    if dev < 0 or v.get_device() != dev:
        _lib.require_cuda(k, v, ke, ve)
        raise ValueError(f"{name}: a cache's tensors must be on one device")
    if len(shape) != 4 or shape != v.shape or dtype is not v.dtype or not (k.is_contiguous() and v.is_contiguous()):
        raise ValueError(f"{name}: a cache's k and v are contiguous tensors [R, kv, T / 64, 64 * hd] of one dtype")
    R, kv, blocks, width = shape
    if width not in (4096, 8192, 16384) or blocks < 1:
        raise ValueError(f"{name}: head_dim must be 64, 128 or 256 (got {tuple(shape)} = [R, kv, T / 64, 64 * hd])")
    T = blocks * _BLOCK
    if dtype is F8:
        want = (R, kv, T)
        if ke is None or ve is None or ke.shape != want or ve.shape != want or ke.dtype is not torch.uint8 \
                or ve.dtype is not torch.uint8 or not (ke.is_contiguous() and ve.is_contiguous()):
            raise ValueError(f"{name}: an e4m3 cache needs contiguous uint8 k_exp and v_exp {list(want)}")
        if ke.get_device() != dev or ve.get_device() != dev:
            raise ValueError(f"{name}: a cache's tensors must be on one device")
        return _lib.F8E4M3, R, kv, width // _BLOCK, T, dev
    if dtype is not torch.bfloat16:
        raise TypeError(f"{name}: a cache is bfloat16 or float8_e4m3fn, got {dtype}")
    if ke is not None or ve is not None:
        raise ValueError(f"{name}: a bf16 cache has no scales")
    return _lib.BF16, R, kv, width // _BLOCK, T, dev


def _int32(name, what, x, n, device):
    """x (a list or CPU tensor, checked to fit, or an int32 tensor on the device) as int32 [n] on the device."""
    if not isinstance(x, torch.Tensor):
        x = torch.tensor(list(x), dtype=torch.int64)
    if n is not None and x.numel() != n:
        raise ValueError(f"{name}: {what} must have {n} entries, got {x.numel()}")
    if x.is_cuda:
        if x.dtype is not torch.int32 or x.get_device() != device.index:
            raise ValueError(f"{name}: {what} on the device must be int32 on {device}")
        return x if x.dim() == 1 and x.is_contiguous() else x.reshape(-1).contiguous()
    if x.dtype.is_floating_point or x.dtype == torch.bool:
        raise TypeError(f"{name}: {what} must be whole numbers")
    return _to_device_int32(x.reshape(-1).to(torch.int64), device)


def _batch(name, rows, cu_seqlens, start, total, n_rows, length, device):
    """Device int32 (rows, cu_seqlens, start) of a batch for a cache of n_rows rows of `length` tokens; what comes from the
    host is checked here, what is on the device is cut to the cache by the kernels."""
    if isinstance(rows, Rows):
        rows = rows.dev
    elif not (isinstance(rows, torch.Tensor) and rows.is_cuda):
        host = [int(r) for r in (rows.tolist() if isinstance(rows, torch.Tensor) else rows)]
        if any(r < 0 or r >= n_rows for r in host):
            raise ValueError(f"{name}: rows must be in [0, {n_rows}), got {host[:8]}")
        rows = host
    rows = _int32(name, "rows", rows, None, device)
    nseq = rows.numel()
    cu = None  # where the lengths are known here
    if isinstance(cu_seqlens, Varlen):
        cu, cu_seqlens = cu_seqlens.host, cu_seqlens.cu
    elif cu_seqlens is not None and not (isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda):
        cu = [int(x) for x in (cu_seqlens.tolist() if isinstance(cu_seqlens, torch.Tensor) else cu_seqlens)]
        if len(cu) != nseq + 1 or cu[0] != 0 or cu[-1] != total or any(y < x for x, y in zip(cu, cu[1:])):
            raise ValueError(f"{name}: cu_seqlens must have {nseq + 1} entries, non-decreasing from 0 to {total}, got {cu[:8]}")
        cu_seqlens = cu
    if cu_seqlens is not None:
        cu_seqlens = _int32(name, "cu_seqlens", cu_seqlens, nseq + 1, device)
    elif nseq and total % nseq:
        raise ValueError(f"{name}: {total} tokens do not divide into {nseq} sequences of one length (give cu_seqlens)")
    elif nseq:
        cu = range(0, total + 1, total // nseq) if total else [0] * (nseq + 1)
    if start is None or not (isinstance(start, torch.Tensor) and start.is_cuda):
        first = [0] * nseq if start is None else start.reshape(-1).tolist() if isinstance(start, torch.Tensor) else list(start)
        lens = [0] * nseq if cu is None else [y - x for x, y in zip(cu, cu[1:])]
        for s, (t, n) in enumerate(zip(first, lens)):
            if t < 0 or t + n > length:
                raise ValueError(f"{name}: sequence {s} ({n} tokens from position start = {t}) does not lie in the cache's "
                                 f"{length} positions")
    if start is not None:
        start = _int32(name, "start", start, nseq, device)
    return rows, cu_seqlens, start, nseq


def _rows_16(x):
    """x [tokens, kv, hd] with unit inner stride and 16-byte aligned rows: itself, or a dense copy."""
    per = 16 // x.element_size()
    if x.stride(2) != 1 or x.data_ptr() % 16 or (x.stride(0) % per and x.shape[0] > 1) or (x.stride(1) % per and x.shape[1] > 1):
        x = x.clone(memory_format=torch.contiguous_format)
    return x, x.stride(0) if x.shape[0] > 1 else x.shape[1] * x.shape[2], x.stride(1) if x.shape[1] > 1 else x.shape[2]


def kv_cache_store(cache, k, v, rows, cu_seqlens=None, start=None):
    """Write packed tokens' keys and values into a cache's rows, quantised as they are written when it is e4m3.
    k, v [tokens, kv, hd] bf16, fp16 or fp32 (as a prefill leaves them: any token and head strides, so a transposed view
    of HF's [kv, tokens, hd] needs no copy).  Sequence s is the tokens cu_seqlens[s] .. cu_seqlens[s + 1] (None: equal
    lengths) and goes to positions start[s], start[s] + 1, .. (None: 0) of cache row rows[s].  rows, cu_seqlens and start:
    int32 tensors on the device, or lists / CPU tensors (a Rows / Varlen where one is at hand), which are
    checked.  Of what is on the device, rows and positions outside the cache are not written; no two sequences may write the same place."""
    name = "kv_cache_store"
    code, R, kv, hd, T, index = _check(name, cache)
    _lib.require_cuda(k, v)
    if k.dim() != 3 or k.shape != v.shape or k.shape[1] != kv or k.shape[2] != hd or k.dtype is not v.dtype:
        raise ValueError(f"{name}: k and v must be [tokens, {kv}, {hd}] of one dtype, got {tuple(k.shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    in_code = _lib.dtype_code(k)
    dev = cache.k.device
    if k.get_device() != index or v.get_device() != index:
        raise ValueError(f"{name}: k and v must be on the cache's device {dev}")
    total = k.shape[0]
    rows, cu, start, nseq = _batch(name, rows, cu_seqlens, start, total, R, T, dev)
    if total == 0 or nseq == 0:
        if total:
            raise ValueError(f"{name}: {total} tokens and no rows")
        return
    k, ks, kh = _rows_16(k)
    v, vs, vh = _rows_16(v)
    _lib.call_on(cache.k, "gdn_kv_store", k.data_ptr(), ks, kh, v.data_ptr(), vs, vh, in_code, cache.k.data_ptr(), cache.v.data_ptr(),
              _lib.ptr(cache.k_exp), _lib.ptr(cache.v_exp), code, R, kv, hd, T, rows.data_ptr(), _lib.ptr(cu),
              _lib.ptr(start), nseq, total, _lib.stream_of(k))


def kv_cache_load(cache, rows, cu_seqlens, start=None, total_tokens=None):
    """The keys and values that a cache holds, as packed bf16 rows: sequence s gives positions start[s] .. start[s] +
    (cu_seqlens[s + 1] - cu_seqlens[s]) - 1 of row rows[s].  Arguments as kv_cache_store; with cu_seqlens on the device give
    ``total_tokens`` (its last entry) too, or it is read back.  Returns (k, v) [total_tokens, kv, hd] bf16; rows and
    positions outside the cache (those on the device) are zeros, and tokens that no sequence covers (behind the last one of a padded batch) hold anything."""
    name = "kv_cache_load"
    code, R, kv, hd, T, _ = _check(name, cache)
    dev = cache.k.device
    if total_tokens is None:
        if cu_seqlens is None:
            raise ValueError(f"{name}: give cu_seqlens or total_tokens")
        total_tokens = cu_seqlens.T if isinstance(cu_seqlens, Varlen) else int(cu_seqlens[-1])
    total = int(total_tokens)
    if total < 0:
        raise ValueError(f"{name}: total_tokens must not be negative")
    rows, cu, start, nseq = _batch(name, rows, cu_seqlens, start, total, R, T, dev)
    if total and not nseq:
        raise ValueError(f"{name}: {total} tokens and no rows")
    k, v = torch.empty(2, total, kv, hd, dtype=torch.bfloat16, device=dev).unbind(0)
    if total:
        _lib.call_on(cache.k, "gdn_kv_load", cache.k.data_ptr(), cache.v.data_ptr(), _lib.ptr(cache.k_exp), _lib.ptr(cache.v_exp), code, R,
                  kv, hd, T, rows.data_ptr(), _lib.ptr(cu), _lib.ptr(start), nseq, total, k.data_ptr(), v.data_ptr(),
                  _lib.stream_of(k))
    return k, v


def cached_attn_workspace(cache, n_heads, prefix=None):
    """The workspace cached_decode_attention needs for this cache and prefix cache (allocate once, reuse per layer and
    step; calls that may overlap need one each)."""
    name = "cached_attn_workspace"
    _, N, kv, hd, T, _ = _check(name, cache)
    P, Tp = (prefix.cache.k.shape[0], prefix.cache.length) if prefix is not None else (0, 0)
    nbytes = int(_lib.lib().gdn_attn_cached_workspace_bytes(N, n_heads, kv, hd, T, P, Tp))
    if nbytes < 0:
        raise ValueError(f"{name}: bad sizes")
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=cache.k.device)


def cached_decode_attention(proj, pos, q_norm, k_norm, inv_freq, cache, n_heads, rotary_dim, eps=1e-6, work=None,
                            prefix=None):
    """gqa_decode_attention over a KVCache: after the fused q|gate|k|v projection of one new token per slot, the q/k
    RMSNorms, partial rotary at each slot's position, K and V quantised into the cache, softmax attention over the
    slot's tokens, times sigmoid(gate).  proj [N, (2 nh + 2 kv) hd] bf16 or that projection's Partials; pos int64 [N] on
    the device; the cache's row n is slot n.  ``prefix`` (a SharedPrefix): slots that continue a prefix attend to it as
    well; pos counts from the prefix's beginning, and the slot's own row holds what follows it.  Returns the gated output
    [N, nh * hd] bf16.  Capturable in a graph (with ``work`` kept by the caller)."""
    name = "cached_decode_attention"
    code, N, kv, hd, T, dev = _check(name, cache)
    nh = n_heads
    width = (2 * nh + 2 * kv) * hd
    part = proj if isinstance(proj, Partials) else None
    if part is not None:
        proj = part.data[0]
    elif proj.dtype is not torch.bfloat16:
        raise ValueError(f"{name}: proj must be bfloat16, got {proj.dtype}")
    if proj.shape != (N, width) or pos.dtype is not torch.int64 or pos.numel() != N:
        _lib.require_cuda(proj, pos)
        raise ValueError(f"{name}: bf16 proj [N, (2 nh + 2 kv) hd] = [{N}, {width}] (or partials of that width) and int64 pos [N] "
                         f"for the cache's N = {N} rows expected")
    if q_norm.numel() != hd or k_norm.numel() != hd:
        raise ValueError(f"{name}: q_norm and k_norm must have head_dim = {hd} entries")
    if rotary_dim and inv_freq.numel() != rotary_dim // 2:
        raise ValueError(f"{name}: inv_freq must have rotary_dim / 2 = {rotary_dim // 2} entries")
    if proj.get_device() != dev or pos.get_device() != dev or q_norm.get_device() != dev or k_norm.get_device() != dev \
            or (rotary_dim and inv_freq.get_device() != dev):
        _lib.require_cuda(proj, pos, q_norm, k_norm)
        raise ValueError(f"{name}: every tensor must be on the cache's device {cache.k.device}")
    if part is None and (proj.stride(1) != 1 or (N > 1 and proj.stride(0) < width)):
        proj = proj.contiguous()
    P, Tp, pre = 0, 0, _NO_PREFIX
    if prefix is not None:
        pc, P, pkv, phd, Tp, pdev = _check(name, prefix.cache)
        if (pc, pkv, phd, pdev) != (code, kv, hd, dev):
            raise ValueError(f"{name}: the prefix cache must have the cache's dtype, kv heads, head_dim and device")
        for what, x, n in (("length", prefix.length, P), ("of", prefix.of, N)):
            if x.get_device() != dev or x.dtype is not torch.int32 or x.numel() != n or not x.is_contiguous():
                raise ValueError(f"{name}: prefix.{what} must be a contiguous int32 tensor of {n} entries on the cache's device")
        c = prefix.cache
        pre = (c.k.data_ptr(), c.v.data_ptr(), _lib.ptr(c.k_exp), _lib.ptr(c.v_exp), prefix.length.data_ptr(),
               prefix.of.data_ptr())
    qn = q_norm if q_norm.dtype is torch.bfloat16 and q_norm.is_contiguous() else q_norm.to(torch.bfloat16).contiguous()
    kn = k_norm if k_norm.dtype is torch.bfloat16 and k_norm.is_contiguous() else k_norm.to(torch.bfloat16).contiguous()
    inv = _lib.f32_dense(inv_freq) if rotary_dim else None
    if not pos.is_contiguous():
        pos = pos.contiguous()
    if work is None:
        work = cached_attn_workspace(cache, nh, prefix)
    elif work.get_device() != dev or not work.is_contiguous():
        raise ValueError(f"{name}: work must be a contiguous tensor on the cache's device")
    out = proj.new_empty((N, nh * hd), dtype=torch.bfloat16)
    stride = proj.stride(0) if N > 1 else width
    _lib.call_on(proj, "gdn_attn_cached", None if part is not None else proj.data_ptr(), stride,
              None if part is None else part.data.data_ptr(), 0 if part is None else part.splits,
              pos.data_ptr(), qn.data_ptr(), kn.data_ptr(), _lib.ptr(inv), cache.k.data_ptr(),
              cache.v.data_ptr(), _lib.ptr(cache.k_exp), _lib.ptr(cache.v_exp), code, T, *pre, P, Tp, out.data_ptr(),
              nh * hd, work.data_ptr(), work.numel() * work.element_size(), N, nh, kv, hd, rotary_dim, float(eps),
              _lib.stream_of(proj))
    return out
