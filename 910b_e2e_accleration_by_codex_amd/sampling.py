"""Sampling from a decode step's logits: temperature, top-k, top-p and min-p with given random numbers.

The reference's engine takes the argmax (src/cb_engine.py:170-172); temperature 0 is that argmax.
"""
import torch

from . import _lib


def sample_workspace(n_rows, vocab, device):
    """The workspace sample_tokens needs for these sizes (allocate once; calls that may overlap need one each)."""
    nbytes = int(_lib.lib().gdn_sample_workspace_bytes(n_rows, vocab))
    if nbytes < 0:
        raise ValueError("sample_workspace: bad sizes")
    return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)


def _param(what, x, N, dtype, device):
    """(device pointer or None, value, tensor kept alive): a number for every row, or a tensor [N] on the device."""
    if not isinstance(x, torch.Tensor):
        return None, x, None
    if dtype is torch.int32 and (x.dtype.is_floating_point or x.dtype is torch.bool):
        raise TypeError(f"sample_tokens: {what} must be whole numbers, got {x.dtype}")
    if not x.is_cuda or x.device != device or x.numel() != N:
        raise ValueError(f"sample_tokens: {what} must be a number or a tensor of {N} entries on {device}")
    if x.dtype is torch.int64 and dtype is torch.int32:
        x = x.clamp(-1, 2 ** 31 - 1)
    if x.dtype is not torch.float64 or dtype is torch.int32:
        x = x.to(dtype)
    x = x.reshape(-1).contiguous()
    return x.data_ptr(), 0, x


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, work=None):
    """One token per row: int64 [N].  logits [N, V] bf16, fp16 or fp32 (a step's output; unit inner stride); u [N] fp32 or
    fp64 in [0, 1), the rows' random numbers.  temperature, top_k, top_p, min_p: numbers (as doubles), or tensors [N] on
    the device (one per request; fp64 ones as they are, others as fp32, top_k as int32).

    With w_i = exp((l_i - max l) / temperature): of the top_k largest logits (<= 0: all; ties go to the lowest index),
    of these the fewest most likely whose mass reaches top_p of their mass, of these those with w_i >= min_p, the
    first index whose running sum of weights exceeds u times their whole sum.  temperature <= 0: the first index of the maximum.
    -inf and NaN logits are never taken; a row of nothing else gives -1.  The same inputs always give the same tokens.
    Capturable in a graph (with ``work`` kept by the caller)."""
    _lib.require_cuda(logits, u)
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError("sample_tokens: logits must be [N, V]")
    N, V = logits.shape
    dev = logits.device
    code = _lib.dtype_code(logits)
    if u.dtype not in (torch.float32, torch.float64) or u.numel() != N or u.device != dev:
        raise ValueError(f"sample_tokens: u must be fp32 or fp64 [{N}] on {dev}")
    # `not (a <= x <= b)` refuses NaN as well
    for what, x, lo, hi in (("temperature", temperature, -1e300, 1e300), ("top_p", top_p, 0, 1), ("min_p", min_p, 0, 1),
                            ("top_k", top_k, -2 ** 31, 2 ** 31 - 1)):
        if not isinstance(x, torch.Tensor) and not lo <= x <= hi:
            raise ValueError(f"sample_tokens: {what} = {x} is outside [{lo}, {hi}]")
    if not isinstance(top_k, torch.Tensor) and int(top_k) != top_k:
        raise TypeError(f"sample_tokens: top_k must be a whole number, got {top_k}")
    t, t1, keep_t = _param("temperature", temperature, N, torch.float32, dev)
    k, k1, keep_k = _param("top_k", top_k, N, torch.int32, dev)
    p, p1, keep_p = _param("top_p", top_p, N, torch.float32, dev)
    m, m1, keep_m = _param("min_p", min_p, N, torch.float32, dev)
    f64 = sum(bit for bit, x in ((1, u), (2, keep_t), (4, keep_p), (8, keep_m)) if x is not None and x.dtype is torch.float64)
    if logits.stride(1) != 1 or (N > 1 and logits.stride(0) < V):  # (one row for all, too)
        logits = logits.contiguous()
    u = u.contiguous()
    out = torch.empty(N, dtype=torch.int64, device=dev)
    if N == 0:
        return out
    if work is None:
        work = sample_workspace(N, V, dev)
    elif not work.is_cuda or work.device != dev or not work.is_contiguous():
        raise ValueError(f"sample_tokens: work must be a contiguous tensor on {dev}")
    _lib.call_on(logits, "gdn_sample", logits.data_ptr(), logits.stride(0) if N > 1 else V, code, u.data_ptr(),
              f64, t, k, p, m, float(t1), int(k1), float(p1), float(m1), out.data_ptr(), N, V,
              work.data_ptr(), work.numel() * work.element_size(), _lib.stream_of(logits))
    return out
