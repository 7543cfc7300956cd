"""Serving: attention over whole prompts, a key/value cache held in 4 bits, and the operators that write, read and shrink it.  The
reference has no counterpart (it trains; its forward takes whole sequences of multiples of 128).

The cache is a pool of pages of 128 tokens (the block of the training path), a uint8 tensor [pages, KV heads, RECORD_BYTES] that the caller
owns (`cache_empty`), with a block table int32 [sequences, pages of a sequence] and lengths int32 [sequences] in device memory: no call
waits for the device, and all of them can be captured in a CUDA graph (after a first call outside of one).  Keys and values are symmetric
4-bit codes with a bf16 scale per token and group of 32 channels, 144 bytes per token and head instead of 512."""
from __future__ import annotations

import contextlib

import numpy as np
import torch

from . import _lib, api, ops

PAGE = 128              # FMSA_CACHE_PAGE: tokens of a page
RECORD_BYTES = 18432    # FMSA_CACHE_RECORD_BYTES: a page of one KV head
HEAD_DIM = 128

_KIND_APPEND, _KIND_ATTEND, _KIND_EVICT, _KIND_PROMPT = 4, 5, 6, 7   # passes.StatusBoard.KINDS


def _on(device):
    """Kernels are launched on `device`, whichever device is the current one."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _no_gradients(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or with tensors that need no gradient")


def _activation(name, t):
    if t.ndim != 4:
        raise ValueError(f"{name} must have shape (B, H, S, D)")
    if t.shape[3] != HEAD_DIM:
        raise NotImplementedError("Headdim must be 128")
    if t.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"flash_msa_b200 supports bf16 and fp16 activations, got {t.dtype}")


def _readable(t):
    """`t` as kernels with plain 16-byte loads read it, copied once if it has to be."""
    t = t.detach()
    if t.stride(3) == 1 and not any(s % 8 for s in t.stride()[:3]) and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check_cache(cache):
    if cache.dtype != torch.uint8 or cache.ndim != 3 or cache.shape[2] != RECORD_BYTES or not cache.is_contiguous():
        raise ValueError(f"cache must be a contiguous uint8 tensor [pages, KV heads, {RECORD_BYTES}] (see cache_empty)")
    if cache.shape[0] == 0 or cache.shape[1] == 0 or cache.data_ptr() % 16:
        raise ValueError("cache must hold at least one page and one head, on a 16-byte boundary")


def _check_table(name, table, device, seqs=None):
    if table.dtype != torch.int32 or table.ndim != 2:
        raise TypeError(f"{name} must be int32 [sequences, pages]")
    if table.device != device:
        raise ValueError(f"{name} must be on the cache's device")
    if table.shape[1] == 0 or (table.shape[1] > 1 and table.stride(1) != 1) or (seqs is not None and table.shape[0] != seqs):
        raise ValueError(f"{name} must have a row of at least one page for every sequence, contiguous in itself")


def _check_lengths(lengths, seqs, device):
    if lengths.dtype != torch.int32 or lengths.ndim != 1:
        raise TypeError("lengths must be int32 [sequences]")
    if lengths.device != device or lengths.shape[0] != seqs or not lengths.is_contiguous():
        raise ValueError("lengths must hold one length per row of block_table, contiguous, on the cache's device")


def _check_weights(weights, cache):
    if weights is None:
        return
    if weights.dtype != torch.float32 or weights.shape != (cache.shape[0], cache.shape[1], PAGE) or not weights.is_contiguous():
        raise ValueError("weights must be a contiguous fp32 tensor [pages, KV heads, 128]")
    if weights.device != cache.device:
        raise ValueError("weights must be on the cache's device")


def _cache_arg(cache, table, lengths):
    return _lib.FmsaCache4(cache.data_ptr(), table.data_ptr(), lengths.data_ptr(), table.stride(0), cache.shape[0], cache.shape[1],
                           table.shape[0], table.shape[1])


def _boundaries(cu_seqlens, total, device):
    """Sequence boundaries int32 [n+1] (or [B, n+1]) on the device.  Those in host memory are checked and travel with a kernel launch; those
    in device memory are taken as they are: nothing waits for them, and whatever they hold, no kernel leaves its tensors for it."""
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.device.type == "cuda":
        if cu_seqlens.device != device:
            raise ValueError("cu_seqlens must be on the inputs' device")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError("cu_seqlens must be int32 or int64")
        return cu_seqlens.to(torch.int32).contiguous()
    cu = torch.as_tensor(cu_seqlens).to(torch.int64).numpy()
    if cu.ndim not in (1, 2) or cu.shape[-1] < 2:
        raise ValueError("cu_seqlens must have shape [n+1] or [B, n+1]")
    if (cu[..., 0] != 0).any() or (cu[..., -1] > total).any() or (cu[..., 1:] < cu[..., :-1]).any():
        raise ValueError("cu_seqlens must rise from 0 to at most the sequence length")
    cu = np.ascontiguousarray(cu, dtype=np.int32)
    if cu.size > ops.MAX_HOST_BOUNDARIES:
        return torch.from_numpy(cu).to(device)
    out = torch.empty(cu.shape, dtype=torch.int32, device=device)
    ops._launch("fmsa_boundaries", 1, _lib.load().fmsa_boundaries(cu.ctypes.data, cu.size, out.data_ptr(), ops._stream(device)), device)
    return out


def cache_empty(n_pages: int, n_kv_heads: int, device="cuda") -> torch.Tensor:
    """A pool of `n_pages` pages of 128 tokens.  (Its bytes are zero; nothing is read that was not appended.)"""
    return torch.zeros(int(n_pages), int(n_kv_heads), RECORD_BYTES, dtype=torch.uint8, device=device)


def cache_unpack(cache: torch.Tensor):
    """fp32 (k, v) [..., 128 tokens, 128 channels] of records [..., RECORD_BYTES], in torch operations on any device: for inspection."""
    def scaled(codes, scales, order):
        n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8                      # [..., 128, 128] in stored order
        return n[..., torch.arange(PAGE, device=cache.device)[:, None], order] * scales.contiguous().view(torch.bfloat16).float().repeat_interleave(32, -1)
    token, ch = torch.arange(PAGE, device=cache.device)[:, None], torch.arange(HEAD_DIM, device=cache.device)[None]
    group, rest = ch // 32, ch % 32
    k_order = ((rest // 8) * 32 + group * 8 + rest % 8).expand(PAGE, -1)
    v_order = ((rest // 4) ^ (token & 4)) * 16 + group * 4 + rest % 4
    kc, ks, vc, vs = (cache[..., lo:hi].unflatten(-1, (PAGE, -1)) for lo, hi in ((0, 8192), (8192, 9216), (9216, 17408), (17408, 18432)))
    return scaled(kc, ks, k_order), scaled(vc, vs, v_order)


def cache_append(cache, k, v, block_table, lengths, cu_seqlens=None, weights=None, return_values=False):
    """Stores new keys and values (B,Hkv,n,128) in the cache; `lengths` count them already.  Without `cu_seqlens` batch element i holds the
    last n tokens of sequence i (rows for which lengths[i] < n leaves no place are skipped: an empty place of a padded batch has length
    0).  With `cu_seqlens` ([sequences+1], as in `flash_msa_varlen_func`, but it may end before n) k and v have one batch element, and its
    rows cu_seqlens[i] .. cu_seqlens[i+1]-1 are the last tokens of sequence i.
    `weights`: fp32 [pages, Hkv, 128] as `cache_attention` collects them; those of the stored tokens become zero.  Returns None, or with
    `return_values` (k, v) as the cache now holds them, in the inputs' type: what a prompt's own attention reads if it is to agree with
    the steps that follow (zeros for skipped rows).
    The largest magnitude of 32 channels is stored exactly to bf16's rounding of a seventh of it; others are within half a scale.  A group
    that holds a value that is not finite reads as NaN, one whose values are all below 2^-80 as zeros.  Values are meant to stay below 2^100."""
    _activation("k", k)
    _activation("v", v)
    _no_gradients("flash_msa_cache_append", k, v)
    _check_cache(cache)
    dev = cache.device
    b, h, n, _ = k.shape
    if v.shape != k.shape or h != cache.shape[1]:
        raise ValueError("k and v must agree, and have the cache's KV heads")
    if v.dtype != k.dtype:
        raise TypeError("k and v must have one dtype")
    if k.device != dev or v.device != dev:
        raise ValueError("k, v and the cache must be on one CUDA device")
    _check_table("block_table", block_table, dev)
    seqs = block_table.shape[0]
    _check_lengths(lengths, seqs, dev)
    _check_weights(weights, cache)
    if cu_seqlens is None and b != seqs:
        raise ValueError("k and v must have one batch element per row of block_table (or one, with cu_seqlens)")
    if cu_seqlens is not None and b != 1:
        raise ValueError("packed k and v must have one batch element")
    if cu_seqlens is not None and tuple(torch.as_tensor(cu_seqlens).shape) != (seqs + 1,):
        raise ValueError("cu_seqlens must hold one boundary more than block_table has rows")
    api._require_cuda(cache)
    with _on(dev):
        if cu_seqlens is not None:
            cu_seqlens = _boundaries(cu_seqlens, n, dev)
        values = (ops._grad_like(k.detach()), ops._grad_like(v.detach())) if return_values else None
        if k.numel() and seqs:
            kr, vr = _readable(k), _readable(v)
            status = api._Status(_KIND_APPEND, dev)
            arg = ops._tensor_arg
            ops._launch("fmsa_cache_append", 1, _lib.load().fmsa_cache_append(
                _cache_arg(cache, block_table, lengths), arg(kr), arg(vr), b, n, ops._dtype_code(k.dtype),
                None if cu_seqlens is None else cu_seqlens.data_ptr(), None if weights is None else weights.data_ptr(),
                arg(values[0]) if values else None, arg(values[1]) if values else None, status.ptr, ops._stream(dev)), dev)
            status.check()
    return values


def cache_attention(q, cache, block_table, lengths, scale: float, sinks=None, weights=None, accumulate=True):
    """Attention of the last n tokens of every sequence, q (B,Hq,n,128), over the cache, which holds those tokens already: query j of
    sequence i sees its first lengths[i] - n + 1 + j tokens.  Returns [B, n, Hq*128]; a row that sees no token is zero.  `sinks` as in
    `flash_msa_func`.  `weights`: fp32 [pages, Hkv, 128]: the probability every token got from this call, summed over its KV head's query
    rows, is added, or written with `accumulate=False` (what `cache_evict` goes by).  With weights, no two sequences may name one page."""
    _activation("q", q)
    _no_gradients("flash_msa_cache_func", q, sinks)
    _check_cache(cache)
    dev = cache.device
    b, hq, n, _ = q.shape
    if q.device != dev:
        raise ValueError("q and the cache must be on one CUDA device")
    if hq == 0 or hq % cache.shape[1]:
        raise ValueError("n_heads must be divisible by n_kv_heads")
    _check_table("block_table", block_table, dev, b)
    _check_lengths(lengths, b, dev)
    _check_weights(weights, cache)
    sinks = api._check_sinks(sinks, q)
    api._require_cuda(cache)
    out = torch.empty(b, n, hq * HEAD_DIM, dtype=q.dtype, device=dev)
    if not out.numel():
        return out
    with _on(dev):
        lib = _lib.load()
        qr, logits = _readable(q), api._sink_logits(sinks)
        nbytes = lib.fmsa_cache_attend_workspace_bytes(b, hq, cache.shape[1], n)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
        status = api._Status(_KIND_ATTEND, dev)
        ops._launch("fmsa_cache_attend", 2 if weights is None else 3, lib.fmsa_cache_attend(
            _cache_arg(cache, block_table, lengths), ops._tensor_arg(qr), hq, n, float(scale), ops._dtype_code(q.dtype),
            None if logits is None else logits.data_ptr(), None if weights is None else weights.data_ptr(), int(bool(accumulate)),
            out.data_ptr(), ws.data_ptr(), nbytes, status.ptr, ops._stream(dev)), dev)
        status.check()
    return out


def cache_evict(cache, weights, block_table, lengths, new_block_table, keep: int, recent: int):
    """Cuts every sequence to `keep` tokens per KV head: the last `recent` ones, and the others of the largest `weights` (ties: the earlier
    one; NaN counts as the largest).  What stays is copied, in its order and with its weights, to the pages that `new_block_table` (int32
    [sequences, at least keep/128 pages]) names; a sequence of at most `keep` tokens is copied whole.  Those pages must be named by no
    other row of either table; the old ones are only read, so pages that sequences share stay what they are.
    Returns (new lengths int32 [B], kept int32 [B, Hkv, keep]: the places the tokens had, -1 behind the last)."""
    _check_cache(cache)
    dev = cache.device
    keep, recent = int(keep), int(recent)
    if weights is None:
        raise ValueError("weights must be a contiguous fp32 tensor [pages, KV heads, 128]")
    _check_weights(weights, cache)
    _check_table("block_table", block_table, dev)
    b = block_table.shape[0]
    _check_lengths(lengths, b, dev)
    _check_table("new_block_table", new_block_table, dev, b)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError("keep must be positive and recent between 0 and keep")
    if new_block_table.shape[1] * PAGE < keep:
        raise ValueError(f"new_block_table has room for {new_block_table.shape[1] * PAGE} tokens, keep is {keep}")
    api._require_cuda(cache)
    new_lengths = torch.empty(b, dtype=torch.int32, device=dev)
    kept = torch.empty(b, cache.shape[1], keep, dtype=torch.int32, device=dev)
    if not b:
        return new_lengths, kept
    with _on(dev):
        status = api._Status(_KIND_EVICT, dev)
        ops._launch("fmsa_cache_evict", 2, _lib.load().fmsa_cache_evict(
            _cache_arg(cache, block_table, lengths), weights.data_ptr(), new_block_table.data_ptr(), new_block_table.stride(0),
            new_block_table.shape[1], keep, recent, new_lengths.data_ptr(), kept.data_ptr(), status.ptr, ops._stream(dev)), dev)
        status.check()
    return new_lengths, kept


def _tma_readable(t):
    """`t` as tile loads read it, copied once if it has to be."""
    t = t.detach()
    st = t.stride()
    if st[3] == 1 and all(s > 0 and s % 8 == 0 for s in st[:3]) and st[2] >= HEAD_DIM and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def prompt_attention(q, k, v, cu_seqlens, scale: float, sinks=None):
    """Dense causal attention over whole prompts of any length, heads grouped: q (B,Hq,S,128), k and v (B,Hkv,S,128), Hq/Hkv at most 128.
    Returns [B, S, Hq*128].  `cu_seqlens` None: every batch element is one sequence.  Otherwise [n+1], or [B,n+1] for a packing per batch
    element: the rows cu_seqlens[i] .. cu_seqlens[i+1]-1 are sequence i, a row sees the rows of its own sequence up to itself; it starts
    at 0 and may end before S (rows behind the last sequence come back zero, whatever they hold).  Boundaries in host memory are checked;
    those in device memory are not waited for, and have to rise from 0 to at most S.  `sinks` as in `flash_msa_func`; scale > 0.
    For serving: it keeps nothing for a backward (training: `flash_msa_func`, `flash_msa_warmup_func`)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        _activation(name, t)
    _no_gradients("flash_msa_prompt_func", q, k, v, sinks)
    b, hq, s, _ = q.shape
    hkv = k.shape[1]
    if k.shape != v.shape or k.shape[0] != b or k.shape[2] != s:
        raise ValueError("q, k, and v must agree on batch, sequence, head dimension, and KV head count")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError("n_heads must be divisible by n_kv_heads")
    if hq // hkv > 128:
        raise NotImplementedError("at most 128 heads may share a KV head")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError("q, k, and v must have one dtype")
    dev = q.device
    if k.device != dev or v.device != dev:
        raise ValueError("q, k, and v must be on one CUDA device")
    if not scale > 0:
        raise ValueError("scale must be positive")
    sinks = api._check_sinks(sinks, q)
    if cu_seqlens is not None:
        shape = tuple(torch.as_tensor(cu_seqlens).shape)
        if len(shape) not in (1, 2) or shape[-1] < 2 or (len(shape) == 2 and shape[0] != b):
            raise ValueError("cu_seqlens must have shape [n+1] or [B, n+1]")
    api._require_cuda(q)
    out = torch.empty(b, s, hq * HEAD_DIM, dtype=q.dtype, device=dev)
    if not out.numel():
        return out
    with _on(dev):
        lib = _lib.load()
        n_seqs, per_batch = 1, 0
        if cu_seqlens is not None:
            cu_seqlens = _boundaries(cu_seqlens, s, dev)
            n_seqs, per_batch = cu_seqlens.shape[-1] - 1, int(cu_seqlens.ndim == 2)
        qr, kr, vr, logits = _tma_readable(q), _tma_readable(k), _tma_readable(v), api._sink_logits(sinks)
        nbytes = lib.fmsa_prompt_workspace_bytes(b, s, hq, hkv, n_seqs)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
        status = api._Status(_KIND_PROMPT, dev)
        ops._launch("fmsa_prompt_fwd", 2, lib.fmsa_prompt_fwd(
            ops._tensor_arg(qr), ops._tensor_arg(kr), ops._tensor_arg(vr), b, s, hq, hkv,
            None if cu_seqlens is None else cu_seqlens.data_ptr(), n_seqs, per_batch, float(scale), ops._dtype_code(q.dtype),
            None if logits is None else logits.data_ptr(), out.data_ptr(), ws.data_ptr(), nbytes, status.ptr, ops._stream(dev)), dev)
        status.check()
    return out
