"""Serving: attention over whole prompts, a key/value cache held in 4 bits, and the operators that write, read and shrink it.  The
reference has no counterpart (it trains; its forward takes whole sequences of multiples of 128).

The cache is a pool of pages of 128 tokens (the block of the training path), a uint8 tensor [pages, KV heads, RECORD_BYTES] that the caller
owns (`cache_empty`), with a block table int32 [sequences, pages of a sequence] and lengths int32 [sequences] in device memory: no call
waits for the device, and all of them can be captured in a CUDA graph (after a first call outside of one).  What those tensors hold the
kernels check: a sequence whose length is beyond its row of the table counts as empty in every call, pages that do not exist are not
touched and attention passes over their tokens, boundaries in device memory that do not rise leave rows undefined; each of these raises, at a later
call or in `check_pending_status()`.  A length below zero is zero.  Keys and values are symmetric 4-bit codes with a bf16 scale per token and group of 32
channels, 144 bytes per token and head instead of 512."""
from __future__ import annotations

import struct

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib, api, ops, passes

PAGE = 128              # FMSA_CACHE_PAGE: tokens of a page
RECORD_BYTES = 18432    # FMSA_CACHE_RECORD_BYTES: a page of one KV head
HEAD_DIM = 128

_KIND_APPEND, _KIND_ATTEND, _KIND_EVICT, _KIND_PROMPT = 4, 5, 6, 7   # passes.StatusBoard.KINDS

# The argument blocks of the header.  One call packs a block: a ctypes structure filled field by field and as many arguments as a block has
# fields took a third of a small call's host time (28 us of which the GPU needs 11, one sequence of 1000 tokens).
_CACHE, _TENSOR = "PPPqiiii", "Pqqq"
_APPEND_ARGS = struct.Struct("@" + _CACHE + 4 * _TENSOR + "PPP" + "iiii")
_ATTEND_ARGS = struct.Struct("@" + _CACHE + _TENSOR + "PPPPqP" + "iiiifi")
_EVICT_ARGS = struct.Struct("@" + _CACHE + "PPqPPP" + "iiii")
_PROMPT_ARGS = struct.Struct("@" + 3 * _TENSOR + "PPPPqP" + "iiiiiiif")
_NO_TENSOR = (0, 0, 0, 0)


_current_device = torch._C._cuda_getDevice
_stream = torch._C._cuda_getCurrentRawStream


def _call(what, launches, fn, block, device):
    """Launches on `device` (an index), whichever device is the current one, on its current stream."""
    if device != _current_device():
        with torch.cuda.device(device):
            return _call(what, launches, fn, block, device)
    if ops.KERNEL_EVENTS is None:
        status = fn(block, _stream(device))
    else:
        with ops._Timed(what, torch.device("cuda", device)):
            status = fn(block, _stream(device))
    if status:
        _lib.check(status, what)
    ops.LAUNCHES += launches


class _Word:
    """Address of the status word of a call of this kind (see `api._Status`, whose word of its own it uses for debugging)."""

    __slots__ = ("own", "ptr")

    def __init__(self, kind, device):
        self.own = api._Status(kind, torch.device("cuda", device)) if api.DEBUG_CHECK_STATUS else None
        self.ptr = self.own.ptr if self.own else passes.status_board.pointer(kind, device)

    def check(self):
        if self.own:
            self.own.check()


def _no_gradients(what, *tensors):
    """These calls keep nothing for a backward, have no tangents and leave nothing in a trace: what would get lost is refused."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or with tensors that need no gradient")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative")
    if torch._C._is_tracing():
        raise RuntimeError(f"{what} cannot be traced")


def _activation(name, t):
    """The shape of an activation."""
    shape = t.shape
    if len(shape) != 4:
        raise ValueError(f"{name} must have shape (B, H, S, D)")
    if shape[3] != HEAD_DIM:
        raise NotImplementedError("Headdim must be 128")
    if t.dtype is not torch.bfloat16 and t.dtype is not torch.float16:
        raise TypeError(f"flash_msa_b200 supports bf16 and fp16 activations, got {t.dtype}")
    return shape


def _readable(t):
    """(`t` as kernels with plain 16-byte loads read it, copied once if it has to be; address and strides)."""
    sb, sh, ss, sd = t.stride()
    ptr = t.data_ptr()
    if sd != 1 or (sb | sh | ss) & 7 or ptr & 15:
        t = t.detach().clone(memory_format=torch.contiguous_format)
        sb, sh, ss, _ = t.stride()
        ptr = t.data_ptr()
    return t, (ptr, sb, sh, ss)


def _tma_readable(t):
    """The same for tile loads."""
    sb, sh, ss, sd = t.stride()
    ptr = t.data_ptr()
    if sd != 1 or (sb | sh | ss) & 7 or ptr & 15 or sb <= 0 or sh <= 0 or ss < HEAD_DIM:
        t = t.detach().clone(memory_format=torch.contiguous_format)
        sb, sh, ss, _ = t.stride()
        ptr = t.data_ptr()
    return t, (ptr, sb, sh, ss)


def _check_cache(cache, table, lengths, weights, seqs=None):
    """Checks what the calls on a cache share.  Returns the fields of its argument block, the number of sequences and the device's index."""
    shape = cache.shape
    if cache.dtype is not torch.uint8 or len(shape) != 3 or shape[2] != RECORD_BYTES or not cache.is_contiguous():
        raise ValueError(f"cache must be a contiguous uint8 tensor [pages, KV heads, {RECORD_BYTES}] (see cache_empty)")
    pages, heads, _ = shape
    records = cache.data_ptr()
    if pages == 0 or heads == 0 or records & 15:
        raise ValueError("cache must hold at least one page and one head, on a 16-byte boundary")
    device = cache.get_device()   # (-1: host memory)
    (n, width), stride = _check_table("block_table", table, device)
    if seqs is not None and n != seqs:
        raise ValueError("block_table must have a row for every sequence")
    if lengths.dtype is not torch.int32 or lengths.ndim != 1:
        raise TypeError("lengths must be int32 [sequences]")
    if lengths.shape[0] != n or lengths.get_device() != device or not lengths.is_contiguous():
        raise ValueError("lengths must hold one length per row of block_table, contiguous, on the cache's device")
    if weights is not None:
        if weights.dtype is not torch.float32 or weights.shape != (pages, heads, PAGE) or not weights.is_contiguous():
            raise ValueError("weights must be a contiguous fp32 tensor [pages, KV heads, 128]")
        if weights.get_device() != device:
            raise ValueError("weights must be on the cache's device")
    return (records, table.data_ptr(), lengths.data_ptr(), stride, pages, heads, n, width), n, device


def _check_table(name, table, device):
    shape = table.shape
    if table.dtype is not torch.int32 or len(shape) != 2:
        raise TypeError(f"{name} must be int32 [sequences, pages]")
    if table.get_device() != device:
        raise ValueError(f"{name} must be on the cache's device")
    stride, inner = table.stride()
    if shape[1] == 0 or (inner != 1 and shape[1] > 1) or stride < 0:
        raise ValueError(f"{name} must have a row of at least one page for every sequence, contiguous in itself")
    return shape, stride


def _require_cuda(device):
    if device < 0:
        raise RuntimeError("flash_msa_b200 requires CUDA tensors (there is no CPU path)")


def _boundaries(cu_seqlens, total, device):
    """Sequence boundaries int32 [n+1] (or [B, n+1]) on the device.  Those in host memory are checked and travel with kernel launches; those
    in device memory are not waited for: the kernels report what does not rise from 0 to at most the rows there are, and leave their tensors for
    nothing."""
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.device.type == "cuda":
        if cu_seqlens.device != device:
            raise ValueError("cu_seqlens must be on the inputs' device")
        if cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise TypeError("cu_seqlens must be int32 or int64")
        return cu_seqlens if cu_seqlens.dtype is torch.int32 and cu_seqlens.is_contiguous() else cu_seqlens.to(torch.int32).contiguous()
    cu = torch.as_tensor(cu_seqlens).to(torch.int64).numpy()
    if cu.ndim not in (1, 2) or cu.shape[-1] < 2:
        raise ValueError("cu_seqlens must have shape [n+1] or [B, n+1]")
    if (cu[..., 0] != 0).any() or (cu[..., -1] > total).any() or (cu[..., 1:] < cu[..., :-1]).any():
        raise ValueError("cu_seqlens must rise from 0 to at most the sequence length")
    cu = np.ascontiguousarray(cu, dtype=np.int32)
    out = torch.empty(cu.shape, dtype=torch.int32, device=device)
    with torch.cuda.device(device):
        _send_boundaries(cu.ctypes.data, cu.size, out.data_ptr(), ops._stream(device), device)
    return out


def _send_boundaries(src, n, dst, stream, device):
    """`n` boundaries from host to device memory, as parameters of as many launches as that takes (a copy from memory that is not pinned would
    wait for the device, and could not be captured)."""
    for at in range(0, n, ops.MAX_HOST_BOUNDARIES):
        count = min(n - at, ops.MAX_HOST_BOUNDARIES)
        ops._launch("fmsa_boundaries", 1, _lib.load().fmsa_boundaries(src + 4 * at, count, dst + 4 * at, stream), device)


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
    rows cu_seqlens[i] .. cu_seqlens[i+1]-1 are the last tokens of sequence i.  No two sequences may name a page that either appends to.
    `weights`: fp32 [pages, Hkv, 128] as `cache_attention` collects them; those of the stored tokens become zero.  Returns None, or with
    `return_values` (k, v) as the cache now holds them, in the inputs' type: what a prompt's own attention reads if it is to agree with
    the steps that follow (zeros for skipped rows).
    The largest magnitude of 32 channels is stored exactly to bf16's rounding of a seventh of it; others are within half a scale.  A group
    that holds a value that is not finite reads as NaN, one whose values are all below 2^-80 as zeros.  Values are meant to stay below 2^100."""
    shape = _activation("k", k)
    if _activation("v", v) != shape:
        raise ValueError("k and v must agree, and have the cache's KV heads")
    if v.dtype is not k.dtype:
        raise TypeError("k and v must have one dtype")
    _no_gradients("flash_msa_cache_append", k, v, weights)
    b, h, n, _ = shape
    fields, seqs, dev = _check_cache(cache, block_table, lengths, weights)
    if h != fields[5]:
        raise ValueError("k and v must agree, and have the cache's KV heads")
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k, v and the cache must be on one CUDA device")
    if cu_seqlens is None:
        if b != seqs:
            raise ValueError("k and v must have one batch element per row of block_table (or one, with cu_seqlens)")
    elif b != 1:
        raise ValueError("packed k and v must have one batch element")
    elif tuple(cu_seqlens.shape if isinstance(cu_seqlens, torch.Tensor) else torch.as_tensor(cu_seqlens).shape) != (seqs + 1,):
        raise ValueError("cu_seqlens must hold one boundary more than block_table has rows")
    _require_cuda(dev)
    k, kf = _readable(k)
    v, vf = _readable(v)
    values, to = None, _NO_TENSOR + _NO_TENSOR
    if return_values:   # (in the inputs' layout; what is readable has its channels innermost and strides of multiples of 8, and so have these)
        ko, vo = values = torch.empty_like(k), torch.empty_like(v)
        to = (ko.data_ptr(), *ko.stride()[:3], vo.data_ptr(), *vo.stride()[:3])
    if b and h and n:
        if cu_seqlens is not None:
            cu_seqlens = _boundaries(cu_seqlens, n, cache.device)
        word = _Word(_KIND_APPEND, dev)
        _call("fmsa_cache_append", 1, _lib.load().fmsa_cache_append, _APPEND_ARGS.pack(
            *fields, *kf, *vf, *to, 0 if cu_seqlens is None else cu_seqlens.data_ptr(), 0 if weights is None else weights.data_ptr(), word.ptr,
            b, n, ops._dtype_code(k.dtype), 0), dev)
        word.check()
    return values


_plans = {}   # what the library says of (operator, device, sizes)


def _plan(device, entry, *sizes):
    """(bytes of the workspace - none where one launch is all -, launches)."""
    key = (entry, device, *sizes)
    got = _plans.get(key)
    if got is None:
        if len(_plans) >= 1024:
            _plans.clear()
        lib = _lib.load()
        with torch.cuda.device(device):
            got = _plans[key] = max(getattr(lib, entry + "_workspace_bytes")(*sizes), 0), getattr(lib, entry + "_launches")(*sizes)
    return got


def cache_attention(q, cache, block_table, lengths, scale: float, sinks=None, weights=None, accumulate=True):
    """Attention of the last n tokens of every sequence, q (B,Hq,n,128), over the cache, which holds those tokens already: query j of
    sequence i sees its first lengths[i] - n + 1 + j tokens.  Returns [B, n, Hq*128]; a row that sees no token is zero.  `sinks` as in
    `flash_msa_func`.  `weights`: fp32 [pages, Hkv, 128]: the probability every token got from this call, summed over its KV head's query
    rows, is added, or written with `accumulate=False` (what `cache_evict` goes by).  With weights, no two sequences may name one page.
    Kernels are chosen by the width of the table: few short sequences are fastest under one that is not much wider than they need.  Of V, a group
    of 32 channels keeps its accuracy down to 2^-20 of its token's largest."""
    b, hq, n, _ = _activation("q", q)
    _no_gradients("flash_msa_cache_func", q, sinks, weights)
    fields, _, dev = _check_cache(cache, block_table, lengths, weights, b)
    if q.get_device() != dev:
        raise ValueError("q and the cache must be on one CUDA device")
    hkv = fields[5]
    if hq == 0 or hq % hkv:
        raise ValueError("n_heads must be divisible by n_kv_heads")
    logits = None if sinks is None else api._sink_logits(api._check_sinks(sinks, q))
    _require_cuda(dev)
    out = q.new_empty((b, n, hq * HEAD_DIM))
    if b == 0 or n == 0:
        return out
    lib = _lib.load()
    nbytes, launches = _plan(dev, "fmsa_cache_attend", b, hq, hkv, n, fields[7], 0 if weights is None else 1)
    q, qf = _readable(q)
    ws = cache.new_empty(nbytes) if nbytes else None
    word = _Word(_KIND_ATTEND, dev)
    _call("fmsa_cache_attend", launches, lib.fmsa_cache_attend, _ATTEND_ARGS.pack(
        *fields, *qf, 0 if logits is None else logits.data_ptr(), 0 if weights is None else weights.data_ptr(), out.data_ptr(),
        0 if ws is None else ws.data_ptr(), nbytes, word.ptr, hq, n, ops._dtype_code(q.dtype), 1 if accumulate else 0, scale, 0), dev)
    word.check()
    return out


def cache_evict(cache, weights, block_table, lengths, new_block_table, keep: int, recent: int):
    """Cuts every sequence to `keep` tokens per KV head: the last `recent` ones, and the others of the largest `weights` (ties: the earlier
    one; NaN counts as the largest).  What stays is copied, in its order and with its weights, to the pages that `new_block_table` (int32
    [sequences, at least keep/128 pages]) names; a sequence of at most `keep` tokens is copied whole.  Those pages must be named by no
    other row of either table; the old ones are only read, so pages that sequences share stay what they are.  (Tokens of pages that do not exist,
    which is reported, count less than any weight and are copied as zeros.)
    Returns (new lengths int32 [B], kept int32 [B, Hkv, keep]: the places the tokens had, -1 behind the last)."""
    keep, recent = int(keep), int(recent)
    if weights is None:
        raise ValueError("weights must be a contiguous fp32 tensor [pages, KV heads, 128]")
    _no_gradients("flash_msa_cache_evict", weights)
    fields, b, dev = _check_cache(cache, block_table, lengths, weights)
    (rows, width), stride = _check_table("new_block_table", new_block_table, dev)
    if rows != b:
        raise ValueError("new_block_table must have a row for every sequence")
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError("keep must be positive and recent between 0 and keep")
    if width * PAGE < keep:
        raise ValueError(f"new_block_table has room for {width * PAGE} tokens, keep is {keep}")
    _require_cuda(dev)
    new_lengths, kept = lengths.new_empty(b), lengths.new_empty((b, fields[5], keep))
    if b:
        word = _Word(_KIND_EVICT, dev)
        _call("fmsa_cache_evict", 2, _lib.load().fmsa_cache_evict, _EVICT_ARGS.pack(
            *fields, weights.data_ptr(), new_block_table.data_ptr(), stride, new_lengths.data_ptr(), kept.data_ptr(), word.ptr, width, keep, recent, 0), dev)
        word.check()
    return new_lengths, kept


def prompt_attention(q, k, v, cu_seqlens, scale: float, sinks=None):
    """Dense causal attention over whole prompts of any length, heads grouped: q (B,Hq,S,128), k and v (B,Hkv,S,128), Hq/Hkv at most 128.
    Returns [B, S, Hq*128].  `cu_seqlens` None: every batch element is one sequence.  Otherwise [n+1], or [B,n+1] for a packing per batch
    element: the rows cu_seqlens[i] .. cu_seqlens[i+1]-1 are sequence i, a row sees the rows of its own sequence up to itself; it starts
    at 0 and may end before S (rows behind the last sequence come back zero, whatever they hold).  Boundaries in host memory are checked;
    those in device memory are not waited for, and have to rise from 0 to at most S (which is reported like the status of other calls, and what
    came back then undefined).  `sinks` as in `flash_msa_func`; scale > 0.
    For serving: it keeps nothing for a backward (training: `flash_msa_func`, `flash_msa_warmup_func`)."""
    b, hq, s, _ = _activation("q", q)
    shape = _activation("k", k)
    if _activation("v", v) != shape or shape[0] != b or shape[2] != s:
        raise ValueError("q, k, and v must agree on batch, sequence, head dimension, and KV head count")
    hkv = shape[1]
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError("n_heads must be divisible by n_kv_heads")
    if hq // hkv > 128:
        raise NotImplementedError("at most 128 heads may share a KV head")
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise TypeError("q, k, and v must have one dtype")
    dev = q.get_device()
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("q, k, and v must be on one CUDA device")
    if not scale > 0:
        raise ValueError("scale must be positive")
    _no_gradients("flash_msa_prompt_func", q, k, v, sinks)
    logits = None if sinks is None else api._sink_logits(api._check_sinks(sinks, q))
    n_seqs, per_batch = 1, 0
    if cu_seqlens is not None:
        shape = tuple(cu_seqlens.shape if isinstance(cu_seqlens, torch.Tensor) else torch.as_tensor(cu_seqlens).shape)
        if len(shape) not in (1, 2) or shape[-1] < 2 or (len(shape) == 2 and shape[0] != b):
            raise ValueError("cu_seqlens must have shape [n+1] or [B, n+1]")
        n_seqs, per_batch = shape[-1] - 1, len(shape) - 1
    _require_cuda(dev)
    out = q.new_empty((b, s, hq * HEAD_DIM))
    if b == 0 or s == 0:
        return out
    lib = _lib.load()
    if cu_seqlens is not None:
        cu_seqlens = _boundaries(cu_seqlens, s, q.device)
    q, qf = _tma_readable(q)
    k, kf = _tma_readable(k)
    v, vf = _tma_readable(v)
    nbytes, launches = _plan(dev, "fmsa_prompt", b, s, hq, hkv, n_seqs)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    word = _Word(_KIND_PROMPT, dev)
    _call("fmsa_prompt_fwd", launches, lib.fmsa_prompt_fwd, _PROMPT_ARGS.pack(
        *qf, *kf, *vf, 0 if cu_seqlens is None else cu_seqlens.data_ptr(), 0 if logits is None else logits.data_ptr(), out.data_ptr(),
        0 if ws is None else ws.data_ptr(), nbytes, word.ptr, b, s, hq, hkv, n_seqs, per_batch, ops._dtype_code(q.dtype), scale), dev)
    word.check()
    return out
