"""Workloads of the serving operators: attention over a whole prompt, and a key/value cache held in 4 bits with what writes it,
reads it and shrinks it.

`run` computes a case in plain torch operations, or, with `own = True`, through the public functions of `flash_msa_b200`; `exact`
computes it in 64 bits.

The cache is a pool of records, uint8 [pages, KV heads, 18432], of 128 tokens each: K codes [128][64 bytes], K scales bf16 [128][4],
V codes [128][64 bytes], V scales bf16 [128][4].  A value is (nibble - 8) * the scale of its token and group of 32 channels.
  K: 16-byte chunk t (0..3) of a row, 32-bit word i (0..3) of the chunk, nibble j (0..7) of the word: channel 32 i + 8 t + j.
  V: 8-byte chunk c (0..7) of token n's row stands at place c ^ (n & 4); its halfword i (0..3), nibble j (0..3): channel 32 i + 4 c + j.
"""
import math

import numpy as np
import torch

own = False

D, PAGE, RECORD = 128, 128, 18432
SCALE = D ** -0.5
K_CODES, K_SCALES, V_CODES, V_SCALES = (0, 8192), (8192, 9216), (9216, 17408), (17408, 18432)


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------

def _case(op, **kw):
    base = dict(op=op, b=1, hq=8, hkv=2, dtype="bf16", layout="bhsd")
    if op == "append":
        base.update(n=1, longest=1024, packed=0)
    elif op == "attend":
        base.update(n=1, longest=1024, sinks=False, weights=False)
    elif op == "evict":
        base.update(longest=1024, keep=512, recent=64)
    elif op == "prompt":
        base.update(s=1024, docs=0, tail=0, sinks=False)
    return dict(base, **kw)


def listed():
    return [
        # One sequence, one new token: what a chat with a single user pays per layer and step for storing it.  Latency.
        _case("append", name="append_step_b1", longest=1000),
        # A full batch, three new tokens each (a draft that is to be checked), activations as a model holds them.
        _case("append", name="append_step_b64", b=64, hkv=8, n=3, longest=8000, dtype="fp16", layout="bshd"),
        # Prompts of a packed prefill going into the cache: seven sequences of unequal length.
        _case("append", name="append_prompt_32k", hkv=8, n=32768, packed=7, longest=0, layout="bshd"),
        # The smallest step: one sequence, a few pages.  Latency.
        _case("attend", name="attend_b1_s1000", hq=16, hkv=2, longest=1000),
        # A serving batch of the 8K shape, lengths from a few tokens to 8K.
        _case("attend", name="attend_b32_s8192", b=32, hq=32, hkv=8, longest=8192),
        # Two long sequences and one KV head: the work has to be split along the sequence.
        _case("attend", name="attend_b2_s65536", b=2, hq=8, hkv=1, longest=65536, dtype="fp16"),
        # Four tokens at once under twelve heads per KV head, with sinks, leaving the weights that an eviction goes by.
        _case("attend", name="attend_b16_n4_weights", b=16, hq=48, hkv=4, n=4, longest=6001, sinks=True, weights=True),
        # One short sequence over its budget.  Latency.
        _case("evict", name="evict_b1_s1100", longest=1100, keep=512, recent=64),
        # A batch at 8K that is cut to half.
        _case("evict", name="evict_b32_s8192", b=32, hkv=8, longest=8192, keep=4000, recent=256),
        # A prefill step of four short prompts of odd lengths, with rows behind the last one.
        _case("prompt", name="prompt_s333_packed", s=333, docs=4, tail=13, hq=16, hkv=2),
        # Packed prefill at 8K: eleven prompts of unequal length, five heads per KV head, sinks.
        _case("prompt", name="prompt_s8100_packed", s=8100, docs=11, hq=20, hkv=4, dtype="fp16", layout="bshd", sinks=True),
        # One 8K prompt at the heads of the benchmark configuration.
        _case("prompt", name="prompt_s8192", s=8192, hq=32, hkv=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One case of the same ranges: one to 64 sequences, lengths from one token to 64K, one to eight KV heads, up to sixteen heads per
    KV head, one to five tokens per step, prompts to 8K of up to sixteen sequences."""
    while True:
        op = rng.choice(["append", "attend", "attend", "evict", "prompt", "prompt"])
        hkv = rng.choice([1, 2, 3, 4, 8])
        c = dict(hkv=hkv, hq=hkv * rng.choice([1, 2, 3, 4, 4, 5, 6, 8, 12, 16]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 layout=rng.choice(["bhsd", "bshd"]))
        if op == "prompt":
            s = _log(rng, 1, 8192)
            c.update(b=rng.choice([1, 1, 1, 2, 3]), s=s, docs=rng.choice([0, rng.randint(1, min(16, s))]), sinks=rng.random() < 0.25)
            c["tail"] = rng.randint(0, s // 4) if c["docs"] and rng.random() < 0.5 else 0
            if c["b"] * c["hq"] * s * s > 32 * 8192 * 8192:
                continue
        elif op == "append" and rng.random() < 0.5:
            c.update(b=1, n=_log(rng, 1, 32768), longest=0)
            c["packed"] = rng.randint(1, min(16, c["n"]))
        else:
            c.update(b=_log(rng, 1, 64), longest=_log(rng, 2, 65536))
            if c["b"] * hkv * c["longest"] > 32 * 8 * 8192:
                continue
            if op == "append":
                c.update(n=min(c["longest"], rng.choice([1, 1, 2, 3, 5])), packed=0)
            elif op == "attend":
                c.update(n=rng.choice([1, 1, 1, 2, 3, 4, 5]), sinks=rng.random() < 0.25, weights=rng.random() < 0.35)
            else:
                c["keep"] = _log(rng, 1, c["longest"])
                c["recent"] = rng.randint(0, c["keep"])
        return _case(op, **c)


def _lengths(case):
    """Tokens in the cache of every sequence: the first one of the full length, the others of some spread, one in eight of them
    without a token (an empty place of the batch)."""
    b, longest, n = case["b"], case["longest"], case.get("n", 1)
    r = np.random.RandomState(longest + 7 * b)
    ls = np.maximum(np.minimum(n, longest), (longest * r.uniform(0.3, 1.0, b)).astype(np.int64))
    ls[r.uniform(size=b) < 0.125] = 0
    ls[0] = longest
    return ls


def _boundaries(total, parts, seed):
    """Where the sequences of a packed call begin and end: unequal lengths, none of them empty."""
    r = np.random.RandomState(seed)
    w = r.uniform(0.3, 1.7, parts)
    cut = np.round(np.cumsum(w) / w.sum() * (total - parts)).astype(np.int64) + np.arange(1, parts + 1)
    return np.concatenate([[0], cut])


def _prompt_cu(case):
    if not case["docs"]:
        return np.array([0, case["s"]])
    docs = min(case["docs"], case["s"] - case["tail"])
    return _boundaries(case["s"] - case["tail"], docs, case["s"] + docs)


def _append_cu(case):
    return _boundaries(case["n"], case["packed"], case["n"])


# ---------------------------------------------------------------------------------------------------------------------
# the cache in plain operations
# ---------------------------------------------------------------------------------------------------------------------

def _quantize(x):
    """(codes -7..7, bf16 scales [..., 4]) of rows x [..., 128].  The scale is the largest magnitude of the group over seven in bf16, 0
    below 2^-80; halves round away from zero, which 64 bits decide (32 could cross the border)."""
    g = x.double().unflatten(-1, (4, 32))
    top = g.abs().amax(-1)
    s = torch.where(top < 2.0 ** -80, torch.zeros_like(top), top / 7).to(torch.float32).to(torch.bfloat16)
    s = torch.where(torch.isfinite(top), s, torch.full_like(s, math.nan))
    d = s.double().unsqueeze(-1)
    q = torch.where(d > 0, torch.sign(g) * torch.floor(g.abs() / d + 0.5), torch.zeros_like(g))
    return q.flatten(-2).to(torch.int8), s


def _pair(nibbles):
    return (nibbles[..., 0::2] | nibbles[..., 1::2] << 4).to(torch.uint8)


def _pack_k(q):
    """Bytes [..., 64] of K codes [..., 128]."""
    n = (q + 8).to(torch.uint8).unflatten(-1, (4, 4, 8)).transpose(-3, -2)   # [chunk t][word i][nibble]
    return _pair(n).flatten(-3)


def _pack_v(q, token):
    """Bytes [..., 64] of V codes [..., 128] of the tokens `token` [...] of a page."""
    n = (q + 8).to(torch.uint8).unflatten(-1, (4, 8, 4)).transpose(-3, -2)   # [chunk c][halfword i][nibble]
    b = _pair(n).flatten(-2)                                                 # [chunk][8 bytes]
    return torch.where((token & 4).bool()[..., None, None], b.roll(4, -2), b).flatten(-2)


def _bf16_bytes(s):
    return s.contiguous().view(torch.uint8)


def _parts(cache):
    """Views of the pool: K codes, K scales, V codes, V scales as bytes, [pages, heads, 128, 64 or 8]."""
    return [cache[..., lo:hi].unflatten(-1, (PAGE, -1)) for lo, hi in (K_CODES, K_SCALES, V_CODES, V_SCALES)]


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _values(cache):
    """fp32 K and V [..., 128 tokens, 128] of records [..., 18432]."""
    kc, ks, vc, vs = (p.contiguous() for p in _parts(cache))
    k = _nibbles(kc).unflatten(-1, (4, 4, 8)).transpose(-3, -2).flatten(-2).float() - 8      # [group][32]
    k = (k * ks.view(torch.bfloat16).float().unsqueeze(-1)).flatten(-2)
    vc = vc.unflatten(-1, (8, 8))
    token = torch.arange(PAGE, device=cache.device)
    vc = torch.where((token & 4).bool()[:, None, None], vc.roll(4, -2), vc).flatten(-2)
    v = _nibbles(vc).unflatten(-1, (8, 4, 4)).transpose(-3, -2).flatten(-2).float() - 8
    v = (v * vs.view(torch.bfloat16).float().unsqueeze(-1)).flatten(-2)
    return k, v


def _append_plain(st):
    """New rows go to the last places of their sequences.  Rows without a place (behind the last sequence, an empty place of the batch)
    write back what the spare page holds."""
    k, v, table, lengths, cache = st["k"], st["v"], st["table"], st["lengths"], st["cache"]
    b, h, n, _ = k.shape
    dev = k.device
    pos = torch.arange(n, device=dev)
    if st["cu"] is None:
        seq = torch.arange(b, device=dev)[:, None].expand(b, n)
        place = lengths.long()[:, None] - n + pos
        valid = place >= 0
    else:
        cu = st["cu"].long()
        seq = (torch.searchsorted(cu, pos, right=True) - 1).clamp(max=table.shape[0] - 1)[None]
        place = lengths.long()[seq] - cu[seq + 1] + pos
        valid = (pos < cu[-1])[None] & (place >= 0)
    place = place.clamp(min=0)
    page = torch.where(valid, table.long()[seq, place // PAGE], torch.full_like(place, cache.shape[0] - 1))[:, None].expand(b, h, n)
    slot = torch.where(valid, place % PAGE, torch.zeros_like(place))[:, None].expand(b, h, n)
    head = torch.arange(h, device=dev)[None, :, None].expand(b, h, n)
    keep = valid[:, None, :, None].expand(b, h, n, 1)
    (qk, sk), (qv, sv) = _quantize(k), _quantize(v)
    for part, new in zip(_parts(cache), (_pack_k(qk), _bf16_bytes(sk), _pack_v(qv, slot), _bf16_bytes(sv))):
        part[page, head, slot] = torch.where(keep, new, part[page, head, slot])
    st["weights"][page, head, slot] = torch.where(keep[..., 0], torch.zeros_like(st["weights"][page, head, slot]), st["weights"][page, head, slot])

    def values(q, s):
        x = (q.float().unflatten(-1, (4, 32)) * s.float().unsqueeze(-1)).flatten(-2)
        return torch.where(keep, x, torch.zeros_like(x)).to(k.dtype)
    return {"k": values(qk, sk), "v": values(qv, sv), "cache": cache, "weights": st["weights"]}


def _attend_plain(st):
    q, cache, table, lengths = st["q"], st["cache"], st["table"], st["lengths"]
    b, hq, n, _ = q.shape
    hkv, w = cache.shape[1], table.shape[1]
    k, v = _values(cache[table.long()])                                        # [b, w, hkv, 128, 128]
    k, v = (x.transpose(1, 2).reshape(b, hkv, w * PAGE, D) for x in (k, v))
    rows = q.float().reshape(b, hkv, hq // hkv * n, D)
    s = rows @ k.transpose(-1, -2) * SCALE
    j = torch.arange(n, device=q.device).repeat(hq // hkv)
    seen = torch.arange(w * PAGE, device=q.device) < (lengths.long()[:, None] - n + 1 + j)[:, None, :, None]   # [b, 1, rows, keys]
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].view(1, hkv, -1, 1).expand(b, hkv, hq // hkv, n).reshape(b, hkv, -1, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == -math.inf, 0)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + torch.exp(sink - top)
    p = p / total.masked_fill(total == 0, 1)
    v = v.masked_fill(~seen.any(2, keepdim=False).unsqueeze(-1), 0)
    out = (p @ v).view(b, hq, n, D).transpose(1, 2).reshape(b, n, hq * D).to(q.dtype)
    if st["weights"] is None:
        return {"out": out}
    new = p.sum(2).view(b, hkv, w, PAGE).transpose(1, 2)
    old = st["weights"][table.long()]
    stored = seen.any(2).view(b, 1, w, PAGE).transpose(1, 2)
    st["weights"][table.long()] = torch.where(stored, new, old)
    return {"out": out, "weights": st["weights"]}


def _evict_plain(st):
    """Keeps the last `recent` tokens and the others of largest weight, in their order, and copies their bytes."""
    cache, weights, table, lengths, to = st["cache"], st["weights"], st["table"], st["lengths"], st["to"]
    keep, recent = st["keep"], st["recent"]
    b, w = table.shape
    h = cache.shape[1]
    dev = cache.device
    n = lengths.long()[:, None, None]
    at = torch.arange(w * PAGE, device=dev)
    score = weights[table.long()].transpose(1, 2).reshape(b, h, w * PAGE)
    score = score.masked_fill(at >= n - recent, math.inf)
    score = score.masked_fill(at >= n, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=w * PAGE)
    left = lengths.long().clamp(max=keep)
    j = torch.arange(keep, device=dev)
    valid = (j < left[:, None, None]).expand(b, h, keep)
    kept = torch.sort(order.masked_fill(~valid, w * PAGE), dim=-1).values
    src = torch.where(valid, kept, torch.zeros_like(kept))
    seq = torch.arange(b, device=dev)[:, None, None].expand(b, h, keep)
    head = torch.arange(h, device=dev)[None, :, None].expand(b, h, keep)
    ps, pd = table.long()[seq, src // PAGE], to.long()[seq, (j // PAGE).expand(b, h, keep)]
    ss, sd = src % PAGE, (j % PAGE).expand(b, h, keep)
    k, ksc, v, vsc = _parts(cache)
    for part in (k, ksc, v, vsc):
        rows = part[ps, head, ss]
        if part is v:
            rows = torch.where(((ss ^ sd) & 4).bool()[..., None, None], rows.unflatten(-1, (8, 8)).roll(4, -2), rows.unflatten(-1, (8, 8))).flatten(-2)
        part[pd, head, sd] = torch.where(valid.unsqueeze(-1), rows, part[pd, head, sd])
    weights[pd, head, sd] = torch.where(valid, weights[ps, head, ss], weights[pd, head, sd])
    return {"lengths": left.to(torch.int32), "kept": torch.where(valid, kept, torch.full_like(kept, -1)).to(torch.int32), "cache": cache,
            "weights": weights}


def _prompt_plain(st):
    q, k, v, cu = st["q"], st["k"], st["v"], st["cu"]
    b, hq, s, _ = q.shape
    hkv = k.shape[1]
    at = torch.arange(s, device=q.device)
    ends = torch.tensor([0, s], device=q.device) if cu is None else cu.long()
    doc = torch.searchsorted(ends, at, right=True)
    real = at < ends[-1]
    seen = (doc[:, None] == doc) & (at <= at[:, None]) & real[:, None]
    x = q.float().view(b, hkv, hq // hkv, s, D) @ k.float().unsqueeze(2).transpose(-1, -2)
    x.mul_(SCALE).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    if st["sinks"] is not None:
        sink = st["sinks"].view(1, hkv, hq // hkv, 1, 1)
        top = torch.maximum(top, sink)
    top = top.masked_fill(top == -math.inf, 0)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = (x @ v.float().unsqueeze(2)) / total.masked_fill(total == 0, 1)
    return {"out": out.view(b, hq, s, D).transpose(1, 2).reshape(b, s, hq * D).to(q.dtype)}


# ---------------------------------------------------------------------------------------------------------------------
# what the tools call
# ---------------------------------------------------------------------------------------------------------------------

def _pool(case, gen, pages):
    """A pool with `pages` pages that hold rows of N(0,1) around a mean per channel, as keys have it."""
    dev = gen.device
    hkv = case["hkv"]
    cache = torch.empty(pages, hkv, RECORD, dtype=torch.uint8, device=dev)
    token = torch.arange(PAGE, device=dev).expand(1, hkv, PAGE)
    for lo in range(0, pages, 256):
        some = cache[lo:lo + 256]
        kv = torch.randn(2, some.shape[0], hkv, PAGE, D, generator=gen, device=dev)
        kv[0] += torch.randn(hkv, 1, D, generator=gen, device=dev)
        g = kv.unflatten(-1, (4, 32))
        sc = (g.abs().amax(-1) / 7).to(torch.bfloat16)
        q = torch.round(g / sc.float().unsqueeze(-1)).clamp_(-7, 7).flatten(-2).to(torch.int8)
        for part, new in zip(_parts(some), (_pack_k(q[0]), _bf16_bytes(sc[0]), _pack_v(q[1], token), _bf16_bytes(sc[1]))):
            part.copy_(new)
    return cache


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = torch.float16 if case["dtype"] == "fp16" else torch.bfloat16
    b, hq, hkv = case["b"], case["hq"], case["hkv"]

    def rows(h, s):
        t = torch.randn(b, h, s, D, generator=gen, device=dev).to(dtype)
        return t.transpose(1, 2).contiguous().transpose(1, 2) if case["layout"] == "bshd" else t

    st = {"op": case["op"], "sinks": None}
    if case.get("sinks"):
        st["sinks"] = torch.randn(hq, generator=gen, device=dev) * 0.7 + 0.5
    if case["op"] == "prompt":
        st.update(q=rows(hq, case["s"]), k=rows(hkv, case["s"]), v=rows(hkv, case["s"]), cu=None)
        if case["docs"]:
            st["cu"] = torch.as_tensor(_prompt_cu(case), dtype=torch.int32, device=dev)
        return st

    if case["op"] == "append" and case["packed"]:
        cu = _append_cu(case)
        lengths = np.diff(cu) + np.random.RandomState(case["n"]).randint(0, 300, case["packed"])   # (behind what the cache holds already)
    else:
        cu, lengths = None, _lengths(case)
    width = max(1, -(-int(lengths.max()) // PAGE))
    seqs = len(lengths)
    own_pages = seqs * width
    new_width = -(-case["keep"] // PAGE) if case["op"] == "evict" else 0
    pages = own_pages + seqs * new_width + 1                      # the last page belongs to no sequence
    perm = torch.randperm(pages - 1, generator=gen, device=dev).to(torch.int32)
    st.update(cache=_pool(case, gen, pages), table=perm[:own_pages].view(seqs, width).contiguous(),
              lengths=torch.as_tensor(lengths, dtype=torch.int32, device=dev))
    # attention weight collected so far: most of it on few tokens
    weights = torch.randn(pages, hkv, PAGE, generator=gen, device=dev).mul_(2).exp_()
    if case["op"] == "append":
        st.update(k=rows(hkv, case["n"]), v=rows(hkv, case["n"]), weights=weights, cu=None)
        if cu is not None:
            st["cu"] = torch.as_tensor(cu, dtype=torch.int32, device=dev)
    elif case["op"] == "attend":
        # (small beside those of one call, so that a comparison sees the latter)
        st.update(q=rows(hq, case["n"]), weights=weights.mul_(1e-6) if case["weights"] else None)
    else:
        st.update(weights=weights, to=perm[own_pages:].view(seqs, new_width).contiguous(), keep=case["keep"], recent=case["recent"])
    return st


def run(state):
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "evict": _evict_plain, "prompt": _prompt_plain}[state["op"]](state)
    import flash_msa_b200 as fm
    with torch.no_grad():
        if state["op"] == "prompt":
            return {"out": fm.flash_msa_prompt_func(state["q"], state["k"], state["v"], state["cu"], SCALE, sinks=state["sinks"])}
        if state["op"] == "append":
            k, v = fm.flash_msa_cache_append(state["cache"], state["k"], state["v"], state["table"], state["lengths"], cu_seqlens=state["cu"],
                                             weights=state["weights"], return_values=True)
            return {"k": k, "v": v, "cache": state["cache"], "weights": state["weights"]}
        if state["op"] == "attend":
            out = fm.flash_msa_cache_func(state["q"], state["cache"], state["table"], state["lengths"], SCALE, sinks=state["sinks"],
                                          weights=state["weights"], accumulate=False)
            return {"out": out} if state["weights"] is None else {"out": out, "weights": state["weights"]}
        lengths, kept = fm.flash_msa_cache_evict(state["cache"], state["weights"], state["table"], state["lengths"], state["to"], state["keep"],
                                                 state["recent"])
        return {"lengths": lengths, "kept": kept, "cache": state["cache"], "weights": state["weights"]}


def work(case):
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "prompt":
        lens = np.diff(_prompt_cu(case))
        pairs = int((lens * (lens + 1) // 2).sum())
        return {"bytes": 2 * D * case["b"] * case["s"] * (2 * hq + 2 * hkv), "flops": 4 * D * case["b"] * hq * pairs}
    if case["op"] == "append":
        rows = case["n"] * hkv if case["packed"] else int((_lengths(case) > 0).sum()) * case["n"] * hkv
        return {"bytes": rows * (8 * D + 144 + 4), "flops": rows * 2 * D * 3}
    lens = _lengths(case)
    if case["op"] == "attend":
        n = case["n"]
        pairs = int(sum(np.maximum(lens - n + 1 + j, 0).sum() for j in range(n)))
        return {"bytes": int(lens.sum()) * hkv * (144 + (4 if case["weights"] else 0)) + 4 * D * case["b"] * n * hq, "flops": 4 * D * hq * pairs}
    left = np.minimum(lens, case["keep"])
    return {"bytes": hkv * (4 * int(lens.sum()) + int(left.sum()) * (2 * 144 + 4 + 4)), "flops": hkv * int(lens.sum())}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence and head by head
# ---------------------------------------------------------------------------------------------------------------------

def _softmax_row_sums(logits, sink):
    """Probabilities of logits [rows, keys] (-inf where hidden) with an optional logit [rows] beside them that takes no value."""
    ref = logits.amax(1)
    if sink is not None:
        ref = torch.maximum(ref, sink)
    ref = torch.nan_to_num(ref, neginf=0.0)
    e = (logits - ref[:, None]).exp()
    z = e.sum(1)
    if sink is not None:
        z = z + (sink - ref).exp()
    return e / torch.where(z > 0, z, torch.ones_like(z))[:, None]


def _read_exact(record):
    """K and V [tokens, 128] in 64 bits of one head's records [pages, 18432], byte by byte from the layout in the docstring."""
    dev = record.device
    tok, ch = torch.arange(PAGE, device=dev)[:, None], torch.arange(D, device=dev)[None]
    group, rest = ch // 32, ch % 32
    k_nib = (rest // 8) * 32 + group * 8 + rest % 8
    v_nib = ((rest // 4) ^ (tok & 4)) * 16 + group * 4 + rest % 4
    found = []
    for codes, scales, nib in ((K_CODES, K_SCALES, k_nib), (V_CODES, V_SCALES, v_nib)):
        byte = record[:, (codes[0] + tok * 64 + nib // 2).reshape(-1)].view(-1, PAGE, D).int()
        q = (byte >> 4 * (nib % 2)) % 16 - 8
        lo = record[:, (scales[0] + tok * 8 + group * 2).reshape(-1)].view(-1, PAGE, D).int()
        hi = record[:, (scales[0] + tok * 8 + group * 2 + 1).reshape(-1)].view(-1, PAGE, D).int()
        found.append((q.double() * ((hi << 24) | (lo << 16)).view(torch.float32).double()).reshape(-1, D))
    return found


def _rounded_exact(x):
    """Rows [..., 128] in 64 bits -> the values that 4 bits hold for them."""
    out = torch.empty_like(x)
    for i in range(4):
        g = x[..., 32 * i:32 * i + 32]
        s = (g.abs().max(-1, keepdim=True).values / 7.0).float().bfloat16().double()
        t = g / s
        out[..., 32 * i:32 * i + 32] = torch.where(t >= 0, (t + 0.5).floor(), (t - 0.5).ceil()) * s
    return out


def exact(case, seed):
    st = prepare(case, seed)
    b, hq, hkv = case["b"], case["hq"], case["hkv"]
    g = hq // hkv
    if case["op"] == "prompt":
        cu = _prompt_cu(case).tolist()
        out = torch.zeros(b, case["s"], hq, D, dtype=torch.float64, device="cuda")
        for i in range(b):
            for h in range(hq):
                for lo, hi in zip(cu[:-1], cu[1:]):
                    logits = st["q"][i, h, lo:hi].double() @ st["k"][i, h // g, lo:hi].double().T * SCALE
                    logits = logits.masked_fill(torch.ones(hi - lo, hi - lo, dtype=torch.bool, device="cuda").triu(1), -math.inf)
                    sink = None if st["sinks"] is None else st["sinks"][h].double().expand(hi - lo)
                    out[i, lo:hi, h] = _softmax_row_sums(logits, sink) @ st["v"][i, h // g, lo:hi].double()
        return {"out": out.flatten(2)}
    if case["op"] == "append":
        rows = {n: _rounded_exact(st[n].double()) for n in ("k", "v")}
        if st["cu"] is None:
            for t in rows.values():
                t[torch.as_tensor(_lengths(case) == 0)] = 0
        return dict(rows, cache=None, weights=None)
    lens = _lengths(case).tolist()
    if case["op"] == "evict":
        return None
    n = case["n"]
    out = torch.zeros(b, n, hq, D, dtype=torch.float64, device="cuda")
    weights = None if st["weights"] is None else st["weights"].double()
    for i, length in enumerate(lens):
        if not length:
            continue
        used = st["table"][i, :-(-length // PAGE)].long()
        for h in range(hkv):
            k, v = (t[:length] for t in _read_exact(st["cache"][used, h]))
            q = st["q"][i, h * g:(h + 1) * g].double().reshape(g * n, D)
            limit = (length - n + 1 + torch.arange(n, device="cuda")).repeat(g)
            logits = (q @ k.T * SCALE).masked_fill(torch.arange(length, device="cuda")[None] >= limit[:, None], -math.inf)
            sink = None if st["sinks"] is None else st["sinks"][h * g:(h + 1) * g].double().repeat_interleave(n)
            p = _softmax_row_sums(logits, sink)
            out[i, :, h * g:(h + 1) * g] = (p @ v).view(g, n, D).transpose(0, 1)
            if weights is not None:
                new = torch.zeros(len(used) * PAGE, dtype=torch.float64, device="cuda")
                new[:length] = p.sum(0)
                keep = torch.arange(len(used) * PAGE, device="cuda") < length
                weights[used, h] = torch.where(keep.view(-1, PAGE), new.view(-1, PAGE), weights[used, h])
    return {"out": out.flatten(2)} if weights is None else {"out": out.flatten(2), "weights": weights}
