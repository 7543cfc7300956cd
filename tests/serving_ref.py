"""The serving operators restated in 64 bits, byte by byte and sequence by sequence, for the tests."""
import math

import torch

D, PAGE, RECORD = 128, 128, 18432
SCALE = D ** -0.5


def _maps():
    """Byte and nibble of every (token, channel) of a record for K and V, and byte of the scale."""
    tok = torch.arange(PAGE).view(-1, 1).expand(PAGE, D)
    ch = torch.arange(D).view(1, -1).expand(PAGE, D)
    i, r = ch // 32, ch % 32
    k = tok * 64 + (r // 8) * 16 + i * 4 + (r % 8) // 2
    v = 9216 + tok * 64 + ((r // 4) ^ (tok & 4)) * 8 + i * 2 + (r % 4) // 2
    return {"k": (k, r % 2, 8192 + tok * 8 + i * 2), "v": (v, r % 2, 17408 + tok * 8 + i * 2)}


MAPS = _maps()


def unpack(records, which):
    """fp64 [..., 128, 128] of records [..., 18432]."""
    byte, odd, scale = (m.to(records.device) for m in MAPS[which])
    q = (records[..., byte].int() >> (4 * odd)) % 16 - 8
    bits = records[..., scale].int() | records[..., scale + 1].int() << 8
    return q.double() * (bits << 16).view(torch.float32).double()


def quantize(x):
    """(codes, fp64 scales [..., 4]) of rows [..., 128]."""
    g = x.double().unflatten(-1, (4, 32))
    top = g.abs().amax(-1)
    s = (top / 7).float().bfloat16().double()
    s[top < 2.0 ** -80] = 0
    s[~torch.isfinite(top)] = math.nan
    t = g / s.unsqueeze(-1)
    q = torch.sign(t) * torch.floor(t.abs() + 0.5)
    return torch.where(s.unsqueeze(-1) > 0, q, torch.zeros_like(q)).flatten(-2), s


def pack_into(record, slot, which, x):
    """Writes the row x [128] at `slot` of one record [18432] (CPU)."""
    q, s = quantize(x)
    byte, odd, scale = (m[slot] for m in MAPS[which])
    for c in range(D):
        b, sh = int(byte[c]), 4 * int(odd[c])
        record[b] = (int(record[b]) & (0xF0 if sh == 0 else 0x0F)) | (int(q[c]) + 8) << sh
    for i in range(4):
        w = int(s[i].to(torch.bfloat16).view(torch.int16)) & 0xFFFF if torch.isfinite(s[i]) else 0x7FFF   # (CUDA's NaN)
        record[int(scale[32 * i])], record[int(scale[32 * i]) + 1] = w & 255, w >> 8


def rows_of(cache, table, length, head, which):
    """fp64 [length, 128]: what sequence row `table` (1-D) holds."""
    pages = table[:-(-length // PAGE)].long()
    return unpack(cache[pages, head], which).reshape(-1, D)[:length]


def softmax(logits, sink=None):
    top = logits.amax(-1, keepdim=True)
    if sink is not None:
        top = torch.maximum(top, sink.view(-1, 1))
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(logits - top)
    z = e.sum(-1, keepdim=True)
    if sink is not None:
        z = z + torch.exp(sink.view(-1, 1) - top)
    return e / torch.where(z == 0, torch.ones_like(z), z)


def attend(q, cache, table, lengths, scale, sinks=None):
    """(out [B,n,Hq,128], tolerance of out, [(seq, head) -> weights of its tokens], the same's tolerance), fp64.

    What the tolerances count: the rounding of the result (half a step); every probability times V's scale is rounded to fp16 once
    (2^-11 relative); a logit is a sum of 128 products in fp32 of whole numbers up to 15 with fp16 queries, held to 2^-19 of the sum of
    its terms' magnitudes, (15 steps at most of 2^-24 each, and as much again for the scales, the row factor and the reference's
    subtraction); the exponential and the reciprocal take 2^-20 together; and what fp16 loses below its normal numbers is at most 2^-30 of the
    largest value per token."""
    b, hq, n, _ = q.shape
    hkv = cache.shape[1]
    g = hq // hkv
    out = torch.zeros(b, n, hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    weights = {}
    half = torch.finfo(q.dtype).eps / 2
    for i, length in enumerate(lengths):
        for h in range(hkv):
            if length == 0:
                continue
            k, v = rows_of(cache, table[i], length, h, "k"), rows_of(cache, table[i], length, h, "v")
            x = q[i, h * g:(h + 1) * g].double().reshape(g * n, D)
            seen = torch.arange(length, device=q.device) < (length - n + 1 + torch.arange(n, device=q.device).repeat(g)).view(-1, 1)
            logits = (x @ k.T * scale).masked_fill(~seen, -math.inf)
            sink = None if sinks is None else sinks[h * g:(h + 1) * g].double().repeat_interleave(n)
            p = softmax(logits, sink)
            y = p @ v
            spread = x.abs() @ (k.abs() + 8 * k.abs().amax(0).max() / 7).T * scale
            err = (2.0 ** -19 * spread.masked_fill(~seen, 0).amax(-1, keepdim=True) + 2.0 ** -20).clamp(max=1)
            e = y.abs() * half + (p @ v.abs()) * (2.0 ** -11 + 2 * err) + length * 2.0 ** -30 * v.abs().amax() * seen.any(-1, keepdim=True)
            out[i, :, h * g:(h + 1) * g] = y.view(g, n, D).transpose(0, 1)
            tol[i, :, h * g:(h + 1) * g] = e.view(g, n, D).transpose(0, 1)
            weights[i, h] = (p.sum(0), (p * 2 * err).sum(0) + 1e-30)
    return out, tol + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps, weights


def evict(weights, table, lengths, keep, recent):
    """[(seq, head) -> kept places] in plain Python."""
    kept = {}
    w = weights.float().cpu()
    for i, length in enumerate(lengths):
        for h in range(weights.shape[1]):
            if length <= keep:
                kept[i, h] = list(range(length))
                continue
            x = [float(w[int(table[i, t // PAGE]), h, t % PAGE]) for t in range(length - recent)]
            order = sorted(range(len(x)), key=lambda t: (-(math.inf if x[t] != x[t] else x[t]), x[t] == x[t], t))
            kept[i, h] = sorted(order[:keep - recent]) + list(range(length - recent, length))
    return kept


def prompt(q, k, v, cu, scale, sinks=None):
    """(out [B,S,Hq,128], tolerance), fp64; `cu`: a list of boundaries per batch element.

    What the tolerance counts: the rounding of the result and that of every probability (half a step of the type each), a logit's sum of 128
    products in fp32 and the scaling (2^-20 of the sum of the terms' magnitudes), the exponential and the division (2^-20), and in fp16
    what is lost below its normal numbers: at most 2^-25 of a probability that is lifted by 2^7, relative to the row's maximum."""
    b, hq, s, _ = q.shape
    g = hq // k.shape[1]
    out = torch.zeros(b, s, hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    half = torch.finfo(q.dtype).eps / 2
    for i in range(b):
        for lo, hi in zip(cu[i][:-1], cu[i][1:]):
            if lo == hi:
                continue
            hidden = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=q.device).triu(1)
            for h in range(hq):
                x, y, z = (t[i, hh, lo:hi].double() for t, hh in ((q, h), (k, h // g), (v, h // g)))
                p = softmax((x @ y.T * scale).masked_fill(hidden, -math.inf), None if sinks is None else sinks[h].double().expand(hi - lo))
                err = (2.0 ** -20 * (x.abs() @ y.abs().T * scale).masked_fill(hidden, 0).amax(-1, keepdim=True) + 2.0 ** -20).clamp(max=1)
                out[i, lo:hi, h] = p @ z
                tol[i, lo:hi, h] = out[i, lo:hi, h].abs() * half + (p @ z.abs()) * (half + 2 * err) + (hi - lo) * 2.0 ** -32 * z.abs().amax()
    return out, tol + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
