"""The cache held in 4 bits on the GPU, against 64-bit restatements (tests/serving_ref.py, which derives the tolerances)."""
import math

import pytest
import torch

from tests import serving_ref as R

pytestmark = pytest.mark.gpu
SCALE = R.SCALE


@pytest.fixture(scope="module")
def fm():
    import flash_msa_b200
    from flash_msa_b200 import api
    api.DEBUG_CHECK_STATUS = True
    yield flash_msa_b200
    api.DEBUG_CHECK_STATUS = False


def layout(t, kind):
    b, h, s, d = t.shape
    if kind == "bshd":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "odd":            # an address off the 16-byte grid: copied once
        return torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)[1:1 + t.numel()].view(t.shape).copy_(t)
    if kind == "wide":           # rows 136 apart
        return torch.zeros(b, h, s, d + 8, dtype=t.dtype, device=t.device)[..., :d].copy_(t)
    return t


def pool(fm, lengths, hkv, seed, spare=1, fill=0xFF, v_size=1.0, k_size=1.0):
    """A pool that holds sequences of these lengths in shuffled pages; every byte that was not appended is `fill` (0xFF: scales are NaN)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, -(-max(lengths) // 128))
    b = len(lengths)
    pages = b * width + spare
    cache = fm.flash_msa_cache_empty(pages, hkv)
    cache.fill_(fill)
    table = torch.randperm(b * width, generator=g, device="cuda").to(torch.int32).view(b, width)
    ls = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    n = sum(lengths)
    if n:
        k, v = (torch.randn(1, hkv, n, 128, generator=g, device="cuda") for _ in range(2))
        k += torch.randn(1, hkv, 1, 128, generator=g, device="cuda")
        cu = [0]
        for x in lengths:
            cu.append(cu[-1] + x)
        fm.flash_msa_cache_append(cache, (k * k_size).to(torch.bfloat16), (v * v_size).to(torch.bfloat16), table, ls, cu_seqlens=cu)
    return cache, table, ls, g


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------

def append_reference(cache, k, v, table, lengths, owner):
    """The pool after the call, and the values it stands for: row (b, j) goes to owner(b, j) = (sequence, place) or None."""
    want, kc, vc = cache.cpu().clone(), k.cpu(), v.cpu()
    vals = [torch.zeros(k.shape, dtype=torch.float64) for _ in range(2)]
    b, h, n, _ = k.shape
    for i in range(b):
        for j in range(n):
            to = owner(i, j)
            if to is None:
                continue
            page = int(table[to[0], to[1] // 128])
            for hh in range(h):
                for which, x, val in (("k", kc, vals[0]), ("v", vc, vals[1])):
                    R.pack_into(want[page, hh], to[1] % 128, which, x[i, hh, j])
                    q, s = R.quantize(x[i, hh, j])
                    val[i, hh, j] = (q.unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten()
    return want, vals


def rows_with_edges(shape, dtype, seed):
    """N(0,1) rows; and in the first ones halves between codes, zeros, extremes of the type, values that are not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    flat = x.view(-1, 128)
    flat[0] = torch.arange(128).remainder(15).sub(7).float() * 0.5 + 0.25 * (torch.arange(128) % 2)   # halves and quarters of a scale of 1/2
    flat[0, ::32] = 3.5
    if flat.shape[0] > 1:
        flat[1, :32] = 0
        flat[1, 32:64] = torch.finfo(dtype).smallest_normal * torch.arange(32)
        flat[1, 64:96] = torch.finfo(dtype).max * (torch.arange(32) / 31 - 0.4)
        flat[1, 96] = math.inf
    if flat.shape[0] > 2:
        flat[2, 3], flat[2, 40], flat[2, 70] = math.nan, -math.inf, -0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["bhsd", "bshd", "odd", "wide"])
@pytest.mark.parametrize("b,h,n,lengths", [(1, 1, 1, [1]), (3, 2, 1, [128, 0, 257]), (2, 3, 5, [130, 5]), (3, 1, 7, [3, 300, 0]), (1, 5, 2, [129])])
def test_append_steps(fm, b, h, n, lengths, kind, dtype):
    g = torch.Generator().manual_seed(n)
    cache = torch.randint(0, 256, (3 * b + 1, h, R.RECORD), generator=g, dtype=torch.uint8).cuda()
    weights = torch.rand(3 * b + 1, h, 128, generator=g).cuda()
    table = torch.randperm(3 * b, generator=g).to(torch.int32).view(b, 3)
    k, v = (rows_with_edges((b, h, n, 128), dtype, seed) for seed in (1, 2))
    want, vals = append_reference(cache, k, v, table, lengths, lambda i, j: (i, lengths[i] - n + j) if lengths[i] - n + j >= 0 else None)
    want_w = weights.clone()
    for i in range(b):
        for t in range(max(0, lengths[i] - n), lengths[i]):
            want_w[table[i, t // 128], :, t % 128] = 0
    got = fm.flash_msa_cache_append(cache, layout(k.cuda(), kind), layout(v.cuda(), kind), table.cuda(),
                                    torch.tensor(lengths, dtype=torch.int32, device="cuda"), weights=weights, return_values=True)
    assert torch.equal(cache.cpu(), want) and torch.equal(weights, want_w)
    for x, val in zip(got, vals):
        y = val.to(torch.float32).to(dtype)   # (exact in fp32: eleven bits)
        assert x.dtype == dtype and x.shape == k.shape
        assert torch.equal(torch.nan_to_num(x.cpu(), nan=-99.0), torch.nan_to_num(y, nan=-99.0))


@pytest.mark.parametrize("host", ["list", "cpu", "cuda", "cuda64"])
@pytest.mark.parametrize("cu,before,n", [([0, 1], [0], 1), ([0, 100, 100, 131], [200, 77, 126], 140), ([0, 0, 3, 3], [5, 0, 0], 9)])
def test_append_packed(fm, cu, before, n, host):
    lengths = [x + cu[i + 1] - cu[i] for i, x in enumerate(before)]
    b = len(lengths)
    table = torch.randperm(3 * b).to(torch.int32).view(b, 3)
    cache = torch.full((3 * b, 2, R.RECORD), 0x5A, dtype=torch.uint8, device="cuda")
    k, v = (rows_with_edges((1, 2, n, 128), torch.bfloat16, seed) for seed in (3, 4))

    def owner(i, j):
        for s in range(b):
            if cu[s] <= j < cu[s + 1]:
                return s, lengths[s] - (cu[s + 1] - j)
        return None
    want, vals = append_reference(cache, k, v, table, lengths, owner)
    given = {"list": cu, "cpu": torch.tensor(cu), "cuda": torch.tensor(cu, dtype=torch.int32).cuda(), "cuda64": torch.tensor(cu).cuda()}[host]
    got = fm.flash_msa_cache_append(cache, k.cuda(), v.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), cu_seqlens=given,
                                    return_values=True)
    assert torch.equal(cache.cpu(), want)
    for x, val in zip(got, vals):
        assert torch.equal(torch.nan_to_num(x.cpu(), nan=-99.0), torch.nan_to_num(val.float().to(x.dtype), nan=-99.0))


def test_append_of_many_random_rows_is_exact(fm):
    """Every code and scale, over magnitudes from subnormal to the type's largest: the quotient is rounded as 64 bits round it."""
    for dtype, top in ((torch.bfloat16, 100.0), (torch.float16, 15.0)):
        g = torch.Generator(device="cuda").manual_seed(9)
        n = 20000
        size = torch.exp2(torch.rand(1, 1, n, 4, 1, generator=g, device="cuda") * (top + 20) - 20)
        x = (torch.randn(1, 1, n, 4, 32, generator=g, device="cuda") * size).flatten(-2).clamp(-6e4 if dtype == torch.float16 else -1e38,
                                                                                               6e4 if dtype == torch.float16 else 1e38).to(dtype)
        grid = torch.randint(-14, 15, x.shape, generator=g, device="cuda").float() * 0.5     # many exact halves
        y = torch.where(torch.rand(1, 1, n, 1, generator=g, device="cuda") < 0.5, (grid * 2.0 ** -3).to(dtype), x)
        pages = -(-n // 128)
        cache = fm.flash_msa_cache_empty(pages, 1)
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        fm.flash_msa_cache_append(cache, x, y, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
        for which, z in (("k", x), ("v", y)):
            q, s = R.quantize(z[0, 0])
            want = (q.unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten(-2)
            assert torch.equal(R.rows_of(cache, table[0], n, 0, which), want)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------

def check_attend(fm, cache, table, ls, lengths, q, sinks=None, weights=None, accumulate=True):
    before = None if weights is None else weights.clone()
    out = fm.flash_msa_cache_func(q, cache, table, ls, SCALE, sinks=sinks, weights=weights, accumulate=accumulate)
    b, hq, n, _ = q.shape
    want, tol, new = R.attend(q, cache, table, lengths, SCALE, sinks)
    assert out.shape == (b, n, hq * 128) and out.dtype == q.dtype
    err = (out.view(b, n, hq, 128).double() - want).abs()
    assert (err <= tol).all(), ((err - tol).max().item(), err.max().item())
    if weights is not None:
        exp = before.double() if accumulate else before.double().clone()
        slack = exp.abs() * 2.0 ** -23
        for (i, h), (w, e) in new.items():
            at = torch.arange(len(w), device="cuda")
            pages = table[i].long()[at // 128]
            if accumulate:
                exp[pages, h, at % 128] += w
            else:
                exp[pages, h, at % 128] = w
            slack[pages, h, at % 128] += e + w * 2.0 ** -20
        assert ((weights.double() - exp).abs() <= slack).all(), (weights.double() - exp).abs().max().item()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,n,lengths", [
    (1, 1, 1, [1]), (2, 2, 1, [16]), (8, 1, 1, [127, 128, 129]), (4, 2, 1, [0, 5, 0, 1000]), (16, 2, 1, [1000]), (9, 1, 1, [300, 40]),
    (16, 1, 1, [17, 500]), (17, 1, 1, [260]), (6, 3, 2, [2, 130, 1, 0]), (12, 1, 4, [3, 257, 900]), (5, 1, 5, [4, 128, 131]), (40, 2, 3, [333]),
    (8, 8, 1, [700] * 30), (4, 1, 1, [6001]), (1, 1, 1, [40000]), (12, 1, 1, [1500, 0, 1537, 64] * 30), (32, 2, 1, [1300] * 60), (4, 1, 3, [9000])])
def test_attention(fm, hq, hkv, n, lengths, dtype):
    cache, table, ls, g = pool(fm, lengths, hkv, seed=hq + n)
    q = torch.randn(len(lengths), hq, n, 128, generator=g, device="cuda").to(dtype)
    check_attend(fm, cache, table, ls, lengths, q)


@pytest.mark.parametrize("kind", ["bshd", "odd", "wide"])
@pytest.mark.parametrize("sinks", [None, 0.0, 9.0, -50.0])
def test_attention_layouts_and_sinks(fm, kind, sinks):
    lengths = [200, 0, 1]
    cache, table, ls, g = pool(fm, lengths, 2, seed=5)
    q = torch.randn(3, 6, 2, 128, generator=g, device="cuda").to(torch.bfloat16)
    s = None if sinks is None else torch.randn(6, generator=g, device="cuda") + sinks
    check_attend(fm, cache, table, ls, lengths, layout(q, kind), s)
    if s is not None:   # logits of another type, and a head that every row of a batch shares by stride 0
        check_attend(fm, cache, table, ls, lengths, q[:1].expand(3, 6, 2, 128), s.to(torch.bfloat16))


@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-4, 1, 1), (30, 1, 1), (1, 1, 1e-18), (1, 1, 1e18), (1e4, 1e-6, 3e4), (1, 30, 1e-7)])
def test_attention_of_other_magnitudes(fm, q_size, k_size, v_size):
    lengths = [900, 77]
    cache, table, ls, g = pool(fm, lengths, 1, seed=6, k_size=k_size, v_size=v_size)
    q = (torch.randn(2, 4, 1, 128, generator=g, device="cuda") * q_size).to(torch.bfloat16)
    check_attend(fm, cache, table, ls, lengths, q)


def test_attention_over_values_of_mixed_size(fm):
    """Scales of V that differ by 2^60 from token to token, rising and falling: the reference follows them."""
    g = torch.Generator(device="cuda").manual_seed(8)
    n = 700
    k, v = (torch.randn(1, 1, n, 128, generator=g, device="cuda") for _ in range(2))
    for size in (torch.linspace(-30, 30, n), torch.linspace(30, -30, n), torch.rand(n) * 60 - 30):
        cache = fm.flash_msa_cache_empty(6, 1)
        table = torch.arange(6, dtype=torch.int32, device="cuda")[None]
        ls = torch.tensor([n], dtype=torch.int32, device="cuda")
        fm.flash_msa_cache_append(cache, k.to(torch.bfloat16), (v * torch.exp2(size).cuda().view(1, 1, n, 1)).to(torch.bfloat16), table, ls)
        q = torch.randn(1, 4, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
        check_attend(fm, cache, table, ls, [n], q)
    v[:, :, ::2] = 0    # tokens that hold zeros, and all of them
    for what in (v, torch.zeros_like(v)):
        fm.flash_msa_cache_append(cache, k.to(torch.bfloat16), what.to(torch.bfloat16), table, ls)
        check_attend(fm, cache, table, ls, [n], q)


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("hq,hkv,n,lengths,sinks", [(4, 2, 1, [1, 0, 300], False), (8, 1, 2, [129, 1], True), (20, 2, 4, [1000, 2], True),
                                                    (3, 3, 1, [5000], False), (48, 1, 1, [700], False)])
def test_attention_weights(fm, hq, hkv, n, lengths, sinks, accumulate):
    cache, table, ls, g = pool(fm, lengths, hkv, seed=hq)
    q = torch.randn(len(lengths), hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda")
    s = torch.randn(hq, generator=g, device="cuda") if sinks else None
    out = check_attend(fm, cache, table, ls, lengths, q, s, w, accumulate)
    again = w.clone()
    assert torch.equal(out, check_attend(fm, cache, table, ls, lengths, q, s, again, accumulate))
    if not accumulate:
        assert torch.equal(again, w)
    check_attend(fm, cache, table, ls, lengths, q, s)     # (a call without weights may sum in another order)


@pytest.mark.parametrize("hq,hkv,n,b,width", [(8, 2, 1, 1, 1), (8, 2, 1, 1, 9), (4, 4, 1, 4, 40), (12, 1, 2, 2, 64), (16, 8, 1, 9, 5), (8, 1, 1, 74, 3), (8, 1, 1, 75, 3),
                                              (4, 4, 1, 40, 70), (24, 1, 1, 1, 300), (2, 1, 1, 700, 2), (12, 1, 1, 32, 40), (32, 2, 1, 37, 17),
                                              (32, 2, 1, 9, 70)])
def test_attention_at_every_number_of_launches(fm, hq, hkv, n, b, width):
    """Few pairs of sequence and KV head go to clusters of 8, 4 or 2 blocks, the others to ranges that cut them: lengths up to what the table
    holds, empty ones, and ones of which most blocks have nothing; and more sequences than a block has threads."""
    from flash_msa_b200 import _lib
    r = torch.Generator().manual_seed(b + width)
    lengths = torch.randint(0, 128 * width + 1, (b,), generator=r).tolist()
    lengths[0] = 128 * width
    if b > 2:
        lengths[1], lengths[2] = 0, 1
    cache, table, ls, g = pool(fm, lengths, hkv, seed=b)
    q = torch.randn(b, hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    check_attend(fm, cache, table, ls, lengths, q, torch.randn(hq, device="cuda"))
    launches = _lib.load().fmsa_cache_attend_launches(b, hq, hkv, n, width, 0)
    assert launches == (1 if (b, width) in ((1, 1), (1, 9), (4, 40), (9, 5), (74, 3), (32, 40), (37, 17), (9, 70)) else 2)


def test_attention_repeats_and_follows_streams(fm):
    lengths = [3000, 10, 513]
    cache, table, ls, g = pool(fm, lengths, 2, seed=3)
    q = torch.randn(3, 8, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    want = fm.flash_msa_cache_func(q, cache, table, ls, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fm.flash_msa_cache_func(q, cache, table, ls, SCALE)
    side.synchronize()
    assert torch.equal(got, want)


def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(fm):
    lengths = [260]
    cache, table, ls, g = pool(fm, lengths, 1, seed=4)
    q = torch.randn(1, 2, 3, 128, generator=g, device="cuda").to(torch.bfloat16)
    want = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(3, 2, 128)
    k, v = (torch.randn(1, 1, 1, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    v[..., 40] = math.inf
    fm.flash_msa_cache_append(cache, k, v, table, ls)              # over the last token, which only the last query sees
    got = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(3, 2, 128)
    assert torch.equal(got[:2], want[:2])
    assert got[2, :, 32:64].isnan().all() and torch.isfinite(got[2, :, :32]).all() and torch.isfinite(got[2, :, 64:]).all()
    k[..., 3] = math.nan
    fm.flash_msa_cache_append(cache, k, v, table, ls)
    got = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(3, 2, 128)
    assert torch.equal(got[:2], want[:2]) and got[2].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("hq,hkv,n,lengths", [
    (17, 1, 1, [1]), (32, 1, 1, [128, 0, 129]), (33, 1, 1, [5000]), (24, 2, 3, [700, 2, 64]), (48, 1, 1, [16] * 20), (64, 1, 1, [300, 40]),
    (13, 1, 5, [4, 128, 1000]), (16, 1, 9, [600, 3]), (3, 1, 43, [40, 500]), (2, 1, 150, [149, 160, 1000]), (20, 1, 1, [30, 0, 200] * 250),
    (40, 2, 1, [20000, 1]), (96, 4, 2, [900, 1300, 5])])
def test_attention_of_many_rows(fm, hq, hkv, n, lengths, sinks, dtype):
    """17 query rows to a KV head and more: blocks of 32, 48 and 64, several blocks, pieces of one page, whole and cut pairs."""
    cache, table, ls, g = pool(fm, lengths, hkv, seed=hq + n)
    q = torch.randn(len(lengths), hq, n, 128, generator=g, device="cuda").to(dtype)
    s = torch.randn(hq, generator=g, device="cuda") if sinks else None
    out = check_attend(fm, cache, table, ls, lengths, q, s)
    w = torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda")
    for accumulate in (True, False):
        assert torch.equal(out, check_attend(fm, cache, table, ls, lengths, q, s, w, accumulate))


@pytest.mark.parametrize("q_size,k_size,v_size", [(1e-4, 1, 1), (30, 1, 1), (1, 1, 1e-18), (1, 1, 1e18), (1e4, 1e-6, 3e4), (1, 30, 1e-7)])
def test_attention_of_many_rows_of_other_magnitudes(fm, q_size, k_size, v_size):
    lengths = [900, 77]
    cache, table, ls, g = pool(fm, lengths, 1, seed=6, k_size=k_size, v_size=v_size)
    q = (torch.randn(2, 24, 1, 128, generator=g, device="cuda") * q_size * torch.logspace(-3, 3, 24, device="cuda").view(1, 24, 1, 1)).to(torch.bfloat16)
    check_attend(fm, cache, table, ls, lengths, q)


def test_attention_of_many_rows_over_values_of_mixed_size(fm):
    """Scales of V that differ by 2^60 from token to token, and by 2^16 within a token; tokens that hold zeros, and all of them."""
    g = torch.Generator(device="cuda").manual_seed(8)
    n = 700
    k, v = (torch.randn(1, 1, n, 128, generator=g, device="cuda") for _ in range(2))
    q = torch.randn(1, 24, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    ls = torch.tensor([n], dtype=torch.int32, device="cuda")
    cache = fm.flash_msa_cache_empty(6, 1)
    groups = torch.exp2(torch.tensor([0.0, -16.0, -5.0, -11.0], device="cuda")).repeat_interleave(32)
    zeros = v.clone()
    zeros[:, :, ::2] = 0
    for what in [v * torch.exp2(size).cuda().view(1, 1, n, 1) for size in (torch.linspace(-30, 30, n), torch.linspace(30, -30, n), torch.rand(n) * 60 - 30)] + [
            v * groups, zeros, torch.zeros_like(v)]:
        fm.flash_msa_cache_append(cache, k.to(torch.bfloat16), what.to(torch.bfloat16), table, ls)
        check_attend(fm, cache, table, ls, [n], q)
    # a group of channels far below the token's largest keeps its accuracy: against the same values with that group alone
    fm.flash_msa_cache_append(cache, k.to(torch.bfloat16), (v * groups).to(torch.bfloat16), table, ls)
    got = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(24, 128)[:, 32:64].float()
    fm.flash_msa_cache_append(cache, k.to(torch.bfloat16), v.to(torch.bfloat16), table, ls)
    want = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(24, 128)[:, 32:64].float() * 2.0 ** -16
    # (both are sums of the same products, with probabilities rounded to fp16 at another place: 2^-11 of the sum of magnitudes, and bf16's step)
    assert (got - want).abs().max() <= 2.0 ** -16 * (2.0 ** -10 * v[..., 32:64].abs().amax() + 2.0 ** -8 * want.abs().max() * 2.0 ** 16)


@pytest.mark.parametrize("hq,n,length,at", [(24, 3, 260, 259), (24, 3, 257, 255), (2, 150, 300, 200), (2, 150, 400, 260), (40, 2, 1, 0)])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them_of_many(fm, hq, n, length, at):
    cache, table, ls, g = pool(fm, [length], 1, seed=4)
    q = torch.randn(1, hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    want = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(n, hq, 128)
    k, v = (torch.randn(1, 1, 1, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    v[..., 40] = math.inf
    fm.flash_msa_cache_append(cache, k, v, table, torch.tensor([at + 1], dtype=torch.int32, device="cuda"))
    first = max(0, at - (length - n))                     # the first query row that sees the token
    got = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(n, hq, 128)
    assert torch.equal(got[:first], want[:first])
    assert got[first:, :, 32:64].isnan().all() and torch.isfinite(got[first:, :, :32]).all() and torch.isfinite(got[first:, :, 64:]).all()
    k[..., 3] = math.nan
    fm.flash_msa_cache_append(cache, k, v, table, torch.tensor([at + 1], dtype=torch.int32, device="cuda"))
    got = fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(n, hq, 128)
    assert torch.equal(got[:first], want[:first]) and got[first:].isnan().all()


def test_attention_of_many_rows_captured(fm):
    """A captured call follows what its tensors hold at each replay; two graphs of the same shapes do not share anything."""
    lengths = [700, 0, 130]
    cache, table, ls, g = pool(fm, lengths, 2, seed=11)
    qs = [torch.randn(3, 40, 1, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    want = [fm.flash_msa_cache_func(q, cache, table, ls, SCALE) for q in qs]
    ws = [torch.zeros(cache.shape[0], 2, 128, device="cuda") for _ in range(2)]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    from flash_msa_b200 import api
    fm.flash_msa_cache_func(qs[0], cache, table, ls, SCALE, weights=ws[0].clone())
    api.DEBUG_CHECK_STATUS = False
    try:
        fm.flash_msa_cache_func(qs[0], cache, table, ls, SCALE, weights=ws[0].clone())
        for graph, q, w in zip(graphs, qs, ws):
            with torch.cuda.graph(graph):
                outs.append(fm.flash_msa_cache_func(q, cache, table, ls, SCALE, weights=w))
    finally:
        api.DEBUG_CHECK_STATUS = True
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
    torch.cuda.synchronize()
    for q, w, out, exp in zip(qs, ws, outs, want):
        assert torch.equal(out, exp)
        one = torch.zeros_like(w)
        fm.flash_msa_cache_func(q, cache, table, ls, SCALE, weights=one, accumulate=False)
        assert torch.equal(w, one + one + one)
    ls.copy_(torch.tensor([1, 0, 129], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    exp = fm.flash_msa_cache_func(qs[0], cache, table, ls, SCALE)
    assert torch.equal(outs[0], exp)
    fm.check_pending_status()


def test_records_beyond_four_gigabytes(fm):
    lengths = [300]
    small, t_small, ls, g = pool(fm, lengths, 2, seed=11)
    pages = 2 ** 32 // (2 * R.RECORD) + 5
    cache = torch.empty(pages, 2, R.RECORD, dtype=torch.uint8, device="cuda")
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device="cuda")
    cache[table[0].long()] = small[t_small[0].long()]
    q = torch.randn(1, 4, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    w, ws = torch.zeros(pages, 2, 128, device="cuda"), torch.zeros(small.shape[0], 2, 128, device="cuda")
    a = fm.flash_msa_cache_func(q, cache, table, ls, SCALE, weights=w)
    assert torch.equal(a, fm.flash_msa_cache_func(q, small, t_small, ls, SCALE, weights=ws))
    assert torch.equal(w[table[0].long()], ws[t_small[0].long()])
    to = torch.tensor([[pages - 2]], dtype=torch.int32, device="cuda")
    _, kept = fm.flash_msa_cache_evict(cache, w, table, ls, to, 100, 20)
    for h in range(2):
        for which in "kv":
            assert torch.equal(R.rows_of(cache, to[0], 100, h, which), R.rows_of(cache, table[0], 300, h, which)[kept[0, h].long()])


def test_pages_that_do_not_exist(fm):
    """They are not touched, and the call says so."""
    cache, table, ls, g = pool(fm, [300, 300], 1, seed=12)
    q = torch.randn(2, 2, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    before = cache.clone()
    w = torch.zeros(cache.shape[0], 1, 128, device="cuda")
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 1] = bad
        for call in (lambda: fm.flash_msa_cache_func(q, cache, t, ls, SCALE), lambda: fm.flash_msa_cache_func(q, cache, t, ls, SCALE, weights=w),
                     lambda: fm.flash_msa_cache_evict(cache, w, t, ls, table[:, :1].contiguous(), 128, 5),
                     lambda: fm.flash_msa_cache_evict(cache, w, table, ls, t[:, 1:2].contiguous(), 128, 5),
                     lambda: fm.flash_msa_cache_append(cache, q[:, :1], q[:, :1], t, ls - 100)):
            with pytest.raises(RuntimeError):
                call()
    with pytest.raises(RuntimeError):                                    # a length that the table has no page for
        fm.flash_msa_cache_append(cache, q[:, :1], q[:, :1], table, ls + 1000)
    assert cache.shape == before.shape
    out = fm.flash_msa_cache_func(q, before, table, ls, SCALE)           # and the next call is fine
    assert torch.isfinite(out.float()).all()


def test_pages_that_do_not_exist_for_many_rows(fm):
    cache, table, ls, g = pool(fm, [300, 300], 1, seed=12)
    q = torch.randn(2, 40, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    want = fm.flash_msa_cache_func(q, cache, table, ls, SCALE)
    before = cache.clone()
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 1] = bad
        w = torch.zeros(cache.shape[0], 1, 128, device="cuda")
        for weights in (None, w):
            with pytest.raises(RuntimeError):
                fm.flash_msa_cache_func(q, cache, t, ls, SCALE, weights=weights)
        unused = [p for p in range(cache.shape[0]) if p not in t.flatten().tolist()]
        assert (w[unused] == 0).all()
    assert torch.equal(cache, before) and torch.equal(fm.flash_msa_cache_func(q, cache, table, ls, SCALE), want)


@pytest.mark.parametrize("hq", [4, 12, 24])
def test_lengths_outside_the_table(fm, hq):
    """Below zero is zero; beyond what the table can hold is reported."""
    cache, table, ls, g = pool(fm, [256, 256, 256], 1, seed=14, spare=3)
    q = torch.randn(3, hq, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.rand(cache.shape[0], 1, 128, device="cuda")
    to = table.numel() + torch.arange(3, dtype=torch.int32, device="cuda").view(3, 1)
    for odd in ([256, 2 ** 31 - 1, 0], [257, 0, 0]):
        ls = torch.tensor(odd, dtype=torch.int32, device="cuda")
        for call in (lambda: fm.flash_msa_cache_func(q, cache, table, ls, SCALE), lambda: fm.flash_msa_cache_func(q, cache, table, ls, SCALE, weights=w),
                     lambda: fm.flash_msa_cache_evict(cache, w, table, ls, to, 100, 5)):
            with pytest.raises(RuntimeError):
                call()
    got = fm.flash_msa_cache_func(q, cache, table, torch.tensor([-(2 ** 31), 256, -1], dtype=torch.int32, device="cuda"), SCALE)
    assert torch.equal(got, fm.flash_msa_cache_func(q, cache, table, torch.tensor([0, 256, 0], dtype=torch.int32, device="cuda"), SCALE))
    assert (got[0] == 0).all() and (got[2] == 0).all()


# ---------------------------------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["random", "ties", "zeros", "odd"])
@pytest.mark.parametrize("lengths,hkv,keep,recent", [([1], 1, 1, 0), ([200], 2, 130, 0), ([200, 0, 129, 500], 3, 129, 129), ([700, 90], 1, 257, 60),
                                                     ([1000], 2, 1, 1), ([3000, 2999], 1, 2998, 7), ([9000, 100], 1, 5000, 100), ([40000], 1, 5000, 100),
                                                     ([1100, 30, 0, 513], 2, 512, 64), ([8000, 1024, 1025], 1, 1024, 0), ([9000, 5], 1, 700, 3)])
def test_evict(fm, lengths, hkv, keep, recent, kind):
    cache, table, ls, g = pool(fm, lengths, hkv, seed=keep, spare=len(lengths) * (-(-keep // 128)) + 2)
    own = len(lengths) * table.shape[1]
    to = (own + torch.randperm(cache.shape[0] - own, generator=g, device="cuda"))[:len(lengths) * (-(-keep // 128))].to(torch.int32).view(len(lengths), -1)
    w = torch.randn(cache.shape[0], hkv, 128, generator=g, device="cuda")
    if kind == "ties":
        w = torch.round(w * 2) / 4                      # a few values, the two zeros among them
    elif kind == "zeros":
        w.zero_()
    elif kind == "odd":
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.05] = math.nan
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.05] = math.inf
        w[torch.rand(w.shape, generator=g, device="cuda") < 0.05] = -math.inf
    old, old_w = cache.clone(), w.clone()
    new_lengths, kept = fm.flash_msa_cache_evict(cache, w, table, ls, to, keep, recent)
    want = R.evict(old_w, table, lengths, keep, recent)
    for i, length in enumerate(lengths):
        n = min(length, keep)
        assert int(new_lengths[i]) == n
        for h in range(hkv):
            assert kept[i, h].tolist() == want[i, h] + [-1] * (keep - n)
            if n:
                at = torch.tensor(want[i, h], device="cuda")
                for which in "kv":
                    assert torch.equal(R.rows_of(cache, to[i], n, h, which), R.rows_of(old, table[i], length, h, which)[at])
                j = torch.arange(n, device="cuda")
                assert torch.equal(w[to[i].long()[j // 128], h, j % 128].nan_to_num(7.0, 8.0, 9.0),
                                   old_w[table[i].long()[at // 128], h, at % 128].nan_to_num(7.0, 8.0, 9.0))
    # nothing else was written: not the old pages, not the places behind the last token
    for i, length in enumerate(lengths):
        n = min(length, keep)
        for p in range(to.shape[1]):
            first = max(0, min(128, n - 128 * p))
            page = int(to[i, p])
            for lo, row in ((0, 64), (8192, 8), (9216, 64), (17408, 8)):
                part = lambda c: c[page, :, lo:lo + 128 * row].view(hkv, 128, row)
                part(cache)[:, :first] = part(old)[:, :first]
            w[page, :, :first] = old_w[page, :, :first]
    assert torch.equal(cache, old) and torch.equal(w.nan_to_num(7.0), old_w.nan_to_num(7.0))


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------

def test_captured_steps(fm):
    """Append and attention in one graph, replayed with new inputs, lengths and tables; two graphs alive at once."""
    lengths = [200, 31]
    cache, table, ls, g = pool(fm, lengths, 2, seed=21, spare=5)
    table = torch.cat([table, torch.full((2, 1), -1, dtype=torch.int32, device="cuda")], 1)
    q, k, v = (torch.randn(2, h, 1, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (8, 2, 2))
    w = torch.zeros(cache.shape[0], 2, 128, device="cuda")
    from flash_msa_b200 import api
    api.DEBUG_CHECK_STATUS = False
    try:
        def step(weights):
            ls.add_(1)
            fm.flash_msa_cache_append(cache, k, v, table, ls, weights=weights)
            return fm.flash_msa_cache_func(q, cache, table, ls, SCALE, weights=weights)
        step(w)
        torch.cuda.synchronize()
        graphs = []
        for weights in (w, None):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(weights)
            graphs.append((graph, out))
        lengths = [int(x) for x in ls]
        for r in range(70):      # across a page boundary of both sequences
            graph, out = graphs[r % 2]
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
            lengths = [x + 1 for x in lengths]
            for i, x in enumerate(lengths):
                if x > 256 and table[i, 2] < 0:
                    table[i, 2] = cache.shape[0] - 1 - i
            graph.replay()
            if r % 23 == 0 or r > 60:
                want, tol, _ = R.attend(q, cache, table, lengths, SCALE)
                assert ((out.view(2, 1, 8, 128).double() - want).abs() <= tol).all()
    finally:
        api.DEBUG_CHECK_STATUS = True
    fm.check_pending_status()


def test_generation(fm):
    """A packed prefill into the cache, steps that attend and weigh, an eviction, and steps on what is left."""
    g = torch.Generator(device="cuda").manual_seed(31)
    b, hq, hkv, prompt = 3, 8, 2, [300, 17, 140]
    width = 4
    cache, w = fm.flash_msa_cache_empty(b * (width + 2), hkv), torch.zeros(b * (width + 2), hkv, 128, device="cuda")
    table = torch.randperm(b * width, generator=g, device="cuda").to(torch.int32).view(b, width)
    ls = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(1, hkv, sum(prompt), 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    cu = [0, 300, 317, 457]
    fm.flash_msa_cache_append(cache, k, v, table, ls, cu_seqlens=cu, weights=w)
    for step in range(6):
        if step == 3:
            new = (b * width + torch.arange(2 * b, device="cuda", dtype=torch.int32)).view(b, 2)
            ls, kept = fm.flash_msa_cache_evict(cache, w, table, ls, new, 150, 32)
            table = new
            assert ls.tolist() == [150, 20, 143]
        ls = ls + 1
        q, kn, vn = (torch.randn(b, h, 1, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv))
        fm.flash_msa_cache_append(cache, kn, vn, table, ls, weights=w)
        check_attend(fm, cache, table, ls, ls.tolist(), q, weights=w)
