"""The serving operators at the ends of what their documentation allows, and on tensors that hold what it does not allow, on the GPU."""
import math

import pytest
import torch

from tests import serving_ref as R
from tests.test_gpu_serving import SCALE, append_reference, check_attend, fm, layout, pool  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def late(fm):  # noqa: F811
    """Calls that return what they computed; what they met is reported by `check_pending_status()`."""
    from flash_msa_b200 import api
    fm.check_pending_status()
    api.DEBUG_CHECK_STATUS = False
    yield fm
    api.DEBUG_CHECK_STATUS = True


def reported(fm):
    with pytest.raises(RuntimeError, match="out-of-range"):
        fm.check_pending_status()
    fm.check_pending_status()


# ---------------------------------------------------------------------------------------------------------------------
# pages that do not exist
# ---------------------------------------------------------------------------------------------------------------------

def without(table, lengths, gone):
    """The table and the lengths of the same sequences without their pages gone[i] (None: all of them)."""
    rows, left = [], []
    for row, length, p in zip(table.tolist(), lengths, gone):
        rows.append(row if p is None else row[:p] + row[p + 1:] + [0])
        left.append(length if p is None else length - min(128, length - 128 * p))
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), left


# The last page only where one row of queries sees every token of it.  Forms: a cluster of either size, ranges of either size, rows of either count.
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("hq,hkv,n,lengths,gone", [
    (4, 1, 1, [1000, 300], [0, 2]), (4, 1, 2, [1000, 40, 900], [7 - 1, None, 0]), (8, 8, 1, [700] * 30, [i % 6 for i in range(30)]),
    (12, 1, 1, [4000, 5120] + [5000] * 30, [0, 39, None] + [i for i in range(29)]), (24, 2, 1, [1280] * 60, [i % 10 for i in range(60)]),
    (24, 1, 1, [700, 100, 1], [0, 0, 0]), (24, 1, 3, [700, 300], [0, 1]), (48, 1, 1, [4000] * 3, [0, 15, 31]), (100, 1, 1, [900, 300], [0, 2]),
    (1, 1, 1, [40000], [100])])
def test_tokens_of_pages_that_do_not_exist_are_hidden(late, hq, hkv, n, lengths, gone, weights):
    """The result is the one without those tokens, whatever the kernels have loaded before: the values that there are lie far below logits of
    zero (which is what nothing looks like), and everything that was not appended is NaN."""
    fm = late  # noqa: F811
    cache, table, ls, g = pool(fm, lengths, hkv, seed=3 * hq + n)
    mean = torch.stack([R.rows_of(cache, table[0], lengths[0], h, "k").mean(0) for h in range(hkv)]).float()
    q = torch.randn(len(lengths), hq, n, 128, generator=g, device="cuda")
    q[:, ::2] -= 20 * mean.repeat_interleave(hq // hkv, 0)[::2].view(1, -1, 1, 128)
    q = q.to(torch.bfloat16)
    t2, l2 = without(table, lengths, gone)
    want, tol, new = R.attend(q, cache, t2, l2, SCALE)
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        t = table.clone()
        for i, p in enumerate(gone):
            if p is not None:
                t[i, p] = bad
        w = torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda") if weights else None
        before = None if w is None else w.double()
        out = fm.flash_msa_cache_func(q, cache, t, ls, SCALE, weights=w)
        reported(fm)
        assert ((out.view(len(lengths), n, hq, 128).double() - want).abs() <= tol).all()
        if weights:
            slack = before.abs() * 2.0 ** -23
            for (i, h), (x, e) in new.items():
                at = torch.arange(len(x), device="cuda")
                before[t2[i].long()[at // 128], h, at % 128] += x
                slack[t2[i].long()[at // 128], h, at % 128] += e + x * 2.0 ** -20
            assert ((w.double() - before).abs() <= slack).all()


@pytest.mark.parametrize("hq", [4, 24])
def test_calls_with_pages_that_do_not_exist_write_nothing_else(late, hq):
    """The pool and the weights, byte by byte, and the next call on the same pool."""
    fm = late  # noqa: F811
    lengths = [300, 300]
    cache, table, ls, g = pool(fm, lengths, 1, seed=12, spare=4)
    q = torch.randn(2, hq, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn(2, 1, 200, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    weights = torch.rand(cache.shape[0], 1, 128, generator=g, device="cuda")
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 1] = bad
        old, w = cache.clone(), weights.clone()
        fm.flash_msa_cache_func(q, cache, t, ls, SCALE, weights=w)
        reported(fm)
        named = [int(x) for x in t.flatten() if 0 <= int(x) < cache.shape[0]]
        others = [p for p in range(cache.shape[0]) if p not in named]
        assert torch.equal(cache, old) and torch.equal(w[others], weights[others])
        # (a list that leads nowhere: nothing is moved)
        w = weights.clone()
        nowhere = torch.tensor([[bad], [bad]], dtype=torch.int32, device="cuda")
        fm.flash_msa_cache_evict(cache, w, table, ls, nowhere, 100, 5)
        reported(fm)
        assert torch.equal(cache, old) and torch.equal(w, weights)
        # (tokens 100 .. 299 of both sequences, of which those on the page that there is not are left out)
        got = fm.flash_msa_cache_append(cache, k, v, t, ls, weights=w, return_values=True)
        reported(fm)
        want, vals = append_reference(old, k, v, t, lengths, lambda i, j: None if i == 1 and (100 + j) // 128 == 1 else (i, 100 + j))
        assert torch.equal(cache.cpu(), want)
        for x, val in zip(got, vals):
            assert torch.equal(x.cpu(), val.to(torch.float32).to(x.dtype))
        for i in range(2):
            for j in range(100, 300):
                if (i, j // 128) != (1, 1):
                    assert w[t[i, j // 128].long(), 0, j % 128] == 0
        assert int((w != weights).sum()) <= 400 - 128
        check_attend(fm, cache, table, ls, lengths, q)


# ---------------------------------------------------------------------------------------------------------------------
# queries and values, in every form
# ---------------------------------------------------------------------------------------------------------------------

# clusters and ranges of eight and of sixteen rows, rows through shared memory in one and in several blocks
FORMS = {"cluster8": (6, 2, 2, [200, 0, 1]), "range8": (16, 8, 2, [130, 700, 0, 1, 257] * 6), "cluster16": (4, 1, 3, [5120] + [300, 0, 3] * 10),
         "range16": (8, 2, 3, [1280, 131, 2, 600] * 15), "rows": (24, 2, 2, [200, 0, 1, 700]), "blocks": (50, 1, 3, [200, 2, 0, 900])}


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("form", list(FORMS))
def test_query_layouts_in_every_form(fm, form, weights):  # noqa: F811
    hq, hkv, n, lengths = FORMS[form]
    cache, table, ls, g = pool(fm, lengths, hkv, seed=81)
    for dtype in (torch.bfloat16, torch.float16):
        q = torch.randn(len(lengths), hq, n, 128, generator=g, device="cuda").to(dtype)
        sinks = torch.randn(hq, generator=g, device="cuda")
        for x in (layout(q, "bshd"), layout(q, "odd"), layout(q, "wide"), q[:1].expand(q.shape), q[:, :1].expand(q.shape), q[:, :, :1].expand(q.shape)):
            w = torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda") if weights else None
            check_attend(fm, cache, table, ls, lengths, x, sinks, w)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("scale", [-0.05, 0.0, 1e-30, 3.0])
def test_scales_and_sinks_in_every_form(fm, form, scale):  # noqa: F811
    """Scales of either sign and none; sinks that take everything, or nothing."""
    hq, hkv, n, lengths = FORMS[form]
    cache, table, ls, g = pool(fm, lengths, hkv, seed=84)
    q = torch.randn(len(lengths), hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    for sinks in (None, torch.tensor([-math.inf, -1e30, 1e4, 0.0] * hq, device="cuda")[:hq].contiguous()):
        out = fm.flash_msa_cache_func(q, cache, table, ls, scale, sinks=sinks)
        want, tol, _ = R.attend(-q if scale < 0 else q, cache, table, lengths, abs(scale), sinks)
        assert ((out.view(want.shape).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("form", list(FORMS))
def test_tables_and_pools_that_are_parts_of_others(fm, form):  # noqa: F811
    """A table of some columns of a wider one, a row that all sequences share, a pool behind other records, keys that heads share by stride 0."""
    hq, hkv, n, lengths = FORMS[form]
    cache, table, ls, g = pool(fm, lengths, hkv, seed=85)
    b, width = table.shape
    q = torch.randn(b, hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    want = check_attend(fm, cache, table, ls, lengths, q)
    wide = torch.full((b, width + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + width] = table
    part = torch.cat([torch.full_like(cache[:3], 0xFF), cache])[3:]
    assert torch.equal(fm.flash_msa_cache_func(q, part, wide[:, 3:3 + width], ls, SCALE), want)
    one = max(range(b), key=lambda i: lengths[i])
    shared, same = table[one:one + 1].expand(b, width), torch.full_like(ls, lengths[one])
    check_attend(fm, cache, shared, same, [lengths[one]] * b, q)
    x = torch.randn(b, 1, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    for kv in (x.expand(b, hkv, 2, 128), x[:1].expand(b, hkv, 2, 128)):
        w = torch.rand(part.shape[0], hkv, 128, generator=g, device="cuda")
        a, c, w2 = part.clone(), cache.clone(), w.clone()
        got = fm.flash_msa_cache_append(a, kv, kv, wide[:, 3:3 + width], ls, weights=w, return_values=True)
        exp = fm.flash_msa_cache_append(c, kv.contiguous(), kv.contiguous(), table, ls, weights=w2, return_values=True)
        assert torch.equal(a, c) and torch.equal(w, w2) and all(torch.equal(y, z) for y, z in zip(got, exp))
    to = torch.full((b, 4), -1, dtype=torch.int32, device="cuda")
    # (the spare page: for the longest sequence, the others are empty)
    to[:, 1] = torch.where(torch.arange(b, device="cuda") == one, b * width, -1)
    few = torch.where(torch.arange(b, device="cuda") == one, ls, 0).to(torch.int32)
    w = torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda")
    kept = fm.flash_msa_cache_evict(cache.clone(), w.clone(), wide[:, 3:3 + width], few, to[:, 1:3], 100, 5)[1]
    ref = R.evict(w, table, few.tolist(), 100, 5)
    assert all(kept[one, h].tolist() == (ref[one, h] + [-1] * 100)[:100] for h in range(hkv))


@pytest.mark.parametrize("form", list(FORMS))
def test_values_that_are_not_finite_in_every_form(fm, form):  # noqa: F811
    """The last token, which only the last query of its sequence sees, and one that all see: other sequences and heads stay what they are bit for
    bit, and other rows but for their rounding; of V only the group of channels that holds the value shows it, K shows it in all of a row, and so
    do the weights."""
    hq, hkv, n, lengths = FORMS[form]
    cache, table, ls, g = pool(fm, lengths, hkv, seed=82)
    b, group = len(lengths), hq // hkv
    q = torch.randn(b, hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    call = lambda w=None: fm.flash_msa_cache_func(q, cache, table, ls, SCALE, weights=w).view(b, n, hkv, group, 128)
    want = call()
    seq = max(range(b), key=lambda i: (lengths[i] < 1000, lengths[i]))
    clean = cache.clone()
    for at in (lengths[seq] - 1, 5):
        rows = slice(n - 1, n) if at > 5 else slice(0, n)                 # of the sequence that see the token
        pairs = torch.ones(b, hkv, dtype=torch.bool, device="cuda")
        pairs[seq, 0] = False

        def alike(a, b):   # two sums of the same products: both within half a step, and 2^-11 of the values (below 8) for each probability
            return ((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -10 * 8).all()
        for which in ("v", "k"):
            cache.copy_(clean)
            record = cache[table[seq, at // 128].long(), 0]
            lo = (17408 if which == "v" else 8192) + at % 128 * 8 + 2     # the scale of the token's second group
            record[lo:lo + 2] = torch.tensor([0xFF, 0x7F], dtype=torch.uint8, device="cuda")
            got = call()
            assert torch.equal(got.transpose(1, 2)[pairs], want.transpose(1, 2)[pairs])
            assert alike(got[seq, :rows.start, 0].float(), want[seq, :rows.start, 0].float())
            seen = got[seq, rows, 0].float()
            if which == "k":
                assert seen.isnan().all()
            else:
                assert seen[..., 32:64].isnan().all()
                left = want[seq, rows, 0].float()
                for c in (slice(0, 32), slice(64, 128)):
                    assert alike(seen[..., c], left[..., c])
            w = torch.zeros(cache.shape[0], hkv, 128, device="cuda")
            call(w)
            page = table[seq, :-(-lengths[seq] // 128)].long()
            mine = w[page, 0].reshape(-1)[:lengths[seq]]
            assert (mine.isnan().all() if which == "k" and at == 5 else mine.isfinite().all() if which == "v" else mine.isnan().any())
            w[page, 0] = 0
            assert w.isfinite().all()


@pytest.mark.parametrize("form", list(FORMS))
def test_groups_of_channels_far_below_the_tokens_largest(fm, form):  # noqa: F811
    """A group 2^16 below the token's largest keeps its accuracy: as the same values with nothing larger beside them."""
    hq, hkv, n, lengths = FORMS[form]
    group = hq // hkv
    g = torch.Generator(device="cuda").manual_seed(83)
    total, b = sum(lengths), len(lengths)
    width = -(-max(lengths) // 128)
    k, v = (torch.randn(1, hkv, total, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    size = torch.exp2(torch.tensor([0.0, -16.0, -5.0, -11.0], device="cuda")).repeat_interleave(32)
    cu = torch.tensor([0] + lengths).cumsum(0).tolist()
    table = torch.arange(b * width, dtype=torch.int32, device="cuda").view(b, width)
    ls = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(b, hq, n, 128, generator=g, device="cuda").to(torch.bfloat16)
    outs = []
    for x in (v * size.to(torch.bfloat16), v):
        cache = fm.flash_msa_cache_empty(b * width, hkv)
        fm.flash_msa_cache_append(cache, k, x, table, ls, cu_seqlens=cu)
        outs.append(fm.flash_msa_cache_func(q, cache, table, ls, SCALE).view(b, n, hq, 128)[..., 32:64].float())
    got, want, top = outs[0] * 2.0 ** 16, outs[1], torch.zeros(b, n, hq, 1, device="cuda")
    for i, length in enumerate(lengths):          # every row's largest probability
        for h in range(hkv if length else 0):
            x = q[i, h * group:(h + 1) * group].double().reshape(group * n, 128)
            seen = torch.arange(length, device="cuda") < (length - n + 1 + torch.arange(n, device="cuda").repeat(group)).view(-1, 1)
            p = R.softmax((x @ R.rows_of(cache, table[i], length, h, "k").T * SCALE).masked_fill(~seen, -math.inf))
            top[i, :, h * group:(h + 1) * group] = p.amax(-1).view(group, n).T.unsqueeze(-1).float()
    # Both are sums of the same products, exact powers of two apart: half a step each, and the rounding of every probability times V's scale to fp16,
    # 2^-11 of the sum of magnitudes each.  What that loses below fp16's normal numbers is at most 2^-25 a token where the token's largest scale
    # makes 2^6 of the row's largest probability: here 2^-31 * 2^16 of a largest value for each token.
    size = v.float().abs().amax()
    assert ((got - want).abs() <= 2.0 ** -10 * size + 2.0 ** -7 * want.abs() + max(lengths) * 2.0 ** -15 * top * size).all()
    assert top.amax() > 0 and want.abs().amax() > 0.1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefill_and_steps_against_what_the_cache_holds(fm, dtype):  # noqa: F811
    """A prompt attended to on the values that the cache gives back, then steps over the cache: each against 64 bits within its own tolerance, which
    a result of zeros is not."""
    g = torch.Generator(device="cuda").manual_seed(23)
    s, new, hq, hkv = 300, 5, 8, 2
    q, k, v = (torch.randn(1, h, s + new, 128, generator=g, device="cuda").to(dtype) for h in (hq, hkv, hkv))
    cache = fm.flash_msa_cache_empty(3, hkv)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    at = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")
    ks, vs = fm.flash_msa_cache_append(cache, k[:, :, :s], v[:, :, :s], table, at(s), return_values=True)
    for x, which in ((ks, "k"), (vs, "v")):
        for h in range(hkv):
            held = R.rows_of(cache, table[0], s, h, which)
            assert torch.equal(x[0, h], held.to(torch.float32).to(dtype))
            given = (k if which == "k" else v)[0, h, :s].double().unflatten(-1, (4, 32))
            top = given.abs().amax(-1, keepdim=True)      # (half a step, and the rounding of the scale times the largest code)
            assert ((held.unflatten(-1, (4, 32)) - given).abs() <= top / 14 * (1 + 2.0 ** -8) + top * 2.0 ** -8).all()
    out = fm.flash_msa_prompt_func(q[:, :, :s], ks, vs, None, SCALE).view(1, s, hq, 128).double()
    want, tol = R.prompt(q[:, :, :s], ks, vs, [[0, s]], SCALE)
    assert ((out - want).abs() <= tol).all() and (want.abs() > tol).double().mean() > 0.9
    for i in range(s, s + new):
        fm.flash_msa_cache_append(cache, k[:, :, i:i + 1], v[:, :, i:i + 1], table, at(i + 1))
        want, tol, _ = R.attend(q[:, :, i:i + 1], cache, table, [i + 1], SCALE)
        out = fm.flash_msa_cache_func(q[:, :, i:i + 1], cache, table, at(i + 1), SCALE).view(1, 1, hq, 128).double()
        assert ((out - want).abs() <= tol).all() and (want.abs() > tol).double().mean() > 0.9


# ---------------------------------------------------------------------------------------------------------------------
# lengths beyond the table
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hq", [4, 12, 24, 100])
@pytest.mark.parametrize("far", [257, 300, 2 ** 31 - 1])
def test_sequences_longer_than_their_row_of_the_table_count_as_empty(late, hq, far):
    """In every call: nothing of them is read, weighed, stored or copied, and the calls say so; the others are what they are."""
    fm = late  # noqa: F811
    cache, table, ls, g = pool(fm, [256, 256, 40, 256], 1, seed=14, spare=8)
    lengths = [256, 0, 40, 0]
    odd = torch.tensor([256, far, 40, far], dtype=torch.int32, device="cuda")
    q = torch.randn(4, hq, 1, 128, generator=g, device="cuda").to(torch.bfloat16)
    want, tol, new = R.attend(q, cache, table, lengths, SCALE)
    for accumulate in (None, False, True):
        w = None if accumulate is None else torch.rand(cache.shape[0], 1, 128, generator=g, device="cuda")
        before = None if w is None else w.clone()
        out = fm.flash_msa_cache_func(q, cache, table, odd, SCALE, weights=w, accumulate=bool(accumulate))
        reported(fm)
        assert ((out.view(4, 1, hq, 128).double() - want).abs() <= tol).all() and (out[1] == 0).all() and (out[3] == 0).all()
        if w is not None:
            touched = torch.zeros(w.shape, dtype=torch.bool, device="cuda")
            for (i, h), (x, _) in new.items():
                at = torch.arange(len(x), device="cuda")
                touched[table[i].long()[at // 128], h, at % 128] = True
            assert torch.equal(w[~touched], before[~touched])
    # eviction
    w = torch.rand(cache.shape[0], 1, 128, generator=g, device="cuda")
    old, old_w = cache.clone(), w.clone()
    to = table.numel() + torch.arange(4, dtype=torch.int32, device="cuda").view(4, 1)
    new_lengths, kept = fm.flash_msa_cache_evict(cache, w, table, odd, to, 100, 7)
    reported(fm)
    assert new_lengths.tolist() == [100, 0, 40, 0] and (kept[1] == -1).all() and (kept[3] == -1).all()
    rest = [p for p in range(cache.shape[0]) if p not in (int(to[0]), int(to[2]))]
    assert torch.equal(cache[rest], old[rest]) and torch.equal(w[rest], old_w[rest])
    # new tokens: as many as the first sequences have room for, and packed ones
    cache.copy_(old)
    k, v = (torch.randn(4, 1, 3, 128, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    for args in (dict(), dict(cu_seqlens=[0, 3, 6, 9, 12])):
        kk, vv = (t.transpose(0, 1).reshape(1, 1, 12, 128) for t in (k, v)) if args else (k, v)
        got = fm.flash_msa_cache_append(cache, kk, vv, table, odd, weights=w, return_values=True, **args)
        reported(fm)
        assert all((x.view(4, 3, 128)[1::2] == 0).all() and (x.view(4, 3, 128)[::2] != 0).any() for x in got)
        pages = [int(table[i, p]) for i in (1, 3) for p in range(2)]
        assert torch.equal(cache[pages], old[pages]) and torch.equal(w[pages], old_w[pages])
        assert not torch.equal(cache[table[0, 1].long()], old[table[0, 1].long()])
        cache.copy_(old)


# ---------------------------------------------------------------------------------------------------------------------
# boundaries
# ---------------------------------------------------------------------------------------------------------------------

def test_many_boundaries_in_host_memory_are_captured(late):
    """More of them than one launch takes: the calls do not wait for the device, and can be captured."""
    fm = late  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(61)
    cu = [0] + torch.randint(0, 5, (2000,), generator=torch.Generator().manual_seed(1)).cumsum(0).tolist()
    n = cu[-1]
    q, k, v = (torch.randn(1, h, n, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 2))
    cache = fm.flash_msa_cache_empty(2000, 2)
    table = torch.arange(2000, dtype=torch.int32, device="cuda").view(2000, 1)
    ls = torch.tensor([b - a for a, b in zip(cu, cu[1:])], dtype=torch.int32, device="cuda")

    def call():
        fm.flash_msa_cache_append(cache, k, v, table, ls, cu_seqlens=cu)
        return fm.flash_msa_prompt_func(q, k, v, cu, SCALE)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    cache.zero_()
    out.zero_()
    graph.replay()
    fm.check_pending_status()
    want, tol = R.prompt(q, k, v, [cu], SCALE)
    assert ((out.view(1, n, 4, 128).double() - want).abs() <= tol).all()
    for i in (0, 1, 895, 896, 897, 1999):
        for h in range(2):
            codes, scales = R.quantize(k[0, h, cu[i]:cu[i + 1]])
            assert torch.equal(R.rows_of(cache, table[i], cu[i + 1] - cu[i], h, "k"), (codes.unflatten(-1, (4, 32)) * scales.unsqueeze(-1)).flatten(-2))


WRONG = [[0, 400, 100, 499], [1, 100, 200, 499], [0, 100, 200, 501], [-5, 0, 200, 499], [0, 2 ** 31 - 1, -2 ** 31, 499], [0, 499, 498, 498], [600, 700, 800, 900]]
RIGHT = [[0, 100, 200, 499], [0, 0, 0, 0], [0, 500, 500, 500], [0, 0, 0, 500], [0, 1, 2, 3]]


@pytest.mark.parametrize("hq,hkv,size", [(4, 2, 1), (8, 8, 20), (4, 2, 2000)])
@pytest.mark.parametrize("cu,wrong", [(c, True) for c in WRONG] + [(c, False) for c in RIGHT])
def test_boundaries_in_device_memory_that_do_not_rise_are_reported(late, cu, wrong, hq, hkv, size):
    """By prompts of few tiles (without a list of them) and of many, for each batch element that has its own, and by packed appends; those that do
    rise are not."""
    fm = late  # noqa: F811
    g = torch.Generator(device="cuda").manual_seed(71)
    n = 500 * size if size < 1000 else 500
    scaled = [max(-2 ** 31, min(2 ** 31 - 1, x * (n // 500))) for x in cu]
    if size == 2000:   # many sequences: what is wrong comes last, or first
        scaled = ([0] * 1200 + scaled) if cu[0] == 0 else scaled + [scaled[-1]] * 1200
    at = torch.tensor(scaled, dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(2, h, n, 128, generator=g, device="cuda").to(torch.bfloat16) for h in (hq, hkv, hkv))
    good = torch.zeros_like(at)
    for given, bad in ((at, wrong), (torch.stack([good, at]), wrong), (torch.stack([at, good]), wrong), (good, False)):
        fm.flash_msa_prompt_func(q, k, v, given, SCALE)
        if bad:
            reported(fm)
        else:
            fm.check_pending_status()
    seqs = len(scaled) - 1
    cache = fm.flash_msa_cache_empty(200, hkv)
    table = torch.zeros(seqs, 200, dtype=torch.int32, device="cuda")      # (what goes where does not matter here)
    fm.flash_msa_cache_append(cache, k[:1], v[:1], table, torch.full((seqs,), 25000, dtype=torch.int32, device="cuda"), cu_seqlens=at)
    if wrong:
        reported(fm)
    else:
        fm.check_pending_status()


# ---------------------------------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------------------------------

def evict_and_check(fm, lengths, hkv, keep, recent, fill_weights, seed, width=None):
    """Lists, and what was copied, against the plain restatement.  `width`: pages of a row of the table, where it is wider than the lengths need."""
    cache, table, ls, g = pool(fm, lengths, hkv, seed=seed, spare=len(lengths) * (-(-keep // 128)))
    own = len(lengths) * table.shape[1]
    to = torch.arange(own, cache.shape[0], dtype=torch.int32, device="cuda").view(len(lengths), -1)
    w = fill_weights(torch.rand(cache.shape[0], hkv, 128, generator=g, device="cuda") + 0.01, g)
    if width is not None:
        table = torch.cat([table, torch.full((len(lengths), width - table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
    old, old_w = cache.clone(), w.clone()
    new_lengths, kept = fm.flash_msa_cache_evict(cache, w, table, ls, to, keep, recent)
    want = R.evict(old_w, table, lengths, keep, recent)
    for i, length in enumerate(lengths):
        n = min(length, keep)
        assert int(new_lengths[i]) == n
        for h in range(hkv):
            assert kept[i, h].tolist() == want[i, h] + [-1] * (keep - n)
            if n == 0:
                continue
            at, j = torch.tensor(want[i, h], device="cuda"), torch.arange(n, device="cuda")
            for which in "kv":
                assert torch.equal(R.rows_of(cache, to[i], n, h, which), R.rows_of(old, table[i], length, h, which)[at])
            assert torch.equal(w[to[i].long()[j // 128], h, j % 128].view(torch.int32), old_w[table[i].long()[at // 128], h, at % 128].view(torch.int32))
    assert torch.equal(cache[:own], old[:own])


def some_nan(share):
    def fill(w, g):
        w[torch.rand(w.shape, generator=g, device="cuda") < share] = math.nan
        return w
    return fill


# (tables of up to 2K, 8K, 32K and more tokens go to different kernels)
@pytest.mark.parametrize("share", [0.5, 0.9, 1.0])
@pytest.mark.parametrize("lengths,hkv,keep,recent", [([1100, 700], 2, 512, 64), ([4100, 900], 2, 512, 64), ([20000], 2, 4000, 256), ([40000], 1, 4000, 256)])
def test_evict_with_more_nan_than_room(fm, lengths, hkv, keep, recent, share):
    """Weights that are NaN for more tokens than stay (a query row that is not finite leaves them), and finite positive ones: the first of the
    NaN ones stay, and nothing is written behind a list."""
    evict_and_check(fm, lengths, hkv, keep, recent, some_nan(share), seed=41)


@pytest.mark.parametrize("keep", [130, 1000])
@pytest.mark.parametrize("length,width", [(1100, 9), (1100, 40), (1100, 200), (1100, 300), (40000, 313)])
def test_evict_takes_tokens_of_pages_that_do_not_exist_last(late, length, width, keep):
    """Whichever kernel the width of the table asks for, and whatever the first page of the pool holds.  What has to stay all the same is copied
    as zeros."""
    fm = late  # noqa: F811
    recent, gone = 30, [0, 3, 4]
    if length > 2000:
        gone = list(range(2, 270))      # (five thousand others)
    cache, table, ls, g = pool(fm, [length], 2, seed=51, spare=8)
    to = (cache.shape[0] - 8 + torch.arange(8, dtype=torch.int32, device="cuda")).view(1, 8)
    w = torch.randn(cache.shape[0], 2, 128, generator=g, device="cuda")
    w[0] += 10
    ref = w.clone()
    t = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    t[:, :table.shape[1]] = table
    for p, bad in zip(gone, (-1, 2 ** 31 - 1, cache.shape[0]) * len(gone)):
        ref[table[0, p].long()] = -math.inf
        t[0, p] = bad
    want = R.evict(ref, table, [length], keep, recent)
    old, old_w = cache.clone(), w.clone()
    cache[to[0].long()] = 0xFF
    new_lengths, kept = fm.flash_msa_cache_evict(cache, w, t, ls, to, keep, recent)
    reported(fm)
    assert new_lengths.tolist() == [keep] and all(kept[0, h].tolist() == want[0, h] for h in range(2))
    for h in range(2):
        at, j = torch.tensor(want[0, h], device="cuda"), torch.arange(keep, device="cuda")
        there = torch.tensor([x // 128 not in gone for x in want[0, h]], device="cuda")
        assert there.all() == (keep == 130 or length > 2000)
        for which in "kv":
            rows = R.rows_of(cache, to[0], keep, h, which)
            assert torch.equal(rows, R.rows_of(old, table[0], length, h, which)[at] * there.view(-1, 1).double())
        assert torch.equal(w[to[0].long()[j // 128], h, j % 128], old_w[table[0].long()[at // 128], h, at % 128] * there)


def ties(w, g):
    return torch.round(w * 4) / 4


@pytest.mark.parametrize("fill", [lambda w, g: w, ties, some_nan(0.5), some_nan(0.01)])
@pytest.mark.parametrize("lengths,hkv,keep,recent", [([20000], 1, 4000, 100), ([1100, 3, 0], 2, 512, 64), ([24676, 24677], 1, 300, 100), ([33000], 1, 32000, 0)])
def test_evict_under_a_table_beyond_32k_tokens(fm, lengths, hkv, keep, recent, fill):  # noqa: F811
    """The form for long tables with sequences whose weights fit its shared memory, just so and just not."""
    evict_and_check(fm, lengths, hkv, keep, recent, fill, seed=42, width=300)
