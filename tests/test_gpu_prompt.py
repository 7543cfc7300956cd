"""Attention over whole prompts on the GPU, against a 64-bit restatement (tests/serving_ref.py, which derives the tolerances)."""
import math

import pytest
import torch

from tests import serving_ref as R
from tests.test_gpu_serving import SCALE, fm, layout  # noqa: F401

pytestmark = pytest.mark.gpu


def inputs(b, hq, hkv, s, seed, dtype=torch.bfloat16, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(b, h, s, 128, generator=g, device="cuda") * size).to(dtype) for h in (hq, hkv, hkv)]


def check(fm, q, k, v, cu=None, sinks=None, given="same"):
    b, hq, s, _ = q.shape
    out = fm.flash_msa_prompt_func(q, k, v, cu if given == "same" else given, SCALE, sinks=sinks)
    lists = [[0, s]] * b if cu is None else cu if isinstance(cu[0], list) else [cu] * b
    want, tol = R.prompt(q, k, v, lists, SCALE, sinks)
    assert out.shape == (b, s, hq * 128) and out.dtype == q.dtype
    err = (out.view(b, s, hq, 128).double() - want).abs()
    assert (err <= tol).all(), ((err - tol).max().item(), err.max().item())
    for i, c in enumerate(lists):
        assert (out[i, c[-1]:] == 0).all()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,hkv,s", [(1, 1, 1, 1), (1, 4, 1, 2), (2, 2, 2, 127), (1, 3, 1, 128), (1, 5, 1, 129), (1, 8, 2, 383), (1, 6, 3, 300), (1, 16, 1, 200),
                                        (1, 12, 1, 257), (1, 128, 1, 65), (1, 100, 1, 40), (3, 4, 2, 1000), (1, 1, 1, 2500), (1, 7, 1, 1409)])
def test_whole_sequences(fm, b, hq, hkv, s, dtype):
    check(fm, *inputs(b, hq, hkv, s, s + hq, dtype))


PACKED = {
    "ragged": (8, 2, 1000, [0, 1, 130, 131, 513, 1000]),
    "tail": (4, 1, 700, [0, 100, 228, 601]),
    "empty_ones": (6, 2, 300, [0, 0, 40, 40, 40, 299, 299]),
    "nothing": (4, 2, 50, [0, 0]),
    "tokens": (5, 1, 40, list(range(41))),
    "per_batch": (4, 2, 520, [[0, 100, 520, 520], [0, 0, 3, 500]]),
    "longer": (2, 1, 3000, [0, 2000, 2100, 3000]),
}


@pytest.mark.parametrize("host", ["list", "cpu", "cuda", "cuda64"])
@pytest.mark.parametrize("name", list(PACKED))
def test_packed(fm, name, host):
    hq, hkv, s, cu = PACKED[name]
    b = len(cu) if isinstance(cu[0], list) else 2 if name == "ragged" else 1
    q, k, v = inputs(b, hq, hkv, s, 7)
    given = {"list": cu, "cpu": torch.tensor(cu), "cuda": torch.tensor(cu, dtype=torch.int32).cuda(), "cuda64": torch.tensor(cu).cuda()}[host]
    check(fm, q, k, v, cu, given=given)


@pytest.mark.parametrize("n", [500, 1200])
def test_many_sequences(fm, n):
    """More boundaries than a kernel parameter holds, among them."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 9, (n,), generator=g)
    cu = [0] + lens.cumsum(0).tolist()
    check(fm, *inputs(1, 4, 2, cu[-1] + 5, 3), cu)


@pytest.mark.parametrize("kind", ["bshd", "odd", "wide"])
@pytest.mark.parametrize("sinks", [None, 0.0, 12.0, -60.0])
def test_layouts_and_sinks(fm, kind, sinks):
    q, k, v = (layout(t, kind) for t in inputs(2, 6, 2, 333, 5))
    s = None if sinks is None else torch.randn(6, device="cuda") + sinks
    check(fm, q, k, v, [0, 200, 300], s)
    check(fm, q[:1].expand(2, 6, 333, 128), k, v, None, s)


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e-3), (torch.bfloat16, 6.0), (torch.float16, 4.0), (torch.float16, 1e-3)])
def test_magnitudes(fm, dtype, size):
    check(fm, *inputs(1, 4, 2, 700, 9, dtype, size))


def test_slices_of_one_buffer(fm):
    qkv = torch.randn(2, 300, 8, 128, device="cuda").to(torch.bfloat16).transpose(1, 2)
    check(fm, qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], [0, 299])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (5, 1)])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(fm, hq, hkv, what, dtype):
    """Later tokens, other sequences and rows behind the last one may hold anything; rows that do see such a value show it."""
    s, cu = 900, [0, 100, 470, 850]
    q, k, v = inputs(1, hq, hkv, s, 13, dtype)
    want = check(fm, q, k, v, cu).view(s, hq, 128)
    for at in (99, 100, 257, 469, 470, 849, 850, 899):
        end = next((c for c in cu if c > at), at)            # the first row behind the sequence that holds it
        for bad in ("v", "k", "q"):
            q2, k2, v2 = q.clone(), k.clone(), v.clone()
            {"q": q2, "k": k2, "v": v2}[bad][:, :, at, 3 if bad == "v" else slice(None)] = what
            got = fm.flash_msa_prompt_func(q2, k2, v2, cu, SCALE).view(s, hq, 128)
            rows = torch.ones(s, dtype=torch.bool, device="cuda")
            rows[at:at + 1 if bad == "q" else end] = False
            assert torch.equal(got[rows], want[rows]), (at, bad)
            if at >= 850:
                continue
            if bad == "v":
                assert torch.equal(got[..., :3], want[..., :3]) and torch.equal(got[..., 4:], want[..., 4:])
                seen = got[~rows][..., 3].float()
                assert (seen.isnan() if what != what else seen == what).all()
            else:
                assert not torch.isfinite(got[at].float()).all(-1).any()
    v2 = v.clone()
    v2[:, :, 150, 3], v2[:, :, 200, 3] = math.inf, -math.inf     # two that meet
    got = fm.flash_msa_prompt_func(q, k, v2, cu, SCALE).view(s, hq, 128)
    assert (got[150:200, :, 3] == math.inf).all() and got[200:470, :, 3].isnan().all() and torch.equal(got[470:], want[470:])


def test_streams_graphs_and_repetition(fm):
    q, k, v = inputs(1, 8, 2, 1100, 17)
    cu = torch.tensor([0, 300, 1000], dtype=torch.int32, device="cuda")
    want = check(fm, q, k, v, [0, 300, 1000], given=cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fm.flash_msa_prompt_func(q, k, v, cu, SCALE)
    side.synchronize()
    assert torch.equal(got, want)
    from flash_msa_b200 import api
    api.DEBUG_CHECK_STATUS = False
    try:
        fm.flash_msa_prompt_func(q, k, v, cu, SCALE)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fm.flash_msa_prompt_func(q, k, v, cu, SCALE)
        for new in ([0, 300, 1000], [0, 1, 1100], [0, 0, 0], [0, 777, 900]):
            cu.copy_(torch.tensor(new, dtype=torch.int32))
            graph.replay()
            ref, tol = R.prompt(q, k, v, [new], SCALE)
            assert ((out.view(1, 1100, 8, 128).double() - ref).abs() <= tol).all()
    finally:
        api.DEBUG_CHECK_STATUS = True
    fm.check_pending_status()


def test_boundaries_in_device_memory_that_fall_or_leave_the_rows(fm):
    """Not what the call allows; but no kernel leaves its tensors for it, and the next call is fine."""
    q, k, v = inputs(1, 4, 2, 500, 19)
    for cu in ([0, 400, 100, 2000], [-5, 600], [700, 800], [0, 2 ** 31 - 1, -2 ** 31, 500] * 4):
        try:
            fm.flash_msa_prompt_func(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), SCALE)
        except RuntimeError as e:
            assert "out-of-range" in str(e)
    check(fm, q, k, v)


def test_prefill_then_steps_agree_with_the_whole_sequence(fm):
    """A prompt attended to on the values that the cache holds, then steps over the cache: the same rows as one causal pass over all of
    them, within both tolerances."""
    g = torch.Generator(device="cuda").manual_seed(23)
    s, new, hq, hkv = 300, 5, 8, 2
    q, k, v = inputs(1, hq, hkv, s + new, 29)
    cache = fm.flash_msa_cache_empty(3, hkv)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    at = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")
    ks, vs = fm.flash_msa_cache_append(cache, k[:, :, :s], v[:, :, :s], table, at(s), return_values=True)
    rows = [fm.flash_msa_prompt_func(q[:, :, :s], ks, vs, None, SCALE)]
    for i in range(s, s + new):
        kn, vn = fm.flash_msa_cache_append(cache, k[:, :, i:i + 1], v[:, :, i:i + 1], table, at(i + 1), return_values=True)
        ks, vs = torch.cat([ks, kn], 2), torch.cat([vs, vn], 2)
        rows.append(fm.flash_msa_cache_func(q[:, :, i:i + 1], cache, table, at(i + 1), SCALE))
    want, tol = R.prompt(q, ks, vs, [[0, s + new]], SCALE)
    held = sum(R.rows_of(cache, table[0], s + new, h, "v").abs().amax() for h in range(hkv))
    # (ks, vs are the cache's values rounded to 16 bits; each of K's roundings moves a logit by at most half a step of its terms)
    slack = 2.0 ** -8 * held * (1 + 4 * SCALE * (q.double().abs().amax(1)[0] @ ks.double().abs().amax(1)[0].T).amax())
    got = torch.cat(rows, 1).view(1, s + new, hq, 128).double()
    assert ((got - want).abs() <= 2 * tol + slack).all()
    assert torch.cat(rows, 1).shape == (1, s + new, hq * 128)
