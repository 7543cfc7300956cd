"""Host side of the serving operators, without a GPU: refusals, boundaries, the layout of the cache."""
import ctypes

import pytest
import torch

import flash_msa_b200 as fm
from flash_msa_b200 import _lib, serving
from tests import serving_ref as R

F = torch.float32
BF = torch.bfloat16


def test_constants_of_the_header():
    import re
    with open(_lib.HEADER_PATH) as f:
        text = f.read()
    for name, value in (("FMSA_CACHE_PAGE", serving.PAGE), ("FMSA_CACHE_RECORD_BYTES", serving.RECORD_BYTES)):
        assert int(re.search(rf"#define {name}\s+(\d+)", text).group(1)) == value


def test_unpack_reads_what_the_layout_says():
    g = torch.Generator().manual_seed(1)
    cache = torch.randint(0, 256, (2, 3, serving.RECORD_BYTES), generator=g, dtype=torch.uint8)
    for lo, hi in ((8192, 9216), (17408, 18432)):
        cache[..., lo:hi] = (torch.rand(2, 3, 512, generator=g) + 0.1).to(BF).view(torch.uint8)
    k, v = fm.flash_msa_cache_unpack(cache)
    assert k.shape == v.shape == (2, 3, 128, 128)
    assert torch.equal(k.double(), R.unpack(cache, "k")) and torch.equal(v.double(), R.unpack(cache, "v"))
    row = torch.randn(128, generator=g).to(BF)
    rec = torch.zeros(serving.RECORD_BYTES, dtype=torch.uint8)
    for slot in (0, 5, 127):
        R.pack_into(rec, slot, "k", row)
        R.pack_into(rec, slot, "v", row)
        q, s = R.quantize(row)
        want = (q.unflatten(-1, (4, 32)) * s.unsqueeze(-1)).flatten()
        got = fm.flash_msa_cache_unpack(rec)
        assert torch.equal(got[0][slot].double(), want) and torch.equal(got[1][slot].double(), want)
        assert ((want - row.double()).abs().view(4, 32) <= s.view(4, 1) / 2 + 2.0 ** -8 * row.double().abs().view(4, 32)).all()


def _call(what, **change):
    """A call of the operator on CPU tensors that is right but for the device, with arguments replaced."""
    a = dict(cache=torch.zeros(4, 2, serving.RECORD_BYTES, dtype=torch.uint8), k=torch.zeros(3, 2, 1, 128, dtype=BF),
             v=torch.zeros(3, 2, 1, 128, dtype=BF), q=torch.zeros(3, 4, 1, 128, dtype=BF), table=torch.zeros(3, 2, dtype=torch.int32),
             lengths=torch.ones(3, dtype=torch.int32), weights=torch.zeros(4, 2, 128), new=torch.zeros(3, 1, dtype=torch.int32), keep=100,
             recent=10, cu=None, sinks=None, pq=torch.zeros(2, 4, 7, 128, dtype=BF), pk=torch.zeros(2, 2, 7, 128, dtype=BF),
             pv=torch.zeros(2, 2, 7, 128, dtype=BF), scale=0.1)
    a.update(change)
    if what == "prompt":
        return fm.flash_msa_prompt_func(a["pq"], a["pk"], a["pv"], a["cu"], a["scale"], sinks=a["sinks"])
    if what == "append":
        return fm.flash_msa_cache_append(a["cache"], a["k"], a["v"], a["table"], a["lengths"], cu_seqlens=a["cu"], weights=a["weights"])
    if what == "attend":
        return fm.flash_msa_cache_func(a["q"], a["cache"], a["table"], a["lengths"], 0.1, sinks=a["sinks"], weights=a["weights"])
    return fm.flash_msa_cache_evict(a["cache"], a["weights"], a["table"], a["lengths"], a["new"], a["keep"], a["recent"])


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


COMMON = [
    (dict(cache=z(4, 2, 100, dtype=torch.uint8)), ValueError), (dict(cache=z(4, 2, 18432)), ValueError),
    (dict(cache=z(4, 4, 18432, dtype=torch.uint8)[:, ::2]), ValueError), (dict(cache=z(0, 2, 18432, dtype=torch.uint8), weights=z(0, 2, 128, dtype=F)), ValueError),
    (dict(table=z(3, 2, dtype=torch.int64)), TypeError), (dict(table=z(3, dtype=torch.int32)), TypeError),
    (dict(table=z(2, 3, dtype=torch.int32).T), ValueError), (dict(table=z(3, 0, dtype=torch.int32)), ValueError),
    (dict(lengths=z(3, dtype=torch.int64)), TypeError), (dict(lengths=z(2, dtype=torch.int32)), ValueError),
    (dict(lengths=z(6, dtype=torch.int32)[::2]), ValueError), (dict(weights=z(4, 2, 128)), ValueError),
    (dict(weights=z(4, 2, 127, dtype=F)), ValueError), (dict(weights=z(4, 2, 256, dtype=F)[..., ::2]), ValueError), (dict(), RuntimeError)]
APPEND = [
    (dict(k=z(3, 2, 1, 64)), NotImplementedError), (dict(k=z(3, 2, 128)), ValueError), (dict(k=z(3, 2, 1, 128, dtype=F)), TypeError),
    (dict(v=z(3, 2, 1, 128, dtype=torch.float16)), TypeError), (dict(v=z(3, 2, 2, 128)), ValueError),
    (dict(k=z(3, 1, 1, 128), v=z(3, 1, 1, 128)), ValueError), (dict(k=z(2, 2, 1, 128), v=z(2, 2, 1, 128)), ValueError),
    (dict(cu=[0, 1, 1, 1]), ValueError), (dict(cu=[0, 1, 1], k=z(1, 2, 5, 128), v=z(1, 2, 5, 128)), ValueError),
    (dict(k=z(3, 2, 1, 128).requires_grad_()), RuntimeError)]
ATTEND = [
    (dict(q=z(3, 5, 1, 128)), ValueError), (dict(q=z(3, 0, 1, 128)), ValueError), (dict(q=z(2, 4, 1, 128)), ValueError), (dict(q=z(3, 4, 1, 64)), NotImplementedError),
    (dict(q=z(3, 4, 1, 128, dtype=F)), TypeError), (dict(sinks=z(3, dtype=F)), ValueError), (dict(q=z(3, 4, 1, 128).requires_grad_()), RuntimeError)]
EVICT = [
    (dict(keep=0), ValueError), (dict(recent=101), ValueError), (dict(recent=-1), ValueError), (dict(keep=129, recent=0), ValueError),
    (dict(new=z(2, 1, dtype=torch.int32)), ValueError), (dict(new=z(3, 1, dtype=torch.int64)), TypeError), (dict(weights=None), ValueError)]

PROMPT = [
    (dict(), RuntimeError), (dict(pq=z(2, 4, 128)), ValueError), (dict(pq=z(2, 5, 7, 128)), ValueError), (dict(pq=z(2, 0, 7, 128)), ValueError),
    (dict(pq=z(2, 258, 7, 128)), NotImplementedError), (dict(pq=z(2, 4, 6, 128)), ValueError), (dict(pq=z(1, 4, 7, 128)), ValueError),
    (dict(pv=z(2, 1, 7, 128)), ValueError), (dict(pk=z(2, 2, 7, 128, dtype=torch.float16)), TypeError), (dict(pv=z(2, 2, 7, 64)), NotImplementedError),
    (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=float("nan")), ValueError), (dict(sinks=z(5, dtype=F)), ValueError),
    (dict(cu=[0]), ValueError), (dict(cu=[[0, 7]]), ValueError), (dict(pk=z(2, 2, 7, 128).requires_grad_()), RuntimeError)]


@pytest.mark.parametrize("what,change,error", [(w, c, e) for w, more in (("append", COMMON + APPEND), ("attend", COMMON + ATTEND),
                                                                         ("evict", COMMON + EVICT), ("prompt", PROMPT)) for c, e in more])
def test_refusals(what, change, error):
    with pytest.raises(error):
        _call(what, **change)


@pytest.mark.parametrize("what", ["append", "attend", "prompt"])
def test_derivatives_and_traces_are_refused(what):
    name = {"append": "k", "attend": "q", "prompt": "pq"}[what]
    shape = (2, 4, 7, 128) if what == "prompt" else (3, 4, 1, 128) if what == "attend" else (3, 2, 1, 128)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z(*shape), z(*shape))
        with pytest.raises(RuntimeError, match="forward-mode"):
            _call(what, **{name: dual})
        with pytest.raises(RuntimeError, match="CUDA"):      # (a level without a tangent is not in the way)
            _call(what)

    def traced(t):
        _call(what, **{name: t})
        return t
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(traced, (z(*shape),))
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        _call(what, **{name: z(*shape).requires_grad_()})


@pytest.mark.parametrize("what", ["append", "attend", "evict"])
def test_weights_that_want_a_gradient_are_refused(what):
    weights = torch.zeros(4, 2, 128, requires_grad=True)     # (the calls write them in place)
    with pytest.raises(RuntimeError, match="no backward"):
        _call(what, weights=weights)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        _call(what, weights=weights)


@pytest.mark.parametrize("cu", [[0, 3, 2], [1, 3], [0, 9], [0], [[[0, 1]]]])
def test_boundaries_that_are_refused(cu):
    with pytest.raises(ValueError):
        serving._boundaries(cu, 8, torch.device("cpu"))


def _block(kind, **change):
    """An argument block that is right but for what `change` replaces (pointers that are never dereferenced)."""
    a = dict(cache=(16, 16, 16, 2, 4, 2, 3, 2), k=(16, 256, 128, 128), v=(16, 256, 128, 128), values=(0,) * 8, q=(16, 256, 128, 128), cu=0, weights=16,
             status=16, b=3, n=1, dtype=0, hq=4, out=256, ws=256, ws_bytes=1 << 40, scale=0.1, new=16, stride=1, width=1, keep=100, recent=10, s=100, hkv=1,
             n_seqs=1)
    a.update(change)
    if kind == "append":
        return serving._APPEND_ARGS.pack(*a["cache"], *a["k"], *a["v"], *a["values"], a["cu"], a["weights"], a["status"], a["b"], a["n"], a["dtype"], 0)
    if kind == "attend":
        return serving._ATTEND_ARGS.pack(*a["cache"], *a["q"], 0, a["weights"], a["out"], a["ws"], a["ws_bytes"], a["status"], a["hq"], a["n"], a["dtype"],
                                         1, a["scale"], 0)
    if kind == "evict":
        return serving._EVICT_ARGS.pack(*a["cache"], a["weights"], a["new"], a["stride"], 16, 16, a["status"], a["width"], a["keep"], a["recent"], 0)
    return serving._PROMPT_ARGS.pack(*a["q"], *a["k"], *a["v"], a["cu"], 0, a["out"], a["ws"], a["ws_bytes"], a["status"], 1, a["s"], a["hq"], a["hkv"],
                                     a["n_seqs"], 0, a["dtype"], a["scale"])


ODD = (0x12, 256, 128, 128)          # off the 16-byte grid
CACHE = (16, 16, 16, 2, 4, 2, 3, 2)
ENTRIES = {"append": "fmsa_cache_append", "attend": "fmsa_cache_attend", "evict": "fmsa_cache_evict", "prompt": "fmsa_prompt_fwd"}
C_REFUSALS = [
    ("append", dict(b=2), -1), ("append", dict(dtype=7), -1), ("append", dict(values=(16, 256, 128, 128, 0, 0, 0, 0)), -1), ("append", dict(k=ODD), -1),
    ("append", dict(v=(0, 256, 128, 128)), -1), ("append", dict(v=(16, 256, 128, 12)), -1), ("append", dict(n=1 << 30), -2), ("append", dict(cache=(16, 16, 16, 2, 1 << 23, 2, 3, 2)), -2), ("append", dict(n=0), -1),
    ("append", dict(status=0), -1), ("append", dict(cu=16), -1),
    ("attend", dict(hq=5), -1), ("attend", dict(q=ODD), -1), ("attend", dict(dtype=-1), -1), ("attend", dict(out=0), -1), ("attend", dict(ws=0), -1),
    ("evict", dict(keep=129, recent=0), -1), ("evict", dict(recent=101), -1), ("evict", dict(keep=0, recent=0), -1), ("evict", dict(weights=0), -1),
    ("evict", dict(new=0), -1), ("evict", dict(cache=CACHE[:6] + (70000, 2)), -2),
    ("prompt", dict(scale=0.0), -1), ("prompt", dict(scale=float("nan")), -1), ("prompt", dict(ws_bytes=100), -3), ("prompt", dict(k=ODD), -1),
    ("prompt", dict(v=(16, 256, 128, 64)), -1), ("prompt", dict(s=(1 << 30) + 1), -2), ("prompt", dict(hq=258), -2), ("prompt", dict(hkv=3), -1),
    ("prompt", dict(out=8), -1), ("prompt", dict(cu=16, n_seqs=0), -1)]
C_REFUSALS += [(k, dict(cache=c), -1) for k in ("append", "attend", "evict") for c in
               ((0,) + CACHE[1:], (8,) + CACHE[1:], (16, 0) + CACHE[2:], CACHE[:4] + (0, 2, 3, 2), CACHE[:7] + (0,), CACHE[:3] + (-1,) + CACHE[4:])]


@pytest.mark.parametrize("kind,change,status", C_REFUSALS)
def test_c_entries_refuse_before_they_touch_anything(kind, change, status):
    lib = _lib.load()
    assert getattr(lib, ENTRIES[kind])(_block(kind, **change), None) == status
    assert getattr(lib, ENTRIES[kind])(None, None) == -1


def test_other_c_entries():
    lib = _lib.load()
    assert lib.fmsa_prompt_workspace_bytes(1, 100, 3, 2, 1) == -1 and lib.fmsa_prompt_workspace_bytes(2, 50000, 4, 2, 3) > 0
    assert lib.fmsa_cache_attend_workspace_bytes(1, 3, 2, 1, 1, 0) == -1
    assert lib.fmsa_boundaries(None, 3, None, None) == -1
    assert lib.fmsa_boundaries((ctypes.c_int32 * 4)(), 897, 0x10, None) == -2


def test_argument_blocks_have_the_size_of_the_headers_structures(tmp_path):
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    assert cc
    names = [("fmsa_cache_append_args", serving._APPEND_ARGS), ("fmsa_cache_attend_args", serving._ATTEND_ARGS),
             ("fmsa_cache_evict_args", serving._EVICT_ARGS), ("fmsa_prompt_args", serving._PROMPT_ARGS)]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "%s"\nint main(void) { printf("%s\\n", %s); return 0; }\n' % (
        _lib.HEADER_PATH, " ".join(["%zu"] * len(names)), ", ".join(f"sizeof({n})" for n, _ in names)))
    subprocess.run([cc, str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == [s.size for _, s in names]
