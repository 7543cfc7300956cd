"""Host side of the serving operators at the ends of what they allow, without a GPU."""
import pytest
import torch

from flash_msa_b200 import _lib
from tests import conftest
from tests.test_serving_host import _block


def test_workspaces_that_are_too_small_are_refused():
    """Sizes that need one on every device."""
    lib = _lib.load()
    need = lib.fmsa_prompt_workspace_bytes(1, 50000, 4, 1, 1)
    assert need > 256
    assert lib.fmsa_prompt_fwd(_block("prompt", s=50000, ws_bytes=need - 1), None) == -3


@pytest.mark.parametrize("there", [False, True])
def test_made_up_addresses_are_kept_from_a_gpu(monkeypatch, there):
    class Item:
        def __init__(self, name):
            self.originalname, self.markers = name, []

        def add_marker(self, m):
            self.markers.append(m.name)
    items = [Item("test_c_entries_refuse_before_they_touch_anything"), Item("test_refusals")]
    monkeypatch.setattr(torch.cuda, "is_available", lambda: there)
    conftest.pytest_collection_modifyitems(items)
    assert [i.markers for i in items] == [["skip"] if there else [], []]


@pytest.mark.parametrize("n", [1, 895, 896, 897, 1792, 5000])
def test_boundaries_go_in_parts_that_a_launch_holds(monkeypatch, n):
    """However many there are: every one once, in its place."""
    import ctypes

    from flash_msa_b200 import ops, serving

    class Library:
        sent = []

        def fmsa_boundaries(self, src, count, dst, stream):
            assert 0 < count <= ops.MAX_HOST_BOUNDARIES and stream == 7
            ctypes.memmove(dst, src, 4 * count)
            self.sent.append(count)
            return 0
    lib = Library()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    src, dst = torch.arange(n, dtype=torch.int32), torch.full((n + 2,), -7, dtype=torch.int32)
    before = ops.LAUNCHES
    serving._send_boundaries(src.data_ptr(), n, dst.data_ptr() + 4, 7, None)
    assert torch.equal(dst[1:-1], src) and dst[0] == dst[-1] == -7
    assert sum(lib.sent) == n and ops.LAUNCHES - before == len(lib.sent) == -(-n // 896)
