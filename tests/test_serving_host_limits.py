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
