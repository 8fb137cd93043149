"""The counter of the extension's kernel launches."""

import pytest

from dtensor_muon_b200.ops import _ext


@pytest.mark.skipif(not _ext.available(), reason="needs the built extension")
def test_the_counter_can_be_set(monkeypatch):
    before = _ext.launch_count
    try:
        _ext.launch_count = 0
        assert _ext.launch_count == 0

        class Module:
            launched = 7

            def launches_counted(self):
                return self.launched

            def rope(self):
                pass

        monkeypatch.setattr(_ext, "_C", _ext._Counted(Module()))
        _ext.launch_count = 0
        _ext._C.rope()
        Module.launched += 2
        assert _ext.launch_count == 3  # it counts on from there
    finally:
        monkeypatch.undo()
        _ext.launch_count = before
    assert _ext.launch_count == before
