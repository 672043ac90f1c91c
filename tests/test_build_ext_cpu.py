"""Building the device extension from a process that runs on it."""

import os

import pytest

from torch_mcpu_b200 import build_ext


def test_a_loaded_extension_is_not_built_and_loaded_again(monkeypatch):
    """A second build, loaded beside the first, would register its operators twice, which ends the process."""
    if not os.path.exists(build_ext.SO):
        pytest.skip("the device extension is not built")
    import torch_mcpu_b200.device  # noqa: F401

    from torch.utils import cpp_extension

    def load(*a, **k):
        raise AssertionError("built again")

    monkeypatch.setattr(cpp_extension, "load", load)
    monkeypatch.setattr(build_ext, "up_to_date", lambda: False)
    assert build_ext.build() == build_ext.SO
