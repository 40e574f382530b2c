"""The extension module belongs to the torch and the Python that it was built for (no GPU)."""
import os
import sysconfig

import pytest
import torch

from oregon_gpt_oss_patching_b200 import _binding, build


def test_another_torch_does_not_take_the_module(monkeypatch):
    build.build()
    assert not build.is_stale() and os.path.exists(build.binding_path())
    for there in (torch.__version__, sysconfig.get_config_var("EXT_SUFFIX")):
        assert there in os.path.basename(build.binding_path())
    monkeypatch.setattr(torch, "__version__", "0.0.0+other")
    assert build.is_stale()
    monkeypatch.setattr(_binding, "_module", None)
    with pytest.raises(RuntimeError, match="has not been built"):
        _binding.load()
