"""The binding's C++ part is loaded only beside the torch and the Python that it was built against (no GPU)."""
import os
import sysconfig

import pytest
import torch

from conftest import load_package


def test_another_torch_is_refused(monkeypatch):
    pkg = load_package()
    args = pkg.cdna4.load_args()
    assert args.built_with == torch.__version__
    monkeypatch.setattr(pkg.cdna4, "_args", None)
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    with pytest.raises(RuntimeError, match="built against torch"):
        pkg.cdna4.load_args()
    monkeypatch.undo()
    assert pkg.cdna4.load_args() is not None


def test_the_file_says_which_python_it_is_for():
    pkg = load_package()
    from ik_llama_cpp_amd.build import BINDING
    assert BINDING.endswith(sysconfig.get_config_var("EXT_SUFFIX")) and os.path.exists(BINDING) and pkg.cdna4.load_args().__file__ == BINDING
