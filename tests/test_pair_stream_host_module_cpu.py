"""The host module is a torch extension: it is loaded with the torch it was compiled against, and with torch's libraries."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from fold_cp_ops_b200 import _lib

REPO = Path(__file__).resolve().parent.parent


def test_another_torch_is_refused(monkeypatch):
    own = _lib.pair_host().torch_version
    for version, fits in ((own, True), (own + "+cu128", True), (own + "a0+git1234", True), (own + "1", False), ("2.1.0+cu121", False)):
        monkeypatch.setattr(_lib, "_pair", None)
        monkeypatch.setattr(torch, "__version__", version)
        if fits:
            _lib.pair_host()
        else:
            with pytest.raises(_lib.TrimulLibraryError, match="built against torch"):
                _lib.pair_host()


def test_the_module_loads_without_torch_imported_before():
    code = "from fold_cp_ops_b200 import _lib; _lib.pair_host()"
    subprocess.run([sys.executable, "-c", code], cwd=REPO, check=True, capture_output=True, timeout=300)
