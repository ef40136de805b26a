"""Loading of the torch extension by several threads, and of one that does not belong to the library (no
GPU needed)."""
import threading
import time
import types

import pytest

from prism_b200 import _lib
from prism_b200 import build as b


class _Loader:
    """Stands in for the extension's loader."""
    loads, abi = 0, None

    def __init__(self, name, path):
        pass

    def create_module(self, spec):
        return types.ModuleType(spec.name)

    def exec_module(self, module):
        type(self).loads += 1
        time.sleep(0.1)
        if self.abi is not None:
            module.abi_version = self.abi
        module.set_error = lambda error: None


@pytest.fixture
def loader(tmp_path, monkeypatch):
    import importlib.machinery
    path = tmp_path / "ext.so"
    path.write_bytes(b"")
    fake = type("Loader", (_Loader,), {"abi": _lib.load().prism_abi_version()})
    monkeypatch.setattr(_lib, "_torch_ops", None)
    monkeypatch.setattr(b, "torch_ops_lib", lambda: str(path))
    monkeypatch.setattr(importlib.machinery, "ExtensionFileLoader", fake)
    return fake


def test_threads_load_it_once(loader):
    got = []
    threads = [threading.Thread(target=lambda: got.append(_lib.torch_ops())) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert loader.loads == 1 and len(got) == 4 and all(m is got[0] for m in got)


@pytest.mark.parametrize("abi", [None, -1])
def test_an_extension_of_another_abi_is_refused(loader, abi):
    loader.abi = abi
    with pytest.raises(_lib.PrismError, match="ABI"):
        _lib.torch_ops()
    loader.abi = _lib.load().prism_abi_version()   # rebuilt
    assert _lib.torch_ops().abi_version == loader.abi
