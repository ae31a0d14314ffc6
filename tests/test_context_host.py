"""Objects of the library that live to the end of the interpreter, without a GPU."""
import pytest

from paged_infer_b200 import _lib, api


@pytest.mark.parametrize("name", ["Context", "Projection", "KvCache", "KvCache8", "StatePool", "LlamaWeights", "LayeredModel"])
def test_closing_after_the_binding_is_gone(monkeypatch, name):
    """What a module holds is closed when the binding's globals are None already; nothing is raised and nothing called."""
    thing = object.__new__(getattr(api, name))
    thing.handle = 1                                     # no address: a call with it would end the process
    monkeypatch.setattr(_lib, "lib", None)
    thing.close()
    thing.handle = None
