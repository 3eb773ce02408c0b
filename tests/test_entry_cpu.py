"""CPU: __graft_entry__.build() compiles every time it is called."""
import importlib.util
import os

import __graft_entry__
from conftest import MODELS


def test_build_compiles_where_a_library_is_there(monkeypatch):
    asked = []
    real = importlib.util.module_from_spec

    def module_from_spec(spec):
        mod = real(spec)
        if spec.name == "ac_build":
            load = spec.loader.exec_module

            def exec_module(m):
                load(m)
                m.build = lambda force=False, **_: asked.append(force) or os.path.join(MODELS, "acnative", "libac_hip.so")
            monkeypatch.setattr(spec.loader, "exec_module", exec_module)
        return mod
    monkeypatch.setattr(importlib.util, "module_from_spec", module_from_spec)
    monkeypatch.delenv("AC_FORCE_BUILD", raising=False)
    monkeypatch.setattr(__graft_entry__, "_write_build_head", lambda where: None)
    __graft_entry__.build()
    assert asked == [True]
