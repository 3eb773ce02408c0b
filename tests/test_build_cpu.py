"""CPU: when build.py takes the library that is there, and when it compiles (the compiler itself is replaced)."""
import importlib.util
import os
import types

import pytest

from conftest import MODELS


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with its outputs in a folder of its own and a compiler that writes empty files and is counted."""
    spec = importlib.util.spec_from_file_location("ac_build_under_test", os.path.join(MODELS, "acnative", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.LIB, mod.OBJ_DIR = str(tmp_path / "libac_hip.so"), str(tmp_path / "build")
    mod.calls = []

    def run(cmd, **_):
        mod.calls.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")
    monkeypatch.setattr(mod.subprocess, "run", run)
    monkeypatch.setenv("HIPCC", os.devnull)
    return mod


def test_a_library_of_the_same_sources_and_flags_is_taken(build):
    assert build.build(verbose=False) == build.LIB
    n = len(build.calls)
    assert n == len(build._sources()) + 1
    build.build(verbose=False)
    assert len(build.calls) == n
    build.build(verbose=False, force=True)
    assert len(build.calls) == 2 * n


@pytest.mark.parametrize("change", ["flags", "file flags", "flag taken out", "library without a record"])
def test_other_flags_compile_again(build, change):
    """A flag can carry correctness (the one against packed fp32 instructions does), so a library of other flags is stale."""
    build.build(verbose=False)
    n = len(build.calls)
    if change == "flags":
        build.FLAGS = build.FLAGS + ["-DAC_OTHER=1"]
    elif change == "file flags":
        build.FILE_FLAGS = {}
    elif change == "flag taken out":
        build.FLAGS = build.FLAGS[:-1]
    else:                                              # as builds before the record left it
        for f in os.listdir(build.OBJ_DIR):
            if not f.endswith(".o"):
                os.remove(os.path.join(build.OBJ_DIR, f))
    build.build(verbose=False)
    assert len(build.calls) == 2 * n
    build.build(verbose=False)
    assert len(build.calls) == 2 * n


def test_a_failed_build_is_not_taken_for_current(build, monkeypatch):
    build.build(verbose=False)
    build.FLAGS = build.FLAGS + ["-DAC_OTHER=1"]
    run = build.subprocess.run
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **_: types.SimpleNamespace(returncode=1, stdout="", stderr="no"))
    with pytest.raises(RuntimeError, match="hipcc failed"):
        build.build(verbose=False)
    monkeypatch.setattr(build.subprocess, "run", run)
    n = len(build.calls)
    build.build(verbose=False)
    assert len(build.calls) > n
