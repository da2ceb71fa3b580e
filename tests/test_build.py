"""What build.py compiles again: with a compiler that only writes down how it was called (no GPU, no hipcc)."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def builder(tmp_path, monkeypatch):
    spec = importlib.util.spec_from_file_location("_dm_build_under_test", os.path.join(ROOT, "diffusion-model_amd", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    csrc, log, cc = tmp_path / "csrc", tmp_path / "log", tmp_path / "cc"
    csrc.mkdir()
    for name in ("a.hip", "b.hip", "common.h"):
        (csrc / name).write_text(name)
    cc.write_text(f'#!/bin/sh\necho "$@" >> {log}\nif [ -e {tmp_path}/fail ]; then exit 1; fi\nwhile [ "$1" != -o ]; do shift; done\necho built > "$2"\n')
    cc.chmod(0o755)
    for name, value in (("CSRC", csrc), ("OBJ", tmp_path / "build"), ("LIBDIR", tmp_path / "lib"), ("LIB", tmp_path / "lib" / "x.so"), ("HIPCC", cc)):
        monkeypatch.setattr(mod, name, str(value))

    def calls(**kw):
        """sources compiled by one build, and whether it linked"""
        log.write_text("")
        mod.build(verbose=False, jobs=1, **kw)
        lines = log.read_text().splitlines()
        return [os.path.basename(w) for ln in lines if "-shared" not in ln for w in ln.split() if w.endswith(".hip")], any("-shared" in ln for ln in lines)

    return mod, calls, tmp_path


def test_compiled_again_when_flags_change(builder, monkeypatch):
    mod, calls, _ = builder
    both = ["a.hip", "b.hip"]
    assert calls() == (both, True)
    assert calls() == ([], False)
    monkeypatch.setattr(mod, "FLAGS", mod.FLAGS + ["-DNEW"])
    assert calls() == (both, True)                             # objects of other flags are not linked
    assert calls() == ([], False)
    assert calls(force=True) == (both, True)


def test_compiled_again_when_sources_change(builder):
    _, calls, tmp = builder
    calls()
    later = os.path.getmtime(tmp / "lib" / "x.so") + 10
    os.utime(tmp / "csrc" / "b.hip", (later, later))
    assert calls() == (["b.hip"], True)
    later += 10
    os.utime(tmp / "csrc" / "common.h", (later, later))
    assert calls()[0] == ["a.hip", "b.hip"]


def test_an_object_without_its_command_or_of_a_failed_build_is_not_taken(builder, monkeypatch):
    mod, calls, tmp = builder
    calls()
    for f in (tmp / "build").iterdir():                        # as builds left them that kept no commands
        if not f.name.endswith(".o"):
            f.unlink()
    assert calls()[0] == ["a.hip", "b.hip"]
    monkeypatch.setattr(mod, "FLAGS", mod.FLAGS + ["-DBAD"])
    (tmp / "fail").write_text("")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        calls()
    (tmp / "fail").unlink()
    assert calls() == (["a.hip", "b.hip"], True)
