"""What the in-tree build rebuilds: every header of ours that a source includes, directly or through another one."""
import importlib.util
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def build():
    spec = importlib.util.spec_from_file_location("paras_build", os.path.join(ROOT, "framework-torch-paras_b200", "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def included(source, dirs):
    found, todo = set(), [source]
    while todo:
        path = todo.pop()
        for name in re.findall(r'^\s*#\s*include\s+"([^"]+)"', open(path).read(), re.M):
            for d in [os.path.dirname(path), *dirs]:
                h = os.path.normpath(os.path.join(d, name))
                if os.path.exists(h) and h not in found:
                    found.add(h)
                    todo.append(h)
    return found


@pytest.mark.parametrize("part", ["lib", "ext"])
def test_a_changed_header_rebuilds_what_includes_it(build, part, monkeypatch):
    deps = {}

    def newer(target, d):
        deps[target] = {os.path.normpath(x) for x in d}
        return False

    monkeypatch.setattr(build, "_newer", newer)
    monkeypatch.setattr(build, "_run", lambda *a: pytest.fail("nothing is to be built"))
    getattr(build, "build_" + part)()
    folder, sources = ("compat", build.CUDA_SOURCES) if part == "lib" else ("", build.EXT_SOURCES)
    for s in sources:
        path = os.path.normpath(os.path.join(build.CSRC, folder, s))
        mine = [d for d in deps.values() if path in d]
        assert len(mine) == 1
        missing = included(path, [build.CSRC, os.path.join(build.CSRC, "compat"), build.INCLUDE]) - mine[0]
        assert not missing, f"{s}: {sorted(missing)}"
